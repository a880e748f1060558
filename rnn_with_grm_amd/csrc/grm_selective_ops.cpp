// torch.ops.grm_cuda: the selective state scan and its short causal convolution, on the CUDA
// key (HIP devices dispatch there in PyTorch-ROCm).  Each op checks its inputs, allocates its
// outputs and workspace with ATen on the inputs' device and calls the C ABI of libgrm_hip.so on
// that device's current stream.  Inputs the kernels do not cover raise; CPU tensors take
// cuda_ops' PyTorch forms and never reach these ops.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <initializer_list>
#include <tuple>

#include "grm_hip.h"

namespace grm_selective {
namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

int dtype_code(const Tensor& t, const char* op, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return GRM_HIP_F32;
    case at::kHalf: return GRM_HIP_F16;
    case at::kBFloat16: return GRM_HIP_BF16;
    default: break;
  }
  TORCH_CHECK_VALUE(false, op, ": ", name, " must be float32, float16 or bfloat16, got ", t.scalar_type());
  return -1;
}

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

void* stream_of(const Tensor& t) {
  return static_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

void check_rc(int rc, const char* op) {
  TORCH_CHECK(rc == GRM_HIP_OK, op, " failed (", rc, "): ", grm_hip_last_error());
}

void check_device(const Tensor& t, const Tensor& like, const char* op, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == like.device(), op, ": ", name, " must be on ", like.device());
}

// A contiguous optional tensor's pointer; `keep` holds what it points into.
void* opt_ptr(const OptTensor& t, Tensor& keep) {
  if (!has(t)) return nullptr;
  keep = t->contiguous();
  return keep.data_ptr();
}

// Rows of the last `inner` dimensions packed, any stride between tokens and sequences: a slice of a
// wider projection is read where it lies.
Tensor packed_rows(const Tensor& t, int64_t inner) {
  int64_t want = 1;
  for (int64_t d = t.dim() - 1; d >= t.dim() - inner; --d) {
    if (t.size(d) != 1 && t.stride(d) != want) return t.contiguous();
    want *= t.size(d);
  }
  for (int64_t d = 0; d < t.dim() - inner; ++d) {  // byte offsets inside a tile of tokens stay below 2^31
    if (t.size(d) != 1 && d > 0 && t.stride(d) > (int64_t{1} << 21)) return t.contiguous();
  }
  return t;
}

int64_t stride_of(const Tensor& t, int64_t dim, int64_t packed) { return t.size(dim) > 1 ? t.stride(dim) : packed; }

const int64_t* lengths_ptr(const OptTensor& lengths, int64_t B, const Tensor& like, const char* op, Tensor& keep) {
  if (!has(lengths)) return nullptr;
  check_device(*lengths, like, op, "lengths");
  TORCH_CHECK_VALUE(lengths->dim() == 1 && lengths->size(0) == B &&
                  (lengths->scalar_type() == at::kLong || lengths->scalar_type() == at::kInt),
              op, ": lengths must be int32 or int64 [batch]");
  keep = lengths->to(at::kLong).contiguous();
  return keep.data_ptr<int64_t>();
}

// ---------------------------------------------------------------------------
// Short convolution.

struct Conv {
  int64_t B, T, C, W;
  int dtype, w_dtype;
};

Conv check_conv(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& state, bool step,
                const char* op) {
  TORCH_CHECK_VALUE(x.dim() == (step ? 2 : 3), op, ": x must be ", step ? "[batch, channels]" : "[batch, seq_len, channels]");
  Conv c{x.size(0), step ? 1 : x.size(1), x.size(-1), 0, dtype_code(x, op, "x"), 0};
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(0) == c.C, op, ": weight must be [channels, width]");
  c.W = weight.size(1);
  TORCH_CHECK_VALUE(c.C >= 1 && c.W >= 2 && c.W <= 4, op, ": needs channels >= 1 and width 2, 3 or 4, got width ", c.W);
  TORCH_CHECK_VALUE(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat, op,
              ": weight must have x's type or be float32");
  c.w_dtype = dtype_code(weight, op, "weight");
  check_device(weight, x, op, "weight");
  if (has(bias)) {
    check_device(*bias, x, op, "bias");
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == c.C && bias->scalar_type() == weight.scalar_type(), op,
                ": bias must be [channels] in weight's type");
  }
  if (has(state)) {
    check_device(*state, x, op, "state");
    TORCH_CHECK_VALUE(state->dim() == 3 && state->size(0) == c.B && state->size(1) == c.W - 1 && state->size(2) == c.C &&
                    state->scalar_type() == x.scalar_type(),
                op, ": state must be [batch, width - 1, channels] in x's type");
  }
  return c;
}

std::tuple<Tensor, Tensor> short_conv_forward(const Tensor& x, const Tensor& weight, const OptTensor& bias,
                                              const OptTensor& state, const OptTensor& lengths, bool silu) {
  const char* op = "short_conv";
  const Conv c = check_conv(x, weight, bias, state, false, op);
  c10::OptionalDeviceGuard guard(x.device());
  Tensor xr = packed_rows(x, 1), w = weight.contiguous(), kb, ks, kl;
  Tensor out = at::empty({c.B, c.T, c.C}, x.options());
  Tensor state_out = at::empty({c.B, c.W - 1, c.C}, x.options());
  const void *bp = opt_ptr(bias, kb), *sp = opt_ptr(state, ks);
  const int64_t* lp = lengths_ptr(lengths, c.B, x, op, kl);
  check_rc(grm_hip_short_conv_fwd(xr.data_ptr(), w.data_ptr(), bp, sp, lp, out.data_ptr(), state_out.data_ptr(), c.B,
                                  c.T, c.C, c.W, stride_of(xr, 0, c.T * c.C), stride_of(xr, 1, c.C), c.dtype,
                                  c.w_dtype, silu, stream_of(x)),
           op);
  return {out, state_out};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> short_conv_backward(const OptTensor& grad_out,
                                                               const OptTensor& grad_state_out, const Tensor& x,
                                                               const Tensor& weight, const OptTensor& bias,
                                                               const OptTensor& state, const OptTensor& lengths,
                                                               bool silu) {
  const char* op = "short_conv backward";
  const Conv c = check_conv(x, weight, bias, state, false, op);
  if (has(grad_out)) {
    check_device(*grad_out, x, op, "grad_out");
    TORCH_CHECK_VALUE(grad_out->sizes() == x.sizes() && grad_out->scalar_type() == x.scalar_type(), op,
                ": grad_out must match x");
  }
  if (has(grad_state_out)) {
    check_device(*grad_state_out, x, op, "grad_state_out");
    TORCH_CHECK_VALUE(grad_state_out->sizes() == at::IntArrayRef({c.B, c.W - 1, c.C}) &&
                    grad_state_out->scalar_type() == x.scalar_type(),
                op, ": grad_state_out must be [batch, width - 1, channels] in x's type");
  }
  c10::OptionalDeviceGuard guard(x.device());
  Tensor xr = packed_rows(x, 1), w = weight.contiguous(), kb, ks, kl, kg, kgs;
  Tensor dx = at::empty({c.B, c.T, c.C}, x.options()), dw = at::empty({c.C, c.W}, weight.options());
  Tensor db = has(bias) ? at::empty({c.C}, weight.options()) : Tensor();
  Tensor dstate = has(state) ? at::empty({c.B, c.W - 1, c.C}, x.options()) : Tensor();
  const void *bp = opt_ptr(bias, kb), *sp = opt_ptr(state, ks), *gp = opt_ptr(grad_out, kg),
             *gsp = opt_ptr(grad_state_out, kgs);
  const int64_t* lp = lengths_ptr(lengths, c.B, x, op, kl);
  const int64_t wsb = grm_hip_short_conv_bwd_workspace(c.B, c.T, c.C, c.W, c.dtype);
  Tensor ws = at::empty({std::max<int64_t>(wsb / 4, 1)}, x.options().dtype(at::kFloat));
  check_rc(grm_hip_short_conv_bwd(xr.data_ptr(), w.data_ptr(), bp, sp, lp, gp, gsp, dx.data_ptr(), dw.data_ptr(),
                                  db.defined() ? db.data_ptr() : nullptr,
                                  dstate.defined() ? dstate.data_ptr() : nullptr, ws.data_ptr(), wsb, c.B, c.T, c.C,
                                  c.W, stride_of(xr, 0, c.T * c.C), stride_of(xr, 1, c.C), c.dtype, c.w_dtype, silu,
                                  stream_of(x)),
           op);
  return {dx, dw, db.defined() ? db : at::empty({0}, weight.options()),
          dstate.defined() ? dstate : at::empty({0}, x.options())};
}

Tensor short_conv_step(const Tensor& x, const Tensor& state, const Tensor& weight, const OptTensor& bias, bool silu,
                       Tensor& state_out) {
  const char* op = "short_conv_step";
  const Conv c = check_conv(x, weight, bias, state, true, op);
  check_device(state_out, x, op, "state_out");
  TORCH_CHECK_VALUE(state_out.sizes() == state.sizes() && state_out.scalar_type() == x.scalar_type() &&
                  state_out.is_contiguous(),
              op, ": state_out must be contiguous and match state");
  c10::OptionalDeviceGuard guard(x.device());
  Tensor xr = packed_rows(x, 1), w = weight.contiguous(), st = state.contiguous(), kb;
  Tensor out = at::empty({c.B, c.C}, x.options());
  const void* bp = opt_ptr(bias, kb);
  check_rc(grm_hip_short_conv_step(xr.data_ptr(), w.data_ptr(), bp, st.data_ptr(), out.data_ptr(),
                                   state_out.data_ptr(), c.B, c.C, c.W, stride_of(xr, 0, c.C), c.dtype, c.w_dtype,
                                   silu, stream_of(x)),
           op);
  return out;
}

}  // namespace
}  // namespace grm_selective

TORCH_LIBRARY_FRAGMENT(grm_cuda, m) {
  m.def("short_conv_forward(Tensor x, Tensor weight, Tensor? bias, Tensor? state, Tensor? lengths, bool silu) -> (Tensor out, Tensor state_out)");
  m.def("short_conv_backward(Tensor? grad_out, Tensor? grad_state_out, Tensor x, Tensor weight, Tensor? bias, Tensor? state, Tensor? lengths, bool silu) -> (Tensor grad_x, Tensor grad_weight, Tensor grad_bias, Tensor grad_state)");
  m.def("short_conv_step(Tensor x, Tensor state, Tensor weight, Tensor? bias, bool silu, Tensor(a!) state_out) -> Tensor");
}

TORCH_LIBRARY_IMPL(grm_cuda, CUDA, m) {
  m.impl("short_conv_forward", grm_selective::short_conv_forward);
  m.impl("short_conv_backward", grm_selective::short_conv_backward);
  m.impl("short_conv_step", grm_selective::short_conv_step);
}
