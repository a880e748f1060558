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

// Autograd's count of writes to an argument: a graph that saved it for its backward then refuses to use what it holds now.
// (No graph can save a tensor made in inference mode, and it has no count.)
void written(Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
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
  // Rows of a sequence lie one behind the other, near enough for 32-bit offsets inside a tile of tokens.
  const int64_t d = t.dim() - inner - 1;
  if (d > 0 && t.size(d) != 1 && (t.stride(d) < want || t.stride(d) > (int64_t{1} << 21))) return t.contiguous();
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

Tensor short_conv_step_out(const Tensor& x, const Tensor& state, const Tensor& weight, const OptTensor& bias, bool silu,
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
  written(state_out);
  return out;
}

std::tuple<Tensor, Tensor> short_conv_step(const Tensor& x, const Tensor& state, const Tensor& weight,
                                           const OptTensor& bias, bool silu) {
  Tensor moved = at::empty(state.sizes(), state.options());
  return {short_conv_step_out(x, state, weight, bias, silu, moved), moved};
}

// ---------------------------------------------------------------------------
// Selective scan.

bool aligned16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// The checked inputs of a call and what keeps their memory alive.
struct Scan {
  int64_t B, T, H, P, G, N;
  grm_hip_selective_args args;
  Tensor keys, values, queries, steps, rates, skip, bias, lengths, memory;
};

Tensor f32_state(const Tensor& t) {
  Tensor m = t.contiguous();
  return aligned16(m) ? m : m.clone();
}

// `step`: one token, without the length's dimension.
Scan check_scan(const Tensor& keys, const Tensor& values, const Tensor& queries, const Tensor& steps,
                const Tensor& rates, const OptTensor& memory, const OptTensor& skip, const OptTensor& step_bias,
                const OptTensor& lengths, bool softplus, bool step, const char* op) {
  const int64_t lead = step ? 1 : 2;
  TORCH_CHECK_VALUE(keys.dim() == lead + 2 && queries.dim() == lead + 2 && values.dim() == lead + 2 &&
                        steps.dim() == lead + 1,
                    op, step ? ": keys and queries must be [batch, groups, key_dim], values [batch, heads, value_dim] and "
                               "steps [batch, heads]"
                             : ": keys and queries must be [batch, seq_len, groups, key_dim], values [batch, seq_len, "
                               "heads, value_dim] and steps [batch, seq_len, heads]");
  Scan s{};
  s.B = values.size(0); s.T = step ? 1 : values.size(1); s.H = values.size(-2); s.P = values.size(-1);
  s.G = keys.size(-2); s.N = keys.size(-1);
  TORCH_CHECK_VALUE(queries.sizes() == keys.sizes() && keys.size(0) == s.B && steps.size(0) == s.B &&
                        steps.size(-1) == s.H && (step || (keys.size(1) == s.T && steps.size(1) == s.T)),
                    op, ": keys, queries, values and steps must agree in batch, length and heads");
  TORCH_CHECK_VALUE(s.G >= 1 && s.H >= 1 && s.P >= 1 && s.H % s.G == 0 && s.N >= 1 && s.N <= 128, op,
                    ": heads must be a multiple of groups and key_dim in [1, 128]");
  const int dt = dtype_code(values, op, "values"), sdt = dtype_code(steps, op, "steps");
  TORCH_CHECK_VALUE(keys.scalar_type() == values.scalar_type() && queries.scalar_type() == values.scalar_type() &&
                        (sdt == dt || sdt == GRM_HIP_F32),
                    op, ": keys, values and queries must share a type, steps have it or float32");
  check_device(keys, values, op, "keys");
  check_device(queries, values, op, "queries");
  check_device(steps, values, op, "steps");
  auto per_head = [&](const Tensor& t, const char* name) {
    check_device(t, values, op, name);
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == s.H && t.scalar_type() == at::kFloat, op, ": ", name,
                      " must be float32 [heads]");
    return t.contiguous();
  };
  s.rates = per_head(rates, "rates");
  if (has(skip)) s.skip = per_head(*skip, "skip");
  if (has(step_bias)) s.bias = per_head(*step_bias, "step_bias");
  if (has(memory)) {
    check_device(*memory, values, op, "memory");
    TORCH_CHECK_VALUE(memory->sizes() == at::IntArrayRef({s.B, s.H, s.P, s.N}) && memory->scalar_type() == at::kFloat,
                      op, ": memory must be float32 [batch, heads, value_dim, key_dim]");
    s.memory = f32_state(*memory);
  }
  s.keys = packed_rows(keys, 2);
  s.values = packed_rows(values, 2);
  s.queries = packed_rows(queries, 2);
  s.steps = packed_rows(steps, 1);
  grm_hip_selective_args& a = s.args;
  a.keys = s.keys.data_ptr(); a.values = s.values.data_ptr(); a.queries = s.queries.data_ptr();
  a.steps = s.steps.data_ptr();
  a.rates = s.rates.data_ptr<float>();
  a.skip = s.skip.defined() ? s.skip.data_ptr<float>() : nullptr;
  a.step_bias = s.bias.defined() ? s.bias.data_ptr<float>() : nullptr;
  a.lengths = lengths_ptr(lengths, s.B, values, op, s.lengths);
  a.memory = s.memory.defined() ? s.memory.data_ptr<float>() : nullptr;
  a.batch = s.B; a.seq_len = s.T; a.heads = s.H; a.value_dim = s.P; a.groups = s.G; a.key_dim = s.N;
  auto strides = [&](const Tensor& t, int64_t width, int64_t* batch, int64_t* token) {
    *batch = stride_of(t, 0, s.T * width);
    *token = step ? width : stride_of(t, 1, width);
  };
  strides(s.keys, s.G * s.N, &a.keys_batch_stride, &a.keys_token_stride);
  strides(s.values, s.H * s.P, &a.values_batch_stride, &a.values_token_stride);
  strides(s.queries, s.G * s.N, &a.queries_batch_stride, &a.queries_token_stride);
  strides(s.steps, s.H, &a.steps_batch_stride, &a.steps_token_stride);
  a.dtype = dt; a.steps_dtype = sdt; a.softplus = softplus;
  return s;
}

Tensor bytes(int64_t n, const Tensor& like) {
  return at::empty({std::max<int64_t>(n, 16)}, like.options().dtype(at::kByte));
}

std::tuple<Tensor, Tensor, Tensor> selective_scan_forward(const Tensor& keys, const Tensor& values,
                                                          const Tensor& queries, const Tensor& steps,
                                                          const Tensor& rates, const OptTensor& memory,
                                                          const OptTensor& skip, const OptTensor& step_bias,
                                                          const OptTensor& lengths, bool softplus, bool save) {
  const char* op = "selective_scan";
  c10::OptionalDeviceGuard guard(values.device());
  const Scan s = check_scan(keys, values, queries, steps, rates, memory, skip, step_bias, lengths, softplus, false, op);
  const auto f32 = values.options().dtype(at::kFloat);
  Tensor hidden = at::empty({s.B, s.T, s.H, s.P}, values.options());
  Tensor memory_out = at::empty({s.B, s.H, s.P, s.N}, f32);
  const int64_t block = grm_hip_selective_scan_block(s.args.dtype);
  Tensor states = save ? at::empty({s.B, (s.T + block - 1) / block, s.H, s.P, s.N}, f32) : at::empty({0}, f32);
  const int64_t wsb = grm_hip_selective_scan_workspace(s.B, s.T, s.H, s.P, s.N, s.args.dtype);
  Tensor ws = bytes(wsb, values);
  check_rc(grm_hip_selective_scan_fwd(&s.args, hidden.data_ptr(), memory_out.data_ptr<float>(),
                                      save ? states.data_ptr<float>() : nullptr, ws.data_ptr(), wsb, stream_of(values)),
           op);
  return {hidden, memory_out, states};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> selective_scan_backward(
    const OptTensor& grad_hidden, const OptTensor& grad_memory_out, const Tensor& keys, const Tensor& values,
    const Tensor& queries, const Tensor& steps, const Tensor& rates, const OptTensor& skip, const OptTensor& step_bias,
    const OptTensor& lengths, const Tensor& states, bool softplus) {
  const char* op = "selective_scan backward";
  c10::OptionalDeviceGuard guard(values.device());
  const Scan s =
      check_scan(keys, values, queries, steps, rates, c10::nullopt, skip, step_bias, lengths, softplus, false, op);
  const auto f32 = values.options().dtype(at::kFloat);
  const int64_t block = grm_hip_selective_scan_block(s.args.dtype);
  check_device(states, values, op, "states");
  TORCH_CHECK_VALUE(states.sizes() == at::IntArrayRef({s.B, (s.T + block - 1) / block, s.H, s.P, s.N}) &&
                        states.scalar_type() == at::kFloat,
                    op, ": states must be what the forward kept");
  Tensor dy, dm, st = f32_state(states);
  if (has(grad_hidden)) {
    check_device(*grad_hidden, values, op, "grad_hidden");
    TORCH_CHECK_VALUE(grad_hidden->sizes() == values.sizes() && grad_hidden->scalar_type() == values.scalar_type(), op,
                      ": grad_hidden must match values");
    dy = grad_hidden->contiguous();
  } else {
    dy = at::zeros(values.sizes(), values.options());
  }
  if (has(grad_memory_out)) {
    check_device(*grad_memory_out, values, op, "grad_memory_out");
    TORCH_CHECK_VALUE(grad_memory_out->sizes() == at::IntArrayRef({s.B, s.H, s.P, s.N}) &&
                          grad_memory_out->scalar_type() == at::kFloat,
                      op, ": grad_memory_out must be float32 [batch, heads, value_dim, key_dim]");
    dm = f32_state(*grad_memory_out);
  }
  Tensor gk = at::empty(keys.sizes(), values.options()), gv = at::empty(values.sizes(), values.options()),
         gq = at::empty(keys.sizes(), values.options()), gst = at::empty(steps.sizes(), steps.options());
  Tensor gr = at::empty({s.H}, f32), gm = at::empty({s.B, s.H, s.P, s.N}, f32), gsk = at::empty({s.H}, f32),
         gb = at::empty({s.H}, f32);
  const int64_t wsb = grm_hip_selective_scan_bwd_workspace(s.B, s.T, s.H, s.P, s.G, s.N, s.args.dtype);
  Tensor ws = bytes(wsb, values);
  check_rc(grm_hip_selective_scan_bwd(&s.args, st.data_ptr<float>(), dy.data_ptr(),
                                      dm.defined() ? dm.data_ptr<float>() : nullptr, gk.data_ptr(), gv.data_ptr(),
                                      gq.data_ptr(), gst.data_ptr(), gr.data_ptr<float>(), gm.data_ptr<float>(),
                                      gsk.data_ptr<float>(), gb.data_ptr<float>(), ws.data_ptr(), wsb,
                                      stream_of(values)),
           op);
  return {gk, gv, gq, gst, gr, gm, gsk, gb};
}

Tensor selective_step_out(const Tensor& keys, const Tensor& values, const Tensor& queries, const Tensor& steps,
                      const Tensor& rates, const Tensor& memory, const OptTensor& skip, const OptTensor& step_bias,
                      bool softplus, Tensor& memory_out) {
  const char* op = "selective_step";
  c10::OptionalDeviceGuard guard(values.device());
  const Scan s = check_scan(keys, values, queries, steps, rates, memory, skip, step_bias, c10::nullopt, softplus, true, op);
  check_device(memory_out, values, op, "memory_out");
  TORCH_CHECK_VALUE(memory_out.sizes() == memory.sizes() && memory_out.scalar_type() == at::kFloat &&
                        memory_out.is_contiguous() && aligned16(memory_out),
                    op, ": memory_out must be contiguous, 16-byte aligned and match memory");
  Tensor hidden = at::empty({s.B, s.H, s.P}, values.options());
  check_rc(grm_hip_selective_step(&s.args, hidden.data_ptr(), memory_out.data_ptr<float>(), stream_of(values)), op);
  written(memory_out);
  return hidden;
}

std::tuple<Tensor, Tensor> selective_step(const Tensor& keys, const Tensor& values, const Tensor& queries,
                                          const Tensor& steps, const Tensor& rates, const Tensor& memory,
                                          const OptTensor& skip, const OptTensor& step_bias, bool softplus) {
  Tensor moved = at::empty(memory.sizes(), memory.options());
  return {selective_step_out(keys, values, queries, steps, rates, memory, skip, step_bias, softplus, moved), moved};
}

}  // namespace
}  // namespace grm_selective

TORCH_LIBRARY_FRAGMENT(grm_cuda, m) {
  m.def("short_conv_forward(Tensor x, Tensor weight, Tensor? bias, Tensor? state, Tensor? lengths, bool silu) -> (Tensor out, Tensor state_out)");
  m.def("short_conv_backward(Tensor? grad_out, Tensor? grad_state_out, Tensor x, Tensor weight, Tensor? bias, Tensor? state, Tensor? lengths, bool silu) -> (Tensor grad_x, Tensor grad_weight, Tensor grad_bias, Tensor grad_state)");
  m.def("short_conv_step(Tensor x, Tensor state, Tensor weight, Tensor? bias, bool silu) -> (Tensor out, Tensor state_out)");
  m.def("short_conv_step_out(Tensor x, Tensor state, Tensor weight, Tensor? bias, bool silu, Tensor(a!) state_out) -> Tensor");
  m.def("selective_scan_forward(Tensor keys, Tensor values, Tensor queries, Tensor steps, Tensor rates, Tensor? memory, Tensor? skip, Tensor? step_bias, Tensor? lengths, bool softplus, bool save) -> (Tensor hidden, Tensor memory_out, Tensor states)");
  m.def("selective_scan_backward(Tensor? grad_hidden, Tensor? grad_memory_out, Tensor keys, Tensor values, Tensor queries, Tensor steps, Tensor rates, Tensor? skip, Tensor? step_bias, Tensor? lengths, Tensor states, bool softplus) -> (Tensor grad_keys, Tensor grad_values, Tensor grad_queries, Tensor grad_steps, Tensor grad_rates, Tensor grad_memory, Tensor grad_skip, Tensor grad_step_bias)");
  m.def("selective_step(Tensor keys, Tensor values, Tensor queries, Tensor steps, Tensor rates, Tensor memory, Tensor? skip, Tensor? step_bias, bool softplus) -> (Tensor hidden, Tensor memory_out)");
  m.def("selective_step_out(Tensor keys, Tensor values, Tensor queries, Tensor steps, Tensor rates, Tensor memory, Tensor? skip, Tensor? step_bias, bool softplus, Tensor(a!) memory_out) -> Tensor");
}

TORCH_LIBRARY_IMPL(grm_cuda, CUDA, m) {
  m.impl("short_conv_forward", grm_selective::short_conv_forward);
  m.impl("short_conv_backward", grm_selective::short_conv_backward);
  m.impl("short_conv_step", grm_selective::short_conv_step);
  m.impl("short_conv_step_out", grm_selective::short_conv_step_out);
  m.impl("selective_scan_forward", grm_selective::selective_scan_forward);
  m.impl("selective_scan_backward", grm_selective::selective_scan_backward);
  m.impl("selective_step", grm_selective::selective_step);
  m.impl("selective_step_out", grm_selective::selective_step_out);
}
