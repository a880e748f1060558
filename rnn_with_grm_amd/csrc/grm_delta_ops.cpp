// torch.ops.grm_cuda: the gated delta rule and the group norm behind it, on the CUDA key (HIP devices dispatch there in PyTorch-ROCm).  Each op
// checks its inputs, allocates its outputs and workspace with ATen on the inputs' device and calls the C ABI of libgrm_hip.so
// on that device's current stream.  Inputs the kernels do not cover raise; CPU tensors take cuda_ops' PyTorch forms.
#include <tuple>

#include "delta_limits.h"
#include "op_checks.h"

namespace grm_delta {
namespace {

using namespace grm_ops;

constexpr int64_t kTokens = 64;  // of a chunk, whose state the forward keeps for the backward

// The checked inputs of a call and what keeps their memory alive.
struct Delta {
  int64_t B, T, H, P, G, N;
  grm_hip_delta_args args;
  Tensor keys, values, queries, strengths, decays, lengths, memory;
};

// `step`: one token, without the length's dimension.
Delta check_delta(const Tensor& keys, const Tensor& values, const Tensor& queries, const Tensor& strengths,
                  const OptTensor& decays, const OptTensor& memory, const OptTensor& lengths, bool step, const char* op) {
  const int64_t lead = step ? 1 : 2;
  TORCH_CHECK_VALUE(keys.dim() == lead + 2 && queries.dim() == lead + 2 && values.dim() == lead + 2 &&
                        strengths.dim() == lead + 1 && (!has(decays) || decays->dim() == lead + 1),
                    op, step ? ": keys and queries must be [batch, groups, key_dim], values [batch, heads, value_dim], "
                               "strengths and log_decays [batch, heads]"
                             : ": keys and queries must be [batch, seq_len, groups, key_dim], values [batch, seq_len, "
                               "heads, value_dim], strengths and log_decays [batch, seq_len, heads]");
  Delta s{};
  s.B = values.size(0); s.T = step ? 1 : values.size(1); s.H = values.size(-2); s.P = values.size(-1);
  s.G = keys.size(-2); s.N = keys.size(-1);
  TORCH_CHECK_VALUE(queries.sizes() == keys.sizes() && keys.size(0) == s.B && strengths.size(0) == s.B &&
                        strengths.size(-1) == s.H && (step || (keys.size(1) == s.T && strengths.size(1) == s.T)) &&
                        (!has(decays) || decays->sizes() == strengths.sizes()),
                    op, ": keys, queries, values, strengths and log_decays must agree in batch, length and heads");
  TORCH_CHECK_VALUE(s.G >= 1 && s.H >= 1 && s.P >= 1 && s.H % s.G == 0 && s.N >= 1 && s.N <= 128, op,
                    ": heads must be a multiple of groups and key_dim in [1, 128]");
  const int dt = dtype_code(values, op, "values"), sdt = dtype_code(strengths, op, "strengths");
  const int ddt = has(decays) ? dtype_code(*decays, op, "log_decays") : GRM_HIP_F32;
  TORCH_CHECK_VALUE(keys.scalar_type() == values.scalar_type() && queries.scalar_type() == values.scalar_type() &&
                        (sdt == dt || sdt == GRM_HIP_F32) && (ddt == dt || ddt == GRM_HIP_F32),
                    op, ": keys, values and queries must share a type, strengths and log_decays have it or float32");
  const char* limit = grmhip::delta_limit(s.B, s.T, s.H, s.P, s.G, s.N, step);
  TORCH_CHECK(limit == nullptr, op, ": ", limit == nullptr ? "" : limit);
  check_device(keys, values, op, "keys");
  check_device(queries, values, op, "queries");
  check_device(strengths, values, op, "strengths");
  if (has(decays)) check_device(*decays, values, op, "log_decays");
  if (has(memory)) {
    check_device(*memory, values, op, "memory");
    TORCH_CHECK_VALUE(memory->sizes() == at::IntArrayRef({s.B, s.H, s.P, s.N}) && memory->scalar_type() == at::kFloat,
                      op, ": memory must be float32 [batch, heads, value_dim, key_dim]");
    s.memory = f32_state(*memory);
  }
  s.keys = packed_rows(keys, 2);
  s.values = packed_rows(values, 2);
  s.queries = packed_rows(queries, 2);
  s.strengths = packed_rows(strengths, 1);
  if (has(decays)) s.decays = packed_rows(*decays, 1);
  grm_hip_delta_args& a = s.args;
  a.keys = s.keys.data_ptr(); a.values = s.values.data_ptr(); a.queries = s.queries.data_ptr();
  a.strengths = s.strengths.data_ptr();
  a.log_decays = s.decays.defined() ? s.decays.data_ptr() : nullptr;
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
  strides(s.strengths, s.H, &a.strengths_batch_stride, &a.strengths_token_stride);
  if (s.decays.defined()) strides(s.decays, s.H, &a.decays_batch_stride, &a.decays_token_stride);
  a.dtype = dt; a.strengths_dtype = sdt; a.decays_dtype = ddt;
  return s;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> delta_scan_forward(const Tensor& keys, const Tensor& values,
                                                              const Tensor& queries, const Tensor& strengths,
                                                              const OptTensor& log_decays, const OptTensor& memory,
                                                              const OptTensor& lengths, bool save) {
  const char* op = "delta_scan";
  c10::OptionalDeviceGuard guard(values.device());
  const Delta s = check_delta(keys, values, queries, strengths, log_decays, memory, lengths, false, op);
  const auto f32 = values.options().dtype(at::kFloat);
  Tensor hidden = at::empty({s.B, s.T, s.H, s.P}, values.options());
  Tensor memory_out = at::empty({s.B, s.H, s.P, s.N}, f32);
  Tensor states = save ? at::empty({s.B, (s.T + kTokens - 1) / kTokens, s.H, s.P, s.N}, f32) : at::empty({0}, f32);
  Tensor miss = save ? at::empty({s.B, s.T, s.H, s.P}, f32) : at::empty({0}, f32);
  const int64_t wsb = grm_hip_delta_scan_workspace(s.B, s.T, s.H, s.P, s.N, s.args.dtype);
  Tensor ws = bytes(wsb, values);
  check_rc(grm_hip_delta_scan_fwd(&s.args, hidden.data_ptr(), memory_out.data_ptr<float>(),
                                  save ? states.data_ptr<float>() : nullptr, save ? miss.data_ptr<float>() : nullptr,
                                  ws.data_ptr(), wsb, stream_of(values)),
           op);
  return {hidden, memory_out, states, miss};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> delta_scan_backward(
    const OptTensor& grad_hidden, const OptTensor& grad_memory_out, const Tensor& keys, const Tensor& values,
    const Tensor& queries, const Tensor& strengths, const OptTensor& log_decays, const OptTensor& lengths,
    const Tensor& states, const Tensor& miss) {
  const char* op = "delta_scan backward";
  c10::OptionalDeviceGuard guard(values.device());
  const Delta s = check_delta(keys, values, queries, strengths, log_decays, c10::nullopt, lengths, false, op);
  const auto f32 = values.options().dtype(at::kFloat);
  check_device(states, values, op, "states");
  check_device(miss, values, op, "miss");
  TORCH_CHECK_VALUE(states.sizes() == at::IntArrayRef({s.B, (s.T + kTokens - 1) / kTokens, s.H, s.P, s.N}) &&
                        states.scalar_type() == at::kFloat && miss.sizes() == values.sizes() &&
                        miss.scalar_type() == at::kFloat,
                    op, ": states and miss must be what the forward kept");
  Tensor dy, dm, st = f32_state(states), ms = miss.contiguous();
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
         gq = at::empty(keys.sizes(), values.options()), gb = at::empty(strengths.sizes(), strengths.options());
  Tensor gd = has(log_decays) ? at::empty(log_decays->sizes(), log_decays->options()) : at::empty({0}, f32);
  Tensor gm = at::empty({s.B, s.H, s.P, s.N}, f32);
  const int64_t wsb = grm_hip_delta_scan_bwd_workspace(s.B, s.T, s.H, s.P, s.G, s.N);
  Tensor ws = bytes(wsb, values);
  check_rc(grm_hip_delta_scan_bwd(&s.args, st.data_ptr<float>(), ms.data_ptr<float>(), dy.data_ptr(),
                                  dm.defined() ? dm.data_ptr<float>() : nullptr, gk.data_ptr(), gv.data_ptr(),
                                  gq.data_ptr(), gb.data_ptr(), has(log_decays) ? gd.data_ptr() : nullptr,
                                  gm.data_ptr<float>(), ws.data_ptr(), wsb, stream_of(values)),
           op);
  return {gk, gv, gq, gb, gd, gm};
}

Tensor step(const Delta& s, const Tensor& values, Tensor& memory_out, const char* op) {
  Tensor hidden = at::empty({s.B, s.H, s.P}, values.options());
  check_rc(grm_hip_delta_step(&s.args, hidden.data_ptr(), memory_out.data_ptr<float>(), stream_of(values)), op);
  return hidden;
}

Tensor delta_step_out(const Tensor& keys, const Tensor& values, const Tensor& queries, const Tensor& strengths,
                      const OptTensor& log_decays, const Tensor& memory, Tensor& memory_out) {
  const char* op = "delta_step";
  c10::OptionalDeviceGuard guard(values.device());
  const Delta s = check_delta(keys, values, queries, strengths, log_decays, memory, c10::nullopt, true, op);
  check_device(memory_out, values, op, "memory_out");
  TORCH_CHECK_VALUE(memory_out.sizes() == memory.sizes() && memory_out.scalar_type() == at::kFloat &&
                        memory_out.is_contiguous() && aligned16(memory_out),
                    op, ": memory_out must be contiguous, 16-byte aligned and match memory");
  Tensor hidden = step(s, values, memory_out, op);
  written(memory_out);
  return hidden;
}

std::tuple<Tensor, Tensor> delta_step(const Tensor& keys, const Tensor& values, const Tensor& queries,
                                      const Tensor& strengths, const OptTensor& log_decays, const Tensor& memory) {
  const char* op = "delta_step";
  c10::OptionalDeviceGuard guard(values.device());
  const Delta s = check_delta(keys, values, queries, strengths, log_decays, memory, c10::nullopt, true, op);
  Tensor moved = at::empty(memory.sizes(), memory.options());
  return {step(s, values, moved, op), moved};
}

// ---------------------------------------------------------------------------
// Group norm.

// Rows of packed channels, any stride between them.
struct Norm {
  int64_t rows, C;
  int dtype, w_dtype;
};

Norm check_norm(const Tensor& x, int64_t groups, const OptTensor& weight, const OptTensor& bias, const OptTensor& gate,
                const char* op) {
  TORCH_CHECK_VALUE(x.dim() == 2, op, ": x must be [rows, channels]");
  Norm n{x.size(0), x.size(1), dtype_code(x, op, "x"), 0};
  TORCH_CHECK_VALUE(n.C >= 1 && groups >= 1 && n.C % groups == 0, op, ": channels must be a multiple of groups");
  TORCH_CHECK_VALUE(n.C / groups <= 4096, op, ": at most 4096 channels a group");
  TORCH_CHECK(n.C <= (int64_t{1} << 21) && n.rows <= (int64_t{1} << 31), op, ": at most 2^21 channels and 2^31 rows");
  n.w_dtype = n.dtype;
  auto param = [&](const OptTensor& t, const char* name) {
    if (!has(t)) return;
    check_device(*t, x, op, name);
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == n.C && (t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat),
                      op, ": ", name, " must be [channels] in x's type or float32");
    n.w_dtype = dtype_code(*t, op, name);
  };
  param(weight, "weight");
  param(bias, "bias");
  TORCH_CHECK_VALUE(!has(weight) || !has(bias) || weight->scalar_type() == bias->scalar_type(), op,
                    ": weight and bias must share a type");
  if (has(gate)) {
    check_device(*gate, x, op, "gate");
    TORCH_CHECK_VALUE(gate->sizes() == x.sizes() && gate->scalar_type() == x.scalar_type(), op, ": gate must match x");
  }
  return n;
}

Tensor packed_channels(const Tensor& t) {
  if ((t.size(1) != 1 && t.stride(1) != 1) || (t.size(0) > 1 && (t.stride(0) < t.size(1) || t.stride(0) > (int64_t{1} << 31))))
    return t.contiguous();
  return t;
}

Tensor group_norm_forward(const Tensor& x, int64_t groups, const OptTensor& weight, const OptTensor& bias,
                          const OptTensor& gate, bool silu, bool center, double eps) {
  const char* op = "group_norm";
  const Norm n = check_norm(x, groups, weight, bias, gate, op);
  c10::OptionalDeviceGuard guard(x.device());
  Tensor xr = packed_channels(x), gr = has(gate) ? packed_channels(*gate) : Tensor(), kw, kb;
  Tensor out = at::empty({n.rows, n.C}, x.options());
  const void *wp = opt_ptr(weight, kw), *bp = opt_ptr(bias, kb);
  check_rc(grm_hip_group_norm_fwd(xr.data_ptr(), wp, bp, gr.defined() ? gr.data_ptr() : nullptr, out.data_ptr(), n.rows, n.C,
                                  groups, stride_of(xr, 0, n.C), gr.defined() ? stride_of(gr, 0, n.C) : n.C, n.dtype, n.w_dtype,
                                  silu, center, static_cast<float>(eps), stream_of(x)),
           op);
  return out;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> group_norm_backward(const Tensor& grad_out, const Tensor& x, int64_t groups,
                                                               const OptTensor& weight, const OptTensor& bias,
                                                               const OptTensor& gate, bool silu, bool center, double eps) {
  const char* op = "group_norm backward";
  const Norm n = check_norm(x, groups, weight, bias, gate, op);
  check_device(grad_out, x, op, "grad_out");
  TORCH_CHECK_VALUE(grad_out.sizes() == x.sizes() && grad_out.scalar_type() == x.scalar_type(), op, ": grad_out must match x");
  c10::OptionalDeviceGuard guard(x.device());
  Tensor xr = packed_channels(x), gr = has(gate) ? packed_channels(*gate) : Tensor(), go = grad_out.contiguous(), kw, kb;
  Tensor dx = at::empty({n.rows, n.C}, x.options());
  Tensor dw = has(weight) ? at::empty({n.C}, weight->options()) : Tensor(), db = has(bias) ? at::empty({n.C}, bias->options()) : Tensor();
  Tensor dg = has(gate) ? at::empty({n.rows, n.C}, x.options()) : Tensor();
  const void *wp = opt_ptr(weight, kw), *bp = opt_ptr(bias, kb);
  const int64_t wsb = grm_hip_group_norm_bwd_workspace(n.rows, n.C, groups);
  Tensor ws = bytes(wsb, x);
  check_rc(grm_hip_group_norm_bwd(xr.data_ptr(), wp, bp, gr.defined() ? gr.data_ptr() : nullptr, go.data_ptr(), dx.data_ptr(),
                                  dw.defined() ? dw.data_ptr() : nullptr, db.defined() ? db.data_ptr() : nullptr,
                                  dg.defined() ? dg.data_ptr() : nullptr, ws.data_ptr(), wsb, n.rows, n.C, groups,
                                  stride_of(xr, 0, n.C), gr.defined() ? stride_of(gr, 0, n.C) : n.C, n.dtype, n.w_dtype, silu,
                                  center, static_cast<float>(eps), stream_of(x)),
           op);
  auto given = [&](const Tensor& t) { return t.defined() ? t : at::empty({0}, x.options()); };
  return {dx, given(dw), given(db), given(dg)};
}

}  // namespace
}  // namespace grm_delta

TORCH_LIBRARY_FRAGMENT(grm_cuda, m) {
  m.def("delta_scan_forward(Tensor keys, Tensor values, Tensor queries, Tensor strengths, Tensor? log_decays, Tensor? memory, Tensor? lengths, bool save) -> (Tensor hidden, Tensor memory_out, Tensor states, Tensor miss)");
  m.def("delta_scan_backward(Tensor? grad_hidden, Tensor? grad_memory_out, Tensor keys, Tensor values, Tensor queries, Tensor strengths, Tensor? log_decays, Tensor? lengths, Tensor states, Tensor miss) -> (Tensor grad_keys, Tensor grad_values, Tensor grad_queries, Tensor grad_strengths, Tensor grad_log_decays, Tensor grad_memory)");
  m.def("group_norm_forward(Tensor x, int groups, Tensor? weight, Tensor? bias, Tensor? gate, bool silu, bool center, float eps) -> Tensor");
  m.def("group_norm_backward(Tensor grad_out, Tensor x, int groups, Tensor? weight, Tensor? bias, Tensor? gate, bool silu, bool center, float eps) -> (Tensor grad_x, Tensor grad_weight, Tensor grad_bias, Tensor grad_gate)");
  m.def("delta_step(Tensor keys, Tensor values, Tensor queries, Tensor strengths, Tensor? log_decays, Tensor memory) -> (Tensor hidden, Tensor memory_out)");
  m.def("delta_step_out(Tensor keys, Tensor values, Tensor queries, Tensor strengths, Tensor? log_decays, Tensor memory, Tensor(a!) memory_out) -> Tensor");
}

TORCH_LIBRARY_IMPL(grm_cuda, CUDA, m) {
  m.impl("delta_scan_forward", grm_delta::delta_scan_forward);
  m.impl("delta_scan_backward", grm_delta::delta_scan_backward);
  m.impl("group_norm_forward", grm_delta::group_norm_forward);
  m.impl("group_norm_backward", grm_delta::group_norm_backward);
  m.impl("delta_step", grm_delta::delta_step);
  m.impl("delta_step_out", grm_delta::delta_step_out);
}
