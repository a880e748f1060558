// Group norm of rows (tokens) with their channels last, its activation or activated gate, and the gradients.
//   n = (x - mean) / sqrt(var + eps) over each group of a row (without centre: x / sqrt(mean x^2 + eps))
//   y = n w + b;  out = y act(gate), without a gate act(y)
// Bound by the rows' bytes.  LG lanes hold a group in registers (EPL channels each), so that a row is read once; mean
// (in two steps) and variance are sums over registers, float32.  A thread keeps its channels over all rows that its workgroup
// walks: weights are loaded once, and their gradients are summed in registers, then over the workgroup in LDS, then over the
// workgroups by a second launch, always in the same order.  16384 bf16 rows of 16 groups of 128 with a gate: 37 us
// (201 MB, 5.4 TB/s); gradients 61 (336 MB, 5.5 TB/s) and 4.6 for the sums.
#include "grm_hip.h"
#include "grm_hip_common.h"

namespace grmhip {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxBlocks = 2048;     // forward: eight workgroups a CU
constexpr int kMaxBwdBlocks = 1024;  // each leaves a row of partial sums
constexpr int kMaxWidth = 4096;      // 64 lanes of 64 channels

struct NormArgs {
  const void *x, *weight, *bias, *gate, *grad;  // weight, bias, gate may be null
  void *out, *dx, *dgate;
  float* part;            // [2, blocks, C]: sums for the weights and the biases of a workgroup
  int64_t rows, xs, gs;   // elements between rows of x and of gate
  int C, groups, width, per_block, row_slots;  // groups of a workgroup, rows it takes at a time
  int w_f32, silu, center;
  float eps;
};

__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }
// z / (1 + e^-z): of minus infinity a NaN, as PyTorch's.
__device__ __forceinline__ float silu(float z) { return z * sigmoid(z); }

template <int LG>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int o = LG / 2; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// Channel of a lane's j-th register: units of eight, or single channels where rows are not whole 16-byte units.
template <int LG, bool VEC>
__device__ __forceinline__ int channel(int l, int j) {
  return VEC ? (j >> 3) * (8 * LG) + 8 * l + (j & 7) : j * LG + l;
}

template <class E, int LG, int EPL, bool VEC>
__device__ __forceinline__ void load_group(const typename ET<E>::raw* p, int width, int l, bool ok, float (&v)[EPL]) {
  if constexpr (VEC) {
#pragma unroll
    for (int u = 0; u < EPL / 8; ++u) {
      const int c = channel<LG, true>(l, 8 * u);
      const U8<E> e = load_u8<E>(p, c, width, ok, true);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[8 * u + i] = ET<E>::to_f(e.e[i]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const int c = channel<LG, false>(l, j);
      v[j] = ok && c < width ? ET<E>::to_f(p[c]) : 0.f;
    }
  }
}
template <class E, int LG, int EPL, bool VEC>
__device__ __forceinline__ void store_group(typename ET<E>::raw* p, int width, int l, const float (&v)[EPL]) {
  if constexpr (VEC) {
#pragma unroll
    for (int u = 0; u < EPL / 8; ++u) {
      const int c = channel<LG, true>(l, 8 * u);
      if (c < width) {
        store4_raw<E>(p + c, f32x4{v[8 * u], v[8 * u + 1], v[8 * u + 2], v[8 * u + 3]});
        store4_raw<E>(p + c + 4, f32x4{v[8 * u + 4], v[8 * u + 5], v[8 * u + 6], v[8 * u + 7]});
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const int c = channel<LG, false>(l, j);
      if (c < width) p[c] = ET<E>::from_f(v[j]);
    }
  }
}
// A weight or bias of this lane's channels, `none` where there is none.
template <class E, int LG, int EPL, bool VEC>
__device__ __forceinline__ void load_param(const NormArgs& a, const void* p, int at, int l, bool ok, float none, float (&v)[EPL]) {
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int c = channel<LG, VEC>(l, j);
    v[j] = none;
    if (p != nullptr && ok && c < a.width)
      v[j] = a.w_f32 ? static_cast<const float*>(p)[at + c] : ET<E>::to_f(static_cast<const typename ET<E>::raw*>(p)[at + c]);
  }
}

// n in the place of x; returns 1 / sqrt(var + eps).
template <int LG, int EPL, bool VEC>
__device__ __forceinline__ float normalise(const NormArgs& a, int l, float (&x)[EPL]) {
  const float inv = 1.f / static_cast<float>(a.width);
  if (a.center) {
    // Twice: the first mean is off by a few steps of the values, the second takes out what that left in every difference.  Of
    // equal values nothing is left: the first differences are a few steps of x each, whose sums are exact.
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < EPL; ++j) s += x[j];
      const float mean = group_sum<LG>(s) / static_cast<float>(a.width);
#pragma unroll
      for (int j = 0; j < EPL; ++j) x[j] = channel<LG, VEC>(l, j) < a.width ? x[j] - mean : 0.f;
    }
  }
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < EPL; ++j) s = fmaf(x[j], x[j], s);
  const float r = 1.f / sqrtf(fmaf(group_sum<LG>(s), inv, a.eps));
#pragma unroll
  for (int j = 0; j < EPL; ++j) x[j] *= r;
  return r;
}

// Where a thread stands: its group's lanes, its group and the first row of its slot.
template <int LG>
struct Place {
  int l, slot, sub, group;
  bool ok;
  int64_t row, step;
  __device__ __forceinline__ explicit Place(const NormArgs& a) {
    l = static_cast<int>(threadIdx.x) % LG;
    slot = static_cast<int>(threadIdx.x) / LG;
    sub = slot / a.per_block;
    group = static_cast<int>(blockIdx.y) * a.per_block + slot % a.per_block;
    ok = sub < a.row_slots && group < a.groups;
    row = static_cast<int64_t>(blockIdx.x) * a.row_slots + sub;
    step = static_cast<int64_t>(gridDim.x) * a.row_slots;
  }
};

template <class E, int LG, int EPL, bool VEC>
__global__ __launch_bounds__(kThreads) void group_norm_kernel(NormArgs a) {
  using raw = typename ET<E>::raw;
  const Place<LG> at(a);
  if (!at.ok) return;  // (whole groups of lanes)
  const int c0 = at.group * a.width;
  float w[EPL], b[EPL];
  load_param<E, LG, EPL, VEC>(a, a.weight, c0, at.l, true, 1.f, w);
  load_param<E, LG, EPL, VEC>(a, a.bias, c0, at.l, true, 0.f, b);
  for (int64_t row = at.row; row < a.rows; row += at.step) {
    float x[EPL], z[EPL];
    load_group<E, LG, EPL, VEC>(static_cast<const raw*>(a.x) + row * a.xs + c0, a.width, at.l, true, x);
    if (a.gate != nullptr) load_group<E, LG, EPL, VEC>(static_cast<const raw*>(a.gate) + row * a.gs + c0, a.width, at.l, true, z);
    normalise<LG, EPL, VEC>(a, at.l, x);
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const float y = fmaf(x[j], w[j], b[j]);
      x[j] = a.gate != nullptr ? y * (a.silu ? silu(z[j]) : z[j]) : a.silu ? silu(y) : y;
    }
    store_group<E, LG, EPL, VEC>(static_cast<raw*>(a.out) + row * a.C + c0, a.width, at.l, x);
  }
}

// dy = dout act(gate), dgate = dout y act'(gate) (without a gate dy = dout act'(y));
// dn = dy w, dx = r (dn - n mean(dn n) - mean(dn)), the last mean where centred; dw = sum dy n, db = sum dy.
template <class E, int LG, int EPL, bool VEC>
__global__ __launch_bounds__(kThreads) void group_norm_bwd_kernel(NormArgs a) {
  using raw = typename ET<E>::raw;
  extern __shared__ float sums[];  // [slots][width]
  const Place<LG> at(a);
  const int c0 = at.group * a.width;
  float w[EPL], b[EPL], dw[EPL], db[EPL];
  load_param<E, LG, EPL, VEC>(a, a.weight, c0, at.l, at.ok, 1.f, w);
  load_param<E, LG, EPL, VEC>(a, a.bias, c0, at.l, at.ok, 0.f, b);
#pragma unroll
  for (int j = 0; j < EPL; ++j) dw[j] = db[j] = 0.f;
  const float inv = 1.f / static_cast<float>(a.width);
  for (int64_t row = at.row; at.ok && row < a.rows; row += at.step) {
    float x[EPL], z[EPL], d[EPL];
    load_group<E, LG, EPL, VEC>(static_cast<const raw*>(a.x) + row * a.xs + c0, a.width, at.l, true, x);
    load_group<E, LG, EPL, VEC>(static_cast<const raw*>(a.grad) + row * a.C + c0, a.width, at.l, true, d);
    if (a.gate != nullptr) load_group<E, LG, EPL, VEC>(static_cast<const raw*>(a.gate) + row * a.gs + c0, a.width, at.l, true, z);
    const float r = normalise<LG, EPL, VEC>(a, at.l, x);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const float y = fmaf(x[j], w[j], b[j]), u = a.gate != nullptr ? z[j] : y;
      float act = u, slope = 1.f;
      if (a.silu) {
        const float sg = sigmoid(u);
        act = u * sg;
        slope = sg * fmaf(u, 1.f - sg, 1.f);
      }
      float dy;
      if (a.gate != nullptr) {
        dy = d[j] * act;
        z[j] = d[j] * y * slope;
      } else {
        dy = d[j] * slope;
      }
      dw[j] = fmaf(dy, x[j], dw[j]);
      db[j] += dy;
      d[j] = dy * w[j];
      s1 += d[j];
      s2 = fmaf(d[j], x[j], s2);
    }
    s2 = group_sum<LG>(s2) * inv;
    s1 = a.center ? group_sum<LG>(s1) * inv : 0.f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) d[j] = r * (d[j] - fmaf(x[j], s2, s1));
    store_group<E, LG, EPL, VEC>(static_cast<raw*>(a.dx) + row * a.C + c0, a.width, at.l, d);
    if (a.gate != nullptr) store_group<E, LG, EPL, VEC>(static_cast<raw*>(a.dgate) + row * a.C + c0, a.width, at.l, z);
  }
  // Over the slots that hold the same group, in their order.
  const int first = static_cast<int>(blockIdx.y) * a.per_block;
  const int cols = (a.groups - first < a.per_block ? a.groups - first : a.per_block) * a.width, slab = a.per_block * a.width;
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
    if (at.ok) {
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        const int c = channel<LG, VEC>(at.l, j);
        if (c < a.width) sums[at.slot * a.width + c] = which ? db[j] : dw[j];
      }
    }
    __syncthreads();
    float* to = a.part + (static_cast<int64_t>(which) * gridDim.x + blockIdx.x) * a.C + first * a.width;
    for (int c = threadIdx.x; c < cols; c += kThreads) {
      float s = 0.f;
      for (int i = 0; i < a.row_slots; ++i) s += sums[i * slab + c];
      to[c] = s;
    }
  }
}

// The workgroups' sums: 32 channels a workgroup, 32 threads a channel (of 1024 rows of sums in 2048 channels 12 us with eight).
constexpr int kSumThreads = 1024;
template <class W>
__global__ __launch_bounds__(kSumThreads) void group_norm_sum_kernel(const float* part, void* dw, void* db, int C, int blocks) {
  __shared__ float s[32][33];
  const int l = static_cast<int>(threadIdx.x) % 32, k = static_cast<int>(threadIdx.x) / 32, c = static_cast<int>(blockIdx.x) * 32 + l;
  const float* p = part + static_cast<int64_t>(blockIdx.y) * blocks * C;
  float v = 0.f;
  if (c < C) {
#pragma unroll 4
    for (int i = k; i < blocks; i += 32) v += p[static_cast<int64_t>(i) * C + c];
  }
  s[k][l] = v;
  __syncthreads();
  // A half wave adds up a channel's 32 sums.
  float t = s[l][k];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor(t, o);
  const int to_c = static_cast<int>(blockIdx.x) * 32 + k;
  void* to = blockIdx.y ? db : dw;
  if (l == 0 && to_c < C && to != nullptr) static_cast<typename ET<W>::raw*>(to)[to_c] = ET<W>::from_f(t);
}

struct Form {
  int lg, epl, per_block, row_slots;
  int64_t group_blocks, row_blocks;
};
Form form_of(int64_t rows, int64_t groups, int64_t width, int most) {
  Form f{};
  f.lg = 1;
  while (f.lg < 64 && f.lg * 8 < width) f.lg *= 2;
  f.epl = 8;
  while (f.lg * f.epl < width) f.epl *= 2;
  const int slots = kThreads / f.lg;
  f.per_block = static_cast<int>(groups < slots ? groups : slots);
  f.row_slots = slots / f.per_block;
  f.group_blocks = (groups + f.per_block - 1) / f.per_block;
  const int64_t need = (rows + f.row_slots - 1) / f.row_slots, room = most / f.group_blocks;
  f.row_blocks = need < room ? need : (room < 1 ? 1 : room);
  if (f.row_blocks < 1) f.row_blocks = 1;
  return f;
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check(int64_t rows, int64_t channels, int64_t groups, int64_t xs, int64_t gs, const void* x, const void* gate, int dtype,
          int weight_dtype, float eps, const char* what) {
  if (rows < 0 || channels < 1 || groups < 1 || channels % groups != 0) {
    set_error("%s: rows must be >= 0 and channels a multiple of groups", what);
    return GRM_HIP_EINVAL;
  }
  if (dtype < 0 || dtype > 2 || (weight_dtype != dtype && weight_dtype != GRM_HIP_F32)) {
    set_error("%s: rows must be float32, float16 or bfloat16, weights the same or float32", what);
    return GRM_HIP_EUNSUPPORTED;
  }
  if (channels / groups > kMaxWidth || channels > (int64_t{1} << 21)) {
    set_error("%s: at most %d channels a group and 2^21 in all", what, kMaxWidth);
    return GRM_HIP_EUNSUPPORTED;
  }
  if (!(eps >= 0.f) || eps > 3.4e38f) {
    set_error("%s: eps must be a number >= 0", what);
    return GRM_HIP_EINVAL;
  }
  if (rows > 0 && x == nullptr) {
    set_error("%s: x is required", what);
    return GRM_HIP_EINVAL;
  }
  // (No product of a row's number and its stride passes 63 bits.)
  const int64_t most = int64_t{1} << 31;
  if (rows > most || (rows > 1 && (xs < channels || xs > most || (gate != nullptr && (gs < channels || gs > most))))) {
    set_error("%s: at most 2^31 rows, strides from the channels' number to 2^31", what);
    return GRM_HIP_EUNSUPPORTED;
  }
  return GRM_HIP_OK;
}

// f(E, LG, EPL, VEC) with one of the compiled forms.
template <class F>
void with_form(int dtype, const Form& fm, bool vec, F f) {
  auto by_vec = [&](auto e, auto lg, auto epl) {
    if (vec) f(e, lg, epl, std::true_type{});
    else f(e, lg, epl, std::false_type{});
  };
  auto by_width = [&](auto e) {
    auto lanes = [&](auto lg) { by_vec(e, lg, std::integral_constant<int, 8>{}); };
    auto deep = [&](auto epl) { by_vec(e, std::integral_constant<int, 64>{}, epl); };
    if (fm.epl == 16) deep(std::integral_constant<int, 16>{});
    else if (fm.epl == 32) deep(std::integral_constant<int, 32>{});
    else if (fm.epl == 64) deep(std::integral_constant<int, 64>{});
    else if (fm.lg == 1) lanes(std::integral_constant<int, 1>{});
    else if (fm.lg == 2) lanes(std::integral_constant<int, 2>{});
    else if (fm.lg == 4) lanes(std::integral_constant<int, 4>{});
    else if (fm.lg == 8) lanes(std::integral_constant<int, 8>{});
    else if (fm.lg == 16) lanes(std::integral_constant<int, 16>{});
    else if (fm.lg == 32) lanes(std::integral_constant<int, 32>{});
    else lanes(std::integral_constant<int, 64>{});
  };
  if (dtype == GRM_HIP_BF16) by_width(BF16{});
  else if (dtype == GRM_HIP_F16) by_width(F16{});
  else by_width(F32{});
}

void fill(NormArgs& a, const Form& f, int64_t rows, int64_t channels, int64_t groups) {
  a.rows = rows;
  a.C = static_cast<int>(channels);
  a.groups = static_cast<int>(groups);
  a.width = static_cast<int>(channels / groups);
  a.per_block = f.per_block;
  a.row_slots = f.row_slots;
}

}  // namespace
}  // namespace grmhip

using namespace grmhip;

extern "C" int grm_hip_group_norm_fwd(const void* x, const void* weight, const void* bias, const void* gate, void* out,
                                      int64_t rows, int64_t channels, int64_t groups, int64_t x_stride, int64_t gate_stride,
                                      int dtype, int weight_dtype, int silu, int center, float eps, void* stream) {
  const char* what = "group_norm";
  if (int rc = check(rows, channels, groups, x_stride, gate_stride, x, gate, dtype, weight_dtype, eps, what)) return rc;
  if (rows == 0) return GRM_HIP_OK;
  if (out == nullptr) {
    set_error("%s: out is required", what);
    return GRM_HIP_EINVAL;
  }
  NormArgs a{};
  a.x = x; a.weight = weight; a.bias = bias; a.gate = gate; a.out = out;
  a.xs = x_stride; a.gs = gate_stride;
  a.w_f32 = weight_dtype == GRM_HIP_F32; a.silu = silu; a.center = center; a.eps = eps;
  const Form f = form_of(rows, groups, channels / groups, kMaxBlocks);
  fill(a, f, rows, channels, groups);
  const bool vec = a.width % 8 == 0 && aligned(x) && aligned(out) && (rows == 1 || x_stride % 8 == 0) &&
                   (gate == nullptr || (aligned(gate) && (rows == 1 || gate_stride % 8 == 0)));
  with_form(dtype, f, vec, [&](auto e, auto lg, auto epl, auto v) {
    group_norm_kernel<decltype(e), decltype(lg)::value, decltype(epl)::value, decltype(v)::value>
        <<<dim3(static_cast<uint32_t>(f.row_blocks), static_cast<uint32_t>(f.group_blocks)), dim3(kThreads), 0,
           static_cast<hipStream_t>(stream)>>>(a);
  });
  return check_launch(what);
}

extern "C" int64_t grm_hip_group_norm_bwd_workspace(int64_t rows, int64_t channels, int64_t groups) {
  if (rows <= 0 || channels < 1 || groups < 1 || channels % groups != 0 || channels > (int64_t{1} << 21)) return 0;
  return 2 * form_of(rows, groups, channels / groups, kMaxBwdBlocks).row_blocks * channels * 4;
}

extern "C" int grm_hip_group_norm_bwd(const void* x, const void* weight, const void* bias, const void* gate, const void* grad_out,
                                      void* grad_x, void* grad_weight, void* grad_bias, void* grad_gate, void* workspace,
                                      int64_t workspace_bytes, int64_t rows, int64_t channels, int64_t groups, int64_t x_stride,
                                      int64_t gate_stride, int dtype, int weight_dtype, int silu, int center, float eps,
                                      void* stream) {
  const char* what = "group_norm backward";
  if (int rc = check(rows, channels, groups, x_stride, gate_stride, x, gate, dtype, weight_dtype, eps, what)) return rc;
  if (rows > 0 && (grad_out == nullptr || grad_x == nullptr || (gate != nullptr && grad_gate == nullptr) || workspace == nullptr ||
                   !aligned(workspace) || workspace_bytes < grm_hip_group_norm_bwd_workspace(rows, channels, groups))) {
    set_error("%s: the gradients and a 16-byte aligned workspace of enough bytes are required", what);
    return GRM_HIP_EINVAL;
  }
  const hipStream_t hs = static_cast<hipStream_t>(stream);
  NormArgs a{};
  a.x = x; a.weight = weight; a.bias = bias; a.gate = gate; a.grad = grad_out; a.dx = grad_x; a.dgate = grad_gate;
  a.part = static_cast<float*>(workspace);
  a.xs = x_stride; a.gs = gate_stride;
  a.w_f32 = weight_dtype == GRM_HIP_F32; a.silu = silu; a.center = center; a.eps = eps;
  const Form f = form_of(rows, groups, channels / groups, kMaxBwdBlocks);
  fill(a, f, rows, channels, groups);
  if (rows > 0) {
    const bool vec = a.width % 8 == 0 && aligned(x) && aligned(grad_out) && aligned(grad_x) && (rows == 1 || x_stride % 8 == 0) &&
                     (gate == nullptr || (aligned(gate) && aligned(grad_gate) && (rows == 1 || gate_stride % 8 == 0)));
    // (At most 64 KB: 256 / LG slots of at most LG EPL channels.)
    const size_t lds = static_cast<size_t>(kThreads / f.lg) * a.width * 4;
    with_form(dtype, f, vec, [&](auto e, auto lg, auto epl, auto v) {
      group_norm_bwd_kernel<decltype(e), decltype(lg)::value, decltype(epl)::value, decltype(v)::value>
          <<<dim3(static_cast<uint32_t>(f.row_blocks), static_cast<uint32_t>(f.group_blocks)), dim3(kThreads), lds, hs>>>(a);
    });
    if (int rc = check_launch(what)) return rc;
  }
  if (grad_weight == nullptr && grad_bias == nullptr) return GRM_HIP_OK;
  const dim3 grid(static_cast<uint32_t>((channels + 31) / 32), 2);
  const int blocks = rows > 0 ? static_cast<int>(f.row_blocks) : 0;  // of no rows: zeros
  if (weight_dtype == GRM_HIP_F32) group_norm_sum_kernel<F32><<<grid, dim3(kSumThreads), 0, hs>>>(a.part, grad_weight, grad_bias, a.C, blocks);
  else if (weight_dtype == GRM_HIP_F16) group_norm_sum_kernel<F16><<<grid, dim3(kSumThreads), 0, hs>>>(a.part, grad_weight, grad_bias, a.C, blocks);
  else group_norm_sum_kernel<BF16><<<grid, dim3(kSumThreads), 0, hs>>>(a.part, grad_weight, grad_bias, a.C, blocks);
  return check_launch(what);
}
