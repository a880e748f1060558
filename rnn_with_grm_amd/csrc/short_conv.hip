// Short causal depthwise convolution with its state, gfx950: whole sequences, the
// gradients, and single tokens.
//
//   pre_t = bias + sum_w weight[:, w] x_{t - W + 1 + w},  out_t = pre_t or silu(pre_t)
//
// with x_{-W+1 .. -1} the state's rows (zeros without one), W = 2 .. 4.  The state that a
// call leaves is the last W - 1 rows of (state, x) before the sequence's length.
//
// Every element of x is wanted by W outputs of its own channel only, so a thread owns 16 bytes of
// channels (backward four channels, whose sums and windows then fit its registers) and walks a run of
// tokens with the last rows in registers: each row is read from HBM once, the W - 1 rows before a run
// a second time, from L2.  Nothing is kept for the backward pass: it forms pre again from x, as cheap
// as reading it back.  The gradient of the weights is summed in registers over a thread's runs, over a
// workgroup's four waves in LDS, and over the workgroups by a second kernel in a fixed order (no
// atomics: the same sums on every run).  All arithmetic is float32, rounded once on output.
//
// HBM bounds the prompts, the launch bounds single tokens: 8 x 2048 tokens x 2304 bf16 channels 36 us
// (151 MB, 4.2 TB/s), with all gradients 104 us (by trace forward 31, backward 64, its weights' sums 4), one
// token of 64 sequences 8 us.
#include <stdint.h>

#include <utility>

#include "f32_tiles.h"
#include "grm_hip.h"
#include "grm_hip_common.h"

namespace grmhip {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxBlocks = 1 << 23;  // thread numbers stay below 2^31

struct ConvArgs {
  const void* x;         // [B, T, C], rows of C, strides below
  const void* weight;    // [C, W]
  const void* bias;      // [C] or null
  const void* state;     // [B, W - 1, C] or null
  const int64_t* lengths;  // [B] or null
  void* out;             // [B, T, C]
  void* state_out;       // [B, W - 1, C]
  const void* dy;        // [B, T, C] or null (zeros)
  const void* dstate_out;  // [B, W - 1, C] or null (zeros)
  void* dx;              // [B, T, C]
  void* dstate;          // [B, W - 1, C] or null
  float* partial;        // [groups][C * (W + 1)]
  int64_t xb, xt;        // elements between sequences and between tokens of x
  int64_t B, T, C;
  int64_t runs;          // runs of a sequence
  int64_t run;           // tokens of one
  int w_f32;             // weight and bias are float32 whatever x is
  int stream;            // outputs are stored past the caches
};

// V consecutive elements as they lie in memory.
template <class E, int V>
struct RawRow {
  typename ET<E>::raw e[V];
};
template <class E, int V>
__device__ __forceinline__ void widen(const RawRow<E, V>& r, float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = ET<E>::to_f(r.e[i]);
}
// The access that a row is read or written in: 16 or 8 bytes, or one element.
template <class E, int V>
using Access = std::conditional_t<V * sizeof(typename ET<E>::raw) == 16, uint32_t __attribute__((ext_vector_type(4))),
                                  std::conditional_t<V * sizeof(typename ET<E>::raw) == 8, uint32_t __attribute__((ext_vector_type(2))),
                                                     typename ET<E>::raw>>;
template <class E, int V>
__device__ __forceinline__ RawRow<E, V> raw_row(const typename ET<E>::raw* p) {
  return __builtin_bit_cast(RawRow<E, V>, *reinterpret_cast<const Access<E, V>*>(p));
}
// The row at p, or zeros: a load that nothing is done to, so that it is waited for where it is used.
template <class E, int V>
__device__ __forceinline__ RawRow<E, V> raw_row_if(const typename ET<E>::raw* p, bool in) {
  Access<E, V> u = {};
  if (in) u = *reinterpret_cast<const Access<E, V>*>(p);
  return __builtin_bit_cast(RawRow<E, V>, u);
}
template <class E, int V>
__device__ __forceinline__ void ld_row(const typename ET<E>::raw* p, float (&v)[V]) {
  widen<E, V>(raw_row<E, V>(p), v);
}

// `stream`: past the caches (see streams()).
template <class E, int V>
__device__ __forceinline__ void st_row(typename ET<E>::raw* p, const float (&v)[V], bool stream = false) {
  RawRow<E, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.e[i] = ET<E>::from_f(v[i]);
  const Access<E, V> q = __builtin_bit_cast(Access<E, V>, r);
  if (stream) __builtin_nontemporal_store(q, reinterpret_cast<Access<E, V>*>(p));
  else *reinterpret_cast<Access<E, V>*>(p) = q;
}

// f(0), ..., f(U - 1) with constants, so that a window's slots are registers by name.
template <int U, class F, int... I>
__device__ __forceinline__ void unrolled(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int U, class F>
__device__ __forceinline__ void unrolled(F f) { unrolled<U>(f, std::make_integer_sequence<int, U>{}); }

// Steps taken at once: a multiple of the window, so that its rows need not move.
template <int W> constexpr int kSteps = W == 3 ? 3 : 4;

template <int V>
__device__ __forceinline__ void zero(float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = 0.f;
}

__device__ __forceinline__ float sigmoid_f(float p) { return __builtin_amdgcn_rcpf(1.f + __expf(-p)); }
// silu(p) or p, in float32.  Kept whole: fused with the rounding to float16 in one form and not in another, the same
// row would differ by a step of float16 between a prompt's aligned and unaligned rows and its single tokens.
template <bool SILU>
__device__ __forceinline__ float activate(float p) {
  if constexpr (!SILU) return p;
  float y = p * sigmoid_f(p);
  asm("" : "+v"(y));
  return y;
}

__device__ __forceinline__ int64_t length_of(const ConvArgs& a, int64_t b) {
  return a.lengths == nullptr ? a.T : max_i64(0, min_i64(a.lengths[b], a.T));
}

// weight[c .. c + V)[0 .. W) and bias of a thread's channels: V W consecutive elements, in 16-byte accesses where
// rows are read so.
template <class D, int V, int W>
__device__ __forceinline__ void ld_weight_as(const ConvArgs& a, int64_t c, float (&w)[W][V], float (&b)[V]) {
  using raw = typename ET<D>::raw;
  const raw *wp = static_cast<const raw*>(a.weight) + c * W, *bp = static_cast<const raw*>(a.bias) + c;
  constexpr int Q = V == 1 ? 1 : V * static_cast<int>(sizeof(raw)) < 16 ? V : 16 / static_cast<int>(sizeof(raw));  // of an access
  RawRow<D, Q> r[V * W / Q], rb[V / Q];
#pragma unroll
  for (int i = 0; i < V * W / Q; ++i) r[i] = raw_row<D, Q>(wp + i * Q);
#pragma unroll
  for (int i = 0; i < V / Q; ++i) rb[i] = raw_row_if<D, Q>(bp + i * Q, a.bias != nullptr);
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][i] = ET<D>::to_f(r[(i * W + j) / Q].e[(i * W + j) % Q]);
    b[i] = ET<D>::to_f(rb[i / Q].e[i % Q]);
  }
}
template <class E, int V, int W>
__device__ __forceinline__ void ld_weight(const ConvArgs& a, int64_t c, float (&w)[W][V], float (&b)[V]) {
  if (a.w_f32) ld_weight_as<F32, V, W>(a, c, w, b);
  else ld_weight_as<E, V, W>(a, c, w, b);
}

// Row t of a sequence, t >= -(W - 1): the state below 0, zeros from `n` on.
template <class E, int V, int W>
__device__ __forceinline__ void ld_x(const ConvArgs& a, int64_t b, int64_t t, int64_t n, int64_t c, float (&v)[V]) {
  using raw = typename ET<E>::raw;
  if (t >= 0 && t < n) {
    ld_row<E, V>(static_cast<const raw*>(a.x) + b * a.xb + t * a.xt + c, v);
  } else if (t < 0 && a.state != nullptr) {
    ld_row<E, V>(static_cast<const raw*>(a.state) + (b * (W - 1) + t + W - 1) * a.C + c, v);
  } else {
    zero<V>(v);
  }
}

// Threads 0 .. B * runs * CV walk runs of tokens; B * (W - 1) * CV more copy the state that
// the call leaves.
template <class E, int V, int W, bool SILU>
__global__ __launch_bounds__(kThreads) void conv_fwd_kernel(ConvArgs a) {
  using raw = typename ET<E>::raw;
  const uint32_t cv = static_cast<uint32_t>(a.C / V), runs = static_cast<uint32_t>(a.runs);
  uint32_t id = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t walks = static_cast<uint32_t>(a.B) * runs * cv;
  if (id >= walks) {
    id -= walks;
    const int64_t c = id % cv * V, r = id / cv % (W - 1), b = id / cv / (W - 1);
    if (b >= a.B) return;
    const int64_t n = length_of(a, b);
    float v[V];
    ld_x<E, V, W>(a, b, n - (W - 1) + r, n, c, v);
    st_row<E, V>(static_cast<raw*>(a.state_out) + (b * (W - 1) + r) * a.C + c, v);
    return;
  }
  const int64_t c = id % cv * V, run = id / cv % runs, b = id / cv / runs;
  const int64_t n = length_of(a, b), t0 = run * a.run, t1 = min_i64(t0 + a.run, a.T);
  // The window's slot of a token is its number in the run, modulo W.
  float w[W][V], bias[V], win[W][V];
  ld_weight<E, V, W>(a, c, w, bias);
#pragma unroll
  for (int j = 1; j < W; ++j) ld_x<E, V, W>(a, b, t0 - W + j, n, c, win[j]);
  const raw* xp = static_cast<const raw*>(a.x) + b * a.xb + c;
  raw* op = static_cast<raw*>(a.out) + b * a.T * a.C + c;
  constexpr int U = kSteps<W>;
  for (int64_t tb = t0; tb < t1; tb += U) {
    RawRow<E, V> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = raw_row_if<E, V>(xp + (tb + u) * a.xt, tb + u < n);
    unrolled<U>([&](auto uc) {
      constexpr int u = decltype(uc)::value;
      widen<E, V>(x[u], win[u % W]);
      float y[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float p = bias[i];
#pragma unroll
        for (int j = 0; j < W; ++j) p = fmaf(w[j][i], win[(u + 1 + j) % W][i], p);
        y[i] = activate<SILU>(p);
        if (tb + u >= n) y[i] = 0.f;
      }
      if (tb + u < t1) st_row<E, V>(op + (tb + u) * a.C, y, a.stream != 0);
    });
  }
}

// Lane = channels, wave = every fourth run from its workgroup's part of all B * runs.
template <class E, int V, int W, bool SILU>
__global__ __launch_bounds__(kThreads) void conv_bwd_kernel(ConvArgs a) {
  using raw = typename ET<E>::raw;
  __shared__ float sums[3][64 * V * (W + 1)];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (static_cast<int64_t>(blockIdx.x) * 64 + lane) * V;
  const bool in = c < a.C;
  float dw[W][V], db[V];
  zero<V>(db);
#pragma unroll
  for (int j = 0; j < W; ++j) zero<V>(dw[j]);
  if (in) {
    float w[W][V], bias[V];
    ld_weight<E, V, W>(a, c, w, bias);
    const int64_t total = a.B * a.runs;
    for (int64_t k = static_cast<int64_t>(blockIdx.y) * 4 + wave; k < total; k += static_cast<int64_t>(gridDim.y) * 4) {
      const int64_t b = k / a.runs, run = k % a.runs;
      const int64_t n = length_of(a, b), t0 = run * a.run, t1 = min_i64(t0 + a.run, a.T);
      const raw* dyp = static_cast<const raw*>(a.dy) + b * a.T * a.C + c;
      float win[W][V], g[W][V];
#pragma unroll
      for (int j = 1; j < W; ++j) {
        ld_x<E, V, W>(a, b, t0 - W + j, n, c, win[j]);
        zero<V>(g[j]);
      }
      // Step t: x_t and g_t = dy_t act'(pre_t) take their slots, and row s = t - W + 1 of dx (below 0: of
      // dstate, by the first run only) has all of its terms.  The rows of U steps are in flight together.
      const int64_t first = run == 0 ? -(W - 1) : t0, end = t1 + W - 1;
      const raw* xp = static_cast<const raw*>(a.x) + b * a.xb + c;
      constexpr int U = kSteps<W>;
      for (int64_t tb = t0; tb < end; tb += U) {
        RawRow<E, V> xr[U], yr[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const bool in = tb + u < n;
          xr[u] = raw_row_if<E, V>(xp + (tb + u) * a.xt, in);
          yr[u] = raw_row_if<E, V>(dyp + (tb + u) * a.C, in && a.dy != nullptr);
        }
        auto steps = [&](auto inner) {  // inner: all of these tokens are the run's own and away from both ends
          constexpr bool INNER = decltype(inner)::value;
          unrolled<U>([&](auto uc) {
            constexpr int u = decltype(uc)::value;
            const int64_t t = tb + u, s = t - W + 1;
            if (!INNER && t >= end) return;
            float dx[V];
            zero<V>(dx);
            const int64_t at = s - (n - (W - 1));  // row of the state left behind that is x_s
            if (!INNER && a.dstate_out != nullptr && at >= 0 && at < W - 1)
              ld_row<E, V>(static_cast<const raw*>(a.dstate_out) + (b * (W - 1) + at) * a.C + c, dx);
            float (&xv)[V] = win[u % W], (&gv)[V] = g[u % W];
            widen<E, V>(xr[u], xv);
            widen<E, V>(yr[u], gv);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              if constexpr (SILU) {
                float p = bias[i];
#pragma unroll
                for (int j = 0; j < W; ++j) p = fmaf(w[j][i], win[(u + 1 + j) % W][i], p);
                const float sg = sigmoid_f(p);
                gv[i] *= sg * fmaf(p, 1.f - sg, 1.f);
              }
              if (!INNER && t >= n) gv[i] = 0.f;
              // The rows past the run are another one's, those past the length nobody's.  They are kept out of the
              // products too: an infinity that the window still holds would make a NaN of a gradient of zero.
              const bool own = INNER || (t < t1 && t < n);
              db[i] += own ? gv[i] : 0.f;
#pragma unroll
              for (int j = 0; j < W; ++j) {
                dw[j][i] = own ? fmaf(gv[i], win[(u + 1 + j) % W][i], dw[j][i]) : dw[j][i];
                dx[i] = fmaf(w[j][i], g[(u + W - j) % W][i], dx[i]);
              }
              if (!INNER && s >= n) dx[i] = 0.f;
            }
            if (!INNER && s < first) return;
            if (INNER || s >= 0) st_row<E, V>(static_cast<raw*>(a.dx) + (b * a.T + s) * a.C + c, dx, a.stream != 0);
            else if (a.dstate != nullptr) st_row<E, V>(static_cast<raw*>(a.dstate) + (b * (W - 1) + s + W - 1) * a.C + c, dx);
          });
        };
        if (tb - W + 1 >= (first > 0 ? first : 0) && tb + U <= (n < t1 ? n : t1)) steps(std::true_type{});
        else steps(std::false_type{});
      }
    }
  }
  // Waves 1 to 3 hand their sums to wave 0.
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int j = 0; j <= W; ++j) {
      if (wave > 0) sums[wave - 1][(lane * V + i) * (W + 1) + j] = j < W ? dw[j < W ? j : 0][i] : db[i];
    }
  }
  __syncthreads();
  if (wave == 0 && in) {
    float* p = a.partial + (static_cast<int64_t>(blockIdx.y) * a.C + c) * (W + 1);
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int j = 0; j <= W; ++j) {
        const int at = (lane * V + i) * (W + 1) + j;
        p[i * (W + 1) + j] = (j < W ? dw[j < W ? j : 0][i] : db[i]) + sums[0][at] + sums[1][at] + sums[2][at];
      }
    }
  }
}

// Sums of the workgroups' parts: 64 elements per workgroup, eight waves an eighth of the parts each.
template <class E, int W>
__global__ __launch_bounds__(512) void conv_weight_kernel(const float* partial, void* dweight, void* dbias, int64_t C,
                                                          int parts, int w_f32) {
  __shared__ float sums[7][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 64 + lane, total = C * (W + 1);
  float s = 0.f;
  if (e < total) {
#pragma unroll 4
    for (int p = wave; p < parts; p += 8) s += partial[static_cast<int64_t>(p) * total + e];
  }
  if (wave > 0) sums[wave - 1][lane] = s;
  __syncthreads();
  if (wave > 0 || e >= total) return;
#pragma unroll
  for (int i = 0; i < 7; ++i) s += sums[i][lane];
  const int64_t c = e / (W + 1);
  const int j = static_cast<int>(e % (W + 1));
  if (j < W) st_state<E>(dweight, c * W + j, w_f32 != 0, s);
  else if (dbias != nullptr) st_state<E>(dbias, c, w_f32 != 0, s);
}

// One token: every thread reads its channels of the state before it writes them, so the state
// may be updated in place.
template <class E, int V, int W, bool SILU>
__global__ __launch_bounds__(kThreads) void conv_step_kernel(ConvArgs a) {
  using raw = typename ET<E>::raw;
  const uint32_t cv = static_cast<uint32_t>(a.C / V), id = blockIdx.x * kThreads + threadIdx.x;
  if (id >= static_cast<uint32_t>(a.B) * cv) return;
  const int64_t c = id % cv * V, b = id / cv;
  float w[W][V], bias[V], win[W][V], y[V];
#pragma unroll
  for (int j = 0; j < W; ++j) ld_x<E, V, W>(a, b, j - (W - 1), 1, c, win[j]);
  ld_weight<E, V, W>(a, c, w, bias);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float p = bias[i];
#pragma unroll
    for (int j = 0; j < W; ++j) p = fmaf(w[j][i], win[j][i], p);
    y[i] = activate<SILU>(p);
  }
  st_row<E, V>(static_cast<raw*>(a.out) + b * a.C + c, y);
#pragma unroll
  for (int j = 1; j < W; ++j) st_row<E, V>(static_cast<raw*>(a.state_out) + (b * (W - 1) + j - 1) * a.C + c, win[j]);
}

// ---------------------------------------------------------------------------

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// More elements than any memory has.  (Below, no product of sizes passes 63 bits.)
bool too_many(int64_t B, int64_t T, int64_t C) {
  const int64_t most = int64_t{1} << 50;
  return B > most || T > most || C > most || (B > 0 && T + 4 > most / B / C);
}

int check_conv(const ConvArgs& a, int64_t width, int dtype, int w_dtype, const char* what) {
  if (a.B < 0 || a.T < 0 || a.C < 1) {
    set_error("%s: batch and seq_len must be >= 0 and channels >= 1", what);
    return GRM_HIP_EINVAL;
  }
  if (width < 2 || width > 4) {
    set_error("%s: width must be 2, 3 or 4, got %lld", what, static_cast<long long>(width));
    return GRM_HIP_EUNSUPPORTED;
  }
  if (too_many(a.B, a.T, a.C)) {
    set_error("%s: too many elements", what);
    return GRM_HIP_EUNSUPPORTED;
  }
  if (dtype < 0 || dtype > 2 || (w_dtype != dtype && w_dtype != GRM_HIP_F32)) {
    set_error("%s: x must be float32, float16 or bfloat16, and weight x's type or float32", what);
    return GRM_HIP_EUNSUPPORTED;
  }
  return GRM_HIP_OK;
}

// Whole 16-byte accesses where every row allows them: 2304 channels of 8 x 2048 bf16 tokens take 30 us so, and
// 49 us element by element.
bool whole_rows(const ConvArgs& a, int dtype) {
  const int64_t v = dtype == GRM_HIP_F32 ? 4 : 8;
  return a.C % v == 0 && a.xb % v == 0 && a.xt % v == 0 && aligned(a.x) && aligned(a.state) && aligned(a.out) &&
         aligned(a.state_out) && aligned(a.weight) && aligned(a.bias) && aligned(a.dy) && aligned(a.dstate_out) && aligned(a.dx) && aligned(a.dstate);
}

// f(E, V, W, SILU): one of the compiled forms, V = 1 or (vec) 16 bytes of elements, at most MOST of them.
template <int MOST, class F>
void with_form(int dtype, bool vec, int64_t width, bool silu, F f) {
  auto by_silu = [&](auto e, auto v, auto w) {
    if (silu) f(e, v, w, std::true_type{});
    else f(e, v, w, std::false_type{});
  };
  auto by_width = [&](auto e, auto v) {
    if (width == 2) by_silu(e, v, std::integral_constant<int, 2>{});
    else if (width == 3) by_silu(e, v, std::integral_constant<int, 3>{});
    else by_silu(e, v, std::integral_constant<int, 4>{});
  };
  auto by_vec = [&](auto e) {
    constexpr int V = sizeof(typename ET<decltype(e)>::raw) == 4 || MOST == 4 ? 4 : 8;
    if (vec) by_width(e, std::integral_constant<int, V>{});
    else by_width(e, std::integral_constant<int, 1>{});
  };
  if (dtype == GRM_HIP_F32) by_vec(F32{});
  else if (dtype == GRM_HIP_F16) by_vec(F16{});
  else by_vec(BF16{});
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Rows of more than the eight 4 MB L2 caches hold are stored past them: what would be written back at the kernel's end
// leaves during it (8 x 2048 tokens of 2304 bf16 channels 38.5 -> 31.7 us; 4 MB outputs the same either way).
int streams(int64_t elements, int dtype) { return elements * (dtype == GRM_HIP_F32 ? 4 : 2) > (int64_t{32} << 20); }

// The backward's runs: about 3000, one and a half for each of the waves that fit the chip at once (8 x 2048 tokens of
// 2304 bf16 channels, forward and backward: 104 us; 2000 runs: 115, 4000: 109), of 16 tokens at least (three rows of each
// run's 19 or more are formed twice).  A thread has four channels: with eight the backward kernel
// measured 96 us, with four 64.  (Not for the waves a SIMD holds: two in both forms, at 256 and 178 registers.)
int64_t bwd_run(int64_t B, int64_t T, int64_t C, bool vec) {
  const int64_t run = ceil_div(B * T * ceil_div(C, 64 * (vec ? 4 : 1)), 3000);
  return run < 16 ? 16 : run < T ? run : (T > 16 ? T : 16);
}
// Workgroups that share the sums, four runs at a time.
int64_t bwd_parts(int64_t B, int64_t T, int64_t run) {
  const int64_t sets = ceil_div(B * ceil_div(T > 0 ? T : 1, run), 4);
  return sets < 1024 ? sets : 1024;
}

}  // namespace
}  // namespace grmhip

using namespace grmhip;

extern "C" int grm_hip_short_conv_fwd(const void* x, const void* weight, const void* bias, const void* state,
                                      const int64_t* lengths, void* out, void* state_out, int64_t batch,
                                      int64_t seq_len, int64_t channels, int64_t width, int64_t x_batch_stride,
                                      int64_t x_token_stride, int dtype, int weight_dtype, int silu, void* stream) {
  ConvArgs a{};
  a.x = x; a.weight = weight; a.bias = bias; a.state = state; a.lengths = lengths; a.out = out;
  a.state_out = state_out; a.xb = x_batch_stride; a.xt = x_token_stride; a.B = batch; a.T = seq_len; a.C = channels;
  a.w_f32 = weight_dtype == GRM_HIP_F32;
  if (int rc = check_conv(a, width, dtype, weight_dtype, "short_conv")) return rc;
  if (batch == 0) return GRM_HIP_OK;
  if (weight == nullptr || state_out == nullptr || (seq_len > 0 && (x == nullptr || out == nullptr))) {
    set_error("short_conv: x, weight, out and state_out are required");
    return GRM_HIP_EINVAL;
  }
  const int64_t es = dtype == GRM_HIP_F32 ? 4 : 2, st_bytes = batch * (width - 1) * channels * es;
  if (ranges_overlap(state, st_bytes, state_out, st_bytes)) {
    set_error("short_conv: state_out may not overlap state");
    return GRM_HIP_EINVAL;
  }
  const bool vec = whole_rows(a, dtype);
  a.stream = streams(batch * a.T * channels, dtype);
  const int64_t cv = vec ? channels / (dtype == GRM_HIP_F32 ? 4 : 8) : channels;
  // Runs of 16 tokens read 3 rows of 19 twice; where that leaves fewer than four waves a SIMD
  // (2^18 threads), runs of 4 give the CUs more to have in flight.
  a.run = batch * ceil_div(seq_len, 16) * cv >= (1 << 18) ? 16 : 4;
  a.runs = ceil_div(seq_len, a.run);
  const int64_t threads = batch * (a.runs + width - 1) * cv, blocks = ceil_div(threads, kThreads);
  if (blocks > kMaxBlocks) {
    set_error("short_conv: too many elements for one launch");
    return GRM_HIP_EUNSUPPORTED;
  }
  with_form<8>(dtype, vec, width, silu != 0, [&](auto e, auto v, auto w, auto act) {
    conv_fwd_kernel<decltype(e), decltype(v)::value, decltype(w)::value, decltype(act)::value>
        <<<dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0, static_cast<hipStream_t>(stream)>>>(a);
  });
  return check_launch("short_conv");
}

extern "C" int64_t grm_hip_short_conv_bwd_workspace(int64_t batch, int64_t seq_len, int64_t channels, int64_t width,
                                                    int dtype) {
  if (batch <= 0 || seq_len < 0 || channels <= 0 || width < 2 || width > 4 || dtype < 0 || dtype > 2 ||
      too_many(batch, seq_len, channels))
    return 0;
  const int64_t a = bwd_parts(batch, seq_len, bwd_run(batch, seq_len, channels, true)),
                b = bwd_parts(batch, seq_len, bwd_run(batch, seq_len, channels, false));
  return (a > b ? a : b) * channels * (width + 1) * 4;
}

extern "C" int grm_hip_short_conv_bwd(const void* x, const void* weight, const void* bias, const void* state,
                                      const int64_t* lengths, const void* grad_out, const void* grad_state_out,
                                      void* grad_x, void* grad_weight, void* grad_bias, void* grad_state,
                                      void* workspace, int64_t workspace_bytes, int64_t batch, int64_t seq_len,
                                      int64_t channels, int64_t width, int64_t x_batch_stride, int64_t x_token_stride,
                                      int dtype, int weight_dtype, int silu, void* stream) {
  ConvArgs a{};
  a.x = x; a.weight = weight; a.bias = bias; a.state = state; a.lengths = lengths; a.dy = grad_out;
  a.dstate_out = grad_state_out; a.dx = grad_x; a.dstate = grad_state; a.partial = static_cast<float*>(workspace);
  a.xb = x_batch_stride; a.xt = x_token_stride; a.B = batch; a.T = seq_len; a.C = channels;
  a.w_f32 = weight_dtype == GRM_HIP_F32;
  if (int rc = check_conv(a, width, dtype, weight_dtype, "short_conv backward")) return rc;
  if (weight == nullptr || grad_weight == nullptr || (batch > 0 && seq_len > 0 && (x == nullptr || grad_x == nullptr))) {
    set_error("short_conv backward: x, weight, grad_x and grad_weight are required");
    return GRM_HIP_EINVAL;
  }
  if (batch > 0 && (workspace == nullptr ||
                    workspace_bytes < grm_hip_short_conv_bwd_workspace(batch, seq_len, channels, width, dtype))) {
    set_error("short_conv backward: workspace too small");
    return GRM_HIP_EINVAL;
  }
  const bool vec = whole_rows(a, dtype);
  a.stream = streams(batch * a.T * channels, dtype);
  const int64_t v = vec ? 4 : 1;
  a.run = bwd_run(batch, seq_len, channels, vec);
  a.runs = ceil_div(seq_len > 0 ? seq_len : 1, a.run);
  const int64_t parts = batch > 0 ? bwd_parts(batch, seq_len, a.run) : 0;
  const int64_t blocks = ceil_div(channels, 64 * v), weight_blocks = ceil_div(channels * (width + 1), 64);
  if (weight_blocks >= kMaxBlocks || blocks > kMaxBlocks) {  // (512 threads a block, fewer than 2^32 in all)
    set_error("short_conv backward: too many elements for one launch");
    return GRM_HIP_EUNSUPPORTED;
  }
  int rc = GRM_HIP_OK;
  with_form<4>(dtype, vec, width, silu != 0, [&](auto e, auto vv, auto w, auto act) {
    using E = decltype(e);
    constexpr int W = decltype(w)::value;
    if (parts > 0) {
      conv_bwd_kernel<E, decltype(vv)::value, W, decltype(act)::value>
          <<<dim3(static_cast<uint32_t>(blocks), static_cast<uint32_t>(parts)), dim3(kThreads), 0,
             static_cast<hipStream_t>(stream)>>>(a);
      if ((rc = check_launch("short_conv backward")) != GRM_HIP_OK) return;
    }
    conv_weight_kernel<E, W><<<dim3(static_cast<uint32_t>(weight_blocks)), dim3(512), 0,
                               static_cast<hipStream_t>(stream)>>>(a.partial, grad_weight, grad_bias, channels,
                                                                   static_cast<int>(parts), a.w_f32);
    rc = check_launch("short_conv backward, weights");
  });
  return rc;
}

extern "C" int grm_hip_short_conv_step(const void* x, const void* weight, const void* bias, const void* state,
                                       void* out, void* state_out, int64_t batch, int64_t channels, int64_t width,
                                       int64_t x_batch_stride, int dtype, int weight_dtype, int silu, void* stream) {
  ConvArgs a{};
  a.x = x; a.weight = weight; a.bias = bias; a.state = state; a.out = out; a.state_out = state_out;
  a.xb = x_batch_stride; a.xt = 0; a.B = batch; a.T = 1; a.C = channels;
  a.w_f32 = weight_dtype == GRM_HIP_F32;
  if (int rc = check_conv(a, width, dtype, weight_dtype, "short_conv_step")) return rc;
  if (batch == 0) return GRM_HIP_OK;
  if (x == nullptr || weight == nullptr || state == nullptr || out == nullptr || state_out == nullptr) {
    set_error("short_conv_step: x, weight, state, out and state_out are required");
    return GRM_HIP_EINVAL;
  }
  const int64_t es = dtype == GRM_HIP_F32 ? 4 : 2, st_bytes = batch * (width - 1) * channels * es;
  if (state != state_out && ranges_overlap(state, st_bytes, state_out, st_bytes)) {
    set_error("short_conv_step: state_out must be the state itself or not overlap it");
    return GRM_HIP_EINVAL;
  }
  const bool vec = whole_rows(a, dtype);
  a.stream = streams(batch * a.T * channels, dtype);
  const int64_t cv = vec ? channels / (dtype == GRM_HIP_F32 ? 4 : 8) : channels;
  const int64_t blocks = ceil_div(batch * cv, kThreads);
  if (blocks > kMaxBlocks) {
    set_error("short_conv_step: too many elements for one launch");
    return GRM_HIP_EUNSUPPORTED;
  }
  with_form<8>(dtype, vec, width, silu != 0, [&](auto e, auto v, auto w, auto act) {
    conv_step_kernel<decltype(e), decltype(v)::value, decltype(w)::value, decltype(act)::value>
        <<<dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0, static_cast<hipStream_t>(stream)>>>(a);
  });
  return check_launch("short_conv_step");
}
