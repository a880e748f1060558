// Pieces shared by the selective scan's kernels (selective_scan.hip, selective_bwd.hip).
//
// Tiles and fragments.  Token tiles lie in LDS row-major, one row a token, rows padded by 16
// bytes so that 16 rows fall on distinct banks.  Two orders of the reduction slots are used:
// along a row (key or value dimensions) slot s of lane group g is element 8g + s; along a column
// (tokens) slots 0-3 are tokens 4g + s and slots 4-7 tokens 16 + 4g + s - 4 of a 32-token step,
// which is how two 16x16 accumulators sit in the registers, so that a product feeds the next one
// without passing through LDS.
#pragma once

#include <stdint.h>

#include <type_traits>

#include "f32_tiles.h"
#include "grm_hip.h"
#include "grm_hip_common.h"

namespace grmhip {

constexpr int kSelRows = 64;  // value rows of a state tile

// Compute type M: BF16 inputs run bf16 MFMA; float32 and float16 inputs run float32 MFMA on float32 tiles (states
// and decayed weights leave float16's range, and splitting both operands into bfloat16 parts would
// cost as many products).
template <class M>
struct SelShape {
  static constexpr bool kHalf = sizeof(typename ET<M>::raw) == 2;
  static constexpr int L = kHalf ? 64 : 32;       // tokens of a walk's chunk
  static constexpr int LB = kHalf ? 128 : 64;     // tokens of a backward chunk (states are kept this often)
  static constexpr int PAD = kHalf ? 8 : 4;       // 16 bytes
  static constexpr int XS = kSelRows + PAD;       // value row stride
  static constexpr int PARTS = kHalf ? 3 : 1;     // bfloat16 parts that hold a float32 (24 bits)
};

struct SelArgs {
  const void* keys;     // [B, T, G, N]
  const void* values;   // [B, T, H, P]
  const void* queries;  // [B, T, G, N]
  const void* steps;    // [B, T, H]
  const float* rates;   // [H]
  const float* skip;    // [H] or null
  const float* bias;    // [H] or null
  const int64_t* lengths;  // [B] or null
  const float* memory;  // [B, H, P, N] or null: the state (or its gradient) that a walk starts from
  void* hidden;         // [B, T, H, P]
  float* memory_out;    // [B, H, P, N]
  float* states;        // [B, nsave, H, P, N] or null
  float* part_state;    // [parts, B, H, P, N]
  double* part_log;     // [parts, B, H]: log2 decay of each part
  int64_t kb, kt, vb, vt, qb, qt, sb, st;  // elements between sequences and between tokens
  int64_t T, nsave, part_tokens;
  int B, H, P, G, N, PT, parts;
  int steps_f32, softplus, vec;
};

__device__ __forceinline__ float exp2_f(float x) { return __builtin_amdgcn_exp2f(x); }

// 2^x of a float64 exponent: a single float would be off by 2^-24 |x|.
__device__ __forceinline__ float exp2_d(double x) {
  const float hi = static_cast<float>(x);
  return exp2_f(hi) * exp2_f(static_cast<float>(x - hi));
}

// Workgroups go round the eight XCDs; this gives each XCD a run of consecutive numbers, so that heads
// that read the same keys and queries share its L2.
__device__ __forceinline__ uint32_t xcd_order(uint32_t block, uint32_t total) {
  const uint32_t per = total >> 3, more = total & 7, x = block & 7;
  return x * per + (x < more ? x : more) + (block >> 3);
}

__device__ __forceinline__ int64_t sel_length(const SelArgs& a, int b) {
  return a.lengths == nullptr ? a.T : max_i64(0, min_i64(a.lengths[b], a.T));
}

// steps + bias of a token, before softplus.
template <class E>
__device__ __forceinline__ float raw_step(const SelArgs& a, int b, int64_t t, int h) {
  const float z = ld_state<E>(a.steps, b * a.sb + t * a.st + h, a.steps_f32 != 0);
  return a.bias == nullptr ? z : z + a.bias[h];
}

__device__ __forceinline__ float step_size(const SelArgs& a, float z) {
  return !a.softplus || z > 20.f ? z : log1pf(__expf(z));
}

// One wave's scan over a chunk's log decays, lane = token.  In log2 units and float64: a chunk's
// sum reaches hundreds, and decays between its tokens are differences of it.  A token's log decay is
// held to at least -200 (a factor of 1e-87, zero in float32), so that sums stay finite.
struct TokenScalars {
  float d;        // step size, 0 for a token behind the length
  double cum;     // log2 of the decay from the chunk's start through this token
  double total;   // of the whole chunk
};

template <class E, int L>
__device__ __forceinline__ TokenScalars token_scalars(const SelArgs& a, int b, int h, int64_t t, int64_t n, float rate) {
  const int lane = lane_id();
  TokenScalars s;
  s.d = lane < L && t < n ? step_size(a, raw_step<E>(a, b, t, h)) : 0.f;
  double l = static_cast<double>(s.d) * static_cast<double>(rate);
  l = l < -200.0 ? -200.0 : l;
  l *= 1.4426950408889634;  // log2(e)
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double up = __shfl_up(l, o);
    if (lane >= o) l += up;
  }
  s.cum = l;
  s.total = __shfl(l, L - 1);
  return s;
}

// Fragment of 16 rows (row + lane % 16), reduction along the row from `col`.
template <class M>
__device__ __forceinline__ Frag8<M> row_frag(const typename ET<M>::raw* tile, int stride, int row, int col) {
  const int lane = lane_id();
  const typename ET<M>::raw* p = tile + (row + (lane & 15)) * stride + col + 8 * (lane >> 4);
  return lds_frag_4x2<M>(p, p + 4);
}

// Fragment of 16 columns (col + lane % 16), reduction over 32 tokens from row `t0`.
template <class M>
__device__ __forceinline__ Frag8<M> col_frag(const typename ET<M>::raw* tile, int stride, int t0, int col) {
  const int lane = lane_id(), g = lane >> 4, n = lane & 15;
  Frag8<M> f;
  if constexpr (sizeof(typename ET<M>::raw) == 2) {
    // The transpose read hands lane i of a 16-lane block X[r0 + e][c0 + i], e = 0..3, when lane s
    // passes &X[r0 + (s >> 2)][c0 + 4 (s & 3)].
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const typename ET<M>::raw* p = tile + (t0 + 4 * g + (n >> 2)) * stride + col + 4 * (n & 3);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 16 * stride));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f.e[e] = static_cast<uint16_t>(lo[e]);
      f.e[4 + e] = static_cast<uint16_t>(hi[e]);
    }
  } else {
    const float* p = tile + (t0 + 4 * g) * stride + col + n;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f.e[e] = p[e * stride];
      f.e[4 + e] = p[(16 + e) * stride];
    }
  }
  return f;
}

// Two accumulators (tokens 0-15 and 16-31 of a step) as one fragment.
template <class M>
__device__ __forceinline__ Frag8<M> pair_frag(f32x4 lo, f32x4 hi) {
  if constexpr (sizeof(typename ET<M>::raw) == 2) {
    return __builtin_bit_cast(Frag8<M>, make_uint4(pack2<M>(lo[0], lo[1]), pack2<M>(lo[2], lo[3]),
                                                   pack2<M>(hi[0], hi[1]), pack2<M>(hi[2], hi[3])));
  } else {
    Frag8<M> f;
#pragma unroll
    for (int e = 0; e < 4; ++e) { f.e[e] = lo[e]; f.e[4 + e] = hi[e]; }
    return f;
  }
}

// Float32 values as PARTS fragments whose sum they are: each the rounded remainder of the ones before.
template <class M, int PARTS>
__device__ __forceinline__ void split_frag(const float (&v)[8], Frag8<M> (&out)[PARTS]) {
  float rest[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) rest[e] = v[e];
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    out[p] = pair_frag<M>(f32x4{rest[0], rest[1], rest[2], rest[3]}, f32x4{rest[4], rest[5], rest[6], rest[7]});
#pragma unroll
    for (int e = 0; e < 8; ++e) rest[e] -= ET<M>::to_f(out[p].e[e]);
  }
}

// Rows [0, ROWS) x [0, COLS) of a tile from global memory into registers (8 elements a unit, units dealt to
// THREADS threads), then into LDS as M.  Rows from `rows` on and columns from `cols` on are zeros.
template <class E, class M, int ROWS, int COLS, int THREADS>
struct TileLoad {
  static constexpr int UPR = COLS / 8, UNITS = ROWS * UPR, PER = (UNITS + THREADS - 1) / THREADS;
  U8<E> r[PER];
  __device__ __forceinline__ void load(const void* base, int64_t at, int64_t stride, int64_t rows, int cols, bool vec,
                                       int tid) {
    const typename ET<E>::raw* p = static_cast<const typename ET<E>::raw*>(base) + at;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = tid + i * THREADS, row = u / UPR, col = u % UPR * 8;
      r[i] = load_u8<E>(p + row * stride, col, cols, u < UNITS && row < rows, vec);
    }
  }
  __device__ __forceinline__ void store(typename ET<M>::raw* tile, int stride, int tid) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = tid + i * THREADS, row = u / UPR, col = u % UPR * 8;
      if (u < UNITS) {
        typename ET<M>::raw* p = tile + row * stride + col;
        if constexpr (sizeof(typename ET<M>::raw) == 2) {
          *reinterpret_cast<uint4*>(p) = __builtin_bit_cast(uint4, r[i]);
        } else {
          float4 lo, hi;
          lo.x = ET<E>::to_f(r[i].e[0]); lo.y = ET<E>::to_f(r[i].e[1]); lo.z = ET<E>::to_f(r[i].e[2]); lo.w = ET<E>::to_f(r[i].e[3]);
          hi.x = ET<E>::to_f(r[i].e[4]); hi.y = ET<E>::to_f(r[i].e[5]); hi.z = ET<E>::to_f(r[i].e[6]); hi.w = ET<E>::to_f(r[i].e[7]);
          reinterpret_cast<float4*>(p)[0] = lo;
          reinterpret_cast<float4*>(p)[1] = hi;
        }
      }
    }
  }
};

// A wave's 16 value rows of a state, rows p0 .. p0 + 15 of [P, N]: acc[nt][r] is row p0 + lane % 16,
// column 16 nt + 4 (lane / 16) + r.
template <int NT>
__device__ __forceinline__ void state_add(f32x4 (&acc)[NT], const float* s, int p0, int P, int N, float scale) {
  const int lane = lane_id(), p = p0 + (lane & 15);
  const bool whole = (N & 3) == 0;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int n = nt * 16 + 4 * (lane >> 4);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (p < P && n < N) {
      const float* q = s + static_cast<int64_t>(p) * N + n;
      if (whole) {
        const float4 u = *reinterpret_cast<const float4*>(q);
        v = f32x4{u.x, u.y, u.z, u.w};
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = n + r < N ? q[r] : 0.f;
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[nt][r] = fmaf(scale, v[r], acc[nt][r]);
  }
}

template <int NT>
__device__ __forceinline__ void state_store(const f32x4 (&acc)[NT], float* s, int p0, int P, int N) {
  const int lane = lane_id(), p = p0 + (lane & 15);
  const bool whole = (N & 3) == 0;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int n = nt * 16 + 4 * (lane >> 4);
    if (p < P && n < N) {
      float* q = s + static_cast<int64_t>(p) * N + n;
      if (whole) {
        *reinterpret_cast<float4*>(q) = make_float4(acc[nt][0], acc[nt][1], acc[nt][2], acc[nt][3]);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (n + r < N) q[r] = acc[nt][r];
        }
      }
    }
  }
}

// acc = decay acc + sum_t weight_t x_t[p] k_t^T over a chunk's L tokens: x the value tile (this wave's 16 rows from
// column `xc`), k the key tile.  weight_t x_t is a float32 number, kept whole as three bfloat16 parts:
// the state is carried over thousands of tokens, where a rounding to fewer bits would add up.
template <class M, int L, int NT>
__device__ __forceinline__ void state_update(f32x4 (&acc)[NT], const typename ET<M>::raw* k, int ks,
                                             const typename ET<M>::raw* x, int xs, int xc, const float* weight,
                                             float decay) {
  constexpr int PARTS = SelShape<M>::PARTS;
  const int g = lane_id() >> 4;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[nt][r] *= decay;
  }
#pragma unroll
  for (int t0 = 0; t0 < L; t0 += 32) {
    const Frag8<M> xf = col_frag<M>(x, xs, t0, xc);
    const f32x4 w0 = *reinterpret_cast<const f32x4*>(weight + t0 + 4 * g);
    const f32x4 w1 = *reinterpret_cast<const f32x4*>(weight + t0 + 16 + 4 * g);
    float v[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = ET<M>::to_f(xf.e[e]) * w0[e];
      v[4 + e] = ET<M>::to_f(xf.e[4 + e]) * w1[e];
    }
    Frag8<M> part[PARTS];
    split_frag<M, PARTS>(v, part);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const Frag8<M> kf = col_frag<M>(k, ks, t0, nt * 16);
#pragma unroll
      for (int p = PARTS - 1; p >= 0; --p) acc[nt] = mfma8(kf, part[p], acc[nt]);
    }
  }
}

// Host side.
inline int64_t sel_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }
int sel_check(const struct grm_hip_selective_args* u, const char* what);
SelArgs sel_args(const struct grm_hip_selective_args* u);
// Tokens of a backward chunk, and time parts of a walk: part_tokens set to a multiple of it.
int64_t sel_block(int dtype);
int sel_parts(int64_t seqs, int64_t T, int dtype, int64_t* part_tokens);
// The state walk alone (selective_scan.hip): part-local sums, or the reverse walk of the backward.
int launch_state_pass(const SelArgs& a, int dtype, bool reverse, bool local, hipStream_t stream, const char* what);

}  // namespace grmhip
