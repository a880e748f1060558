// Pieces shared by the selective scan's kernels (selective_scan.hip, selective_bwd.hip).
//
// Tiles and fragments.  Tiles lie in LDS row-major (a row is a token, or a value row of a state).  Two orders of the reduction slots are used:
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

// Compute type M: BF16 inputs run bf16 MFMA; float32 and float16 inputs run float32 MFMA on float32 tiles, which keeps
// every bit in one product.  (bfloat16 parts would do too, a float16 number being two of them and a float32 one
// three: four products for q . k of float16, six for a state's update, of a sixteenth of the cycles each.  That form is not
// built; the float32 one is 7 to 14 times its floor in bytes at 5 x 777 float16 tokens x 12 heads.)
template <class M>
struct SelShape {
  static constexpr bool kHalf = sizeof(typename ET<M>::raw) == 2;
  static constexpr int L = kHalf ? 64 : 32;       // tokens of a walk's chunk
  static constexpr int LB = kHalf ? 128 : 64;     // tokens of a backward chunk (states are kept this often)
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
  int stream;  // outputs are stored past the caches
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

// A token's entry of steps as it lies in memory (16 bits in the low half), 0 where not `live`.  Nothing is
// done to it here, so that a load ahead of time is waited for where it is used.
template <class E>
__device__ __forceinline__ uint32_t load_step(const SelArgs& a, int b, int64_t t, int h, bool live) {
  const int64_t at = b * a.sb + t * a.st + h;
  uint32_t v = 0;
  if (a.steps_f32 || std::is_same_v<E, F32>) {
    if (live) v = static_cast<const uint32_t*>(a.steps)[at];
  } else {
    if (live) v = static_cast<const uint16_t*>(a.steps)[at];
  }
  return v;
}
template <class E>
__device__ __forceinline__ float step_value(const SelArgs& a, uint32_t v) {
  if constexpr (std::is_same_v<E, F32>) return __uint_as_float(v);
  else return a.steps_f32 ? __uint_as_float(v) : ET<E>::to_f(static_cast<uint16_t>(v));
}
// steps + bias of a token, before softplus.
template <class E>
__device__ __forceinline__ float raw_step(const SelArgs& a, int b, int64_t t, int h) {
  const float z = step_value<E>(a, load_step<E>(a, b, t, h, true));
  return a.bias == nullptr ? z : z + a.bias[h];
}

__device__ __forceinline__ float step_size(const SelArgs& a, float z) {
  return !a.softplus || z > 20.f ? z : log1pf(__expf(z));
}

// x of the lane that a DPP control names, 0 where it names none or the row mask leaves this row out.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_f64(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// Inclusive prefix sum over the wave: inside rows of 16 lanes, then from row to row.
__device__ __forceinline__ double wave_prefix(double x) {
  x += dpp_f64<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
  x += dpp_f64<0x112, 0xf>(x);
  x += dpp_f64<0x114, 0xf>(x);
  x += dpp_f64<0x118, 0xf>(x);
  x += dpp_f64<0x142, 0xa>(x);  // lane 15 of rows 0 and 2 to the next row
  x += dpp_f64<0x143, 0xc>(x);  // lane 31 to rows 2 and 3
  return x;
}
__device__ __forceinline__ double lane_value(double x, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(b), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(b >> 32), lane);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// One wave's scan over a chunk's log decays, lane = token.  In log2 units and float64: a chunk's
// sum reaches hundreds, and decays between its tokens are differences of it.  A token's log decay is
// held to at least -200 (a factor of 1e-87, zero in float32), so that sums stay finite.
struct TokenScalars {
  float d;        // step size, 0 for a token behind the length
  double cum;     // log2 of the decay from the chunk's start through this token
  double total;   // of the whole chunk
};

template <int L>
__device__ __forceinline__ TokenScalars token_scalars(const SelArgs& a, float z, bool live, float rate) {
  TokenScalars s;
  s.d = lane_id() < L && live ? step_size(a, z) : 0.f;
  double l = live ? static_cast<double>(s.d) * static_cast<double>(rate) : 0.0;  // (the rate may be infinite)
  l = l < -200.0 ? -200.0 : l;
  l *= 1.4426950408889634;  // log2(e)
  s.cum = wave_prefix(l);
  s.total = lane_value(s.cum, L - 1);
  return s;
}

// LDS tiles with rows of W elements, padded against bank conflicts (64 banks of 4 bytes).  Measured with
// SQ_LDS_BANK_CONFLICT, clocks per read of one wave:
//                                     rows 4 banks apart   8 banks apart
//   transpose read (8 rows x 32 bytes)        4                  2
//   16 bytes of each of 16 rows               8                  4
//   8 bytes of each of 16 rows                2                  4
// COLS: 8 banks apart modulo 64, for tiles read by columns (and rows in 16 bytes); else 4, for tiles
// read by rows in 8 bytes.  (XORed granules without padding are as good for the transpose reads, but
// their addresses differ from lane to lane, so that the two halves of a fragment are no constant
// distance apart: slower.)  Float32 tiles: 4 banks apart.
template <class M, int W, bool COLS>
struct SelTile {
  static constexpr bool kHalf = SelShape<M>::kHalf;
  static constexpr int STRIDE = W + (!kHalf ? 4 : COLS ? 16 : 8);
  __device__ __forceinline__ static int at(int row, int col) { return row * STRIDE + col; }
};

// Fragment of 16 rows (row + lane % 16), reduction along the row from `col`.
template <class T, class M>
__device__ __forceinline__ Frag8<M> row_frag(const typename ET<M>::raw* tile, int row, int col, int lane = lane_id()) {
  const typename ET<M>::raw* p = tile + T::at(row + (lane & 15), col + 8 * (lane >> 4));
  if constexpr (sizeof(typename ET<M>::raw) == 2) return __builtin_bit_cast(Frag8<M>, *reinterpret_cast<const uint4*>(p));
  else return lds_frag_4x2<M>(p, p + 4);
}

// The same with the reduction in the tokens' slot order (4g + s, 16 + 4g + s).
template <class T, class M>
__device__ __forceinline__ Frag8<M> row_frag_t(const typename ET<M>::raw* tile, int row, int col, int lane = lane_id()) {
  const int r = row + (lane & 15), c = col + 4 * (lane >> 4);
  return lds_frag_4x2<M>(tile + T::at(r, c), tile + T::at(r, c + 16));
}

// Fragment of 16 columns (col + lane % 16), reduction over the 16 tokens from row `t0` and the 16 from row `t1`.
template <class T, class M>
__device__ __forceinline__ Frag8<M> col_frag2(const typename ET<M>::raw* tile, int t0, int t1, int col, int lane = lane_id()) {
  const int g = lane >> 4, n = lane & 15;
  Frag8<M> f;
  if constexpr (sizeof(typename ET<M>::raw) == 2) {
    // The transpose read hands lane i of a 16-lane block X[r0 + e][c0 + i], e = 0..3, when lane s
    // passes &X[r0 + (s >> 2)][c0 + 4 (s & 3)].
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const typename ET<M>::raw* p = tile + T::at(4 * g + (n >> 2), col + 4 * (n & 3));
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + t0 * T::STRIDE));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + t1 * T::STRIDE));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f.e[e] = static_cast<uint16_t>(lo[e]);
      f.e[4 + e] = static_cast<uint16_t>(hi[e]);
    }
  } else {
    constexpr int S = T::STRIDE;
    const float* p = tile + 4 * g * S + col + n;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f.e[e] = p[(t0 + e) * S];
      f.e[4 + e] = p[(t1 + e) * S];
    }
  }
  return f;
}
template <class T, class M>
__device__ __forceinline__ Frag8<M> col_frag(const typename ET<M>::raw* tile, int t0, int col, int lane = lane_id()) {
  return col_frag2<T, M>(tile, t0, t0 + 16, col, lane);
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

// What a rounded part leaves of v: of an infinity the same infinity, so that products with its parts have its sign.
template <class M>
__device__ __forceinline__ float part_rest(float v, typename ET<M>::raw part) {
  return v - __builtin_amdgcn_fmed3f(ET<M>::to_f(part), -3.4028235e38f, 3.4028235e38f);
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
    for (int e = 0; e < 8; ++e) rest[e] = part_rest<M>(rest[e], out[p].e[e]);
  }
}

// Two accumulators as pair_frag, in parts.
template <class M, int PARTS>
__device__ __forceinline__ void split_pair(f32x4 lo, f32x4 hi, Frag8<M> (&out)[PARTS]) {
  const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  split_frag<M, PARTS>(v, out);
}

// Rows [0, ROWS) x [0, COLS) of a tile from global memory into registers (8 elements a unit, units dealt to
// THREADS threads), then into LDS as M.  Rows from `rows` on and columns from `cols` on are zeros: they
// lie outside the buffer resource or are sent there, so no load stands behind a branch and all stay in
// flight until the tile is stored.
// VEC: every row's units are whole 16-byte accesses.
template <class E, class T, class M, bool VEC, int ROWS, int COLS, int THREADS>
struct TileLoad {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  static constexpr int ES = static_cast<int>(sizeof(typename ET<E>::raw));
  static constexpr int UPR = COLS / 8, UNITS = ROWS * UPR, PER = (UNITS + THREADS - 1) / THREADS, W = ES / 2;
  static constexpr int DROW = THREADS / UPR;  // rows between a thread's units
  static_assert(THREADS % UPR == 0 && (UNITS % THREADS == 0 || PER == 1), "a thread's units share a column");
  u32x4 r[PER][W];
  // Byte offset of this thread's first unit, out of range where its column is.  Rows past `rows` rely on the range check,
  // so the rows' steps are added here and not left to the scalar offset, which the check need not see.
  uint32_t off;
  int at;           // element in the LDS tile
  int step, width;  // bytes from row to row, columns

  // stride in elements, at least cols.
  __device__ __forceinline__ void init(int64_t stride, int cols, int tid) {
    step = static_cast<int>(stride) * ES;
    width = cols;
    const int row = tid / UPR, col = tid % UPR * 8;
    off = col < cols && tid < UNITS ? row * step + col * ES : kBufOOB;
    at = T::at(row, col);
  }
  // base: the first row's first element.
  __device__ __forceinline__ void load(const typename ET<E>::raw* base, int64_t rows, int tid) {
    const int n = static_cast<int>(max_i64(0, min_i64(rows, ROWS)));
    const __amdgpu_buffer_rsrc_t rsrc =
        make_rsrc(base, n > 0 ? static_cast<uint32_t>((n - 1) * step + width * ES) : 0u);
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
#pragma unroll
        for (int w = 0; w < W; ++w)
          r[i][w] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, off + static_cast<uint32_t>(i * DROW * step + 16 * w), 0, 0);
      }
    } else {
      const int col = tid % UPR * 8;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int row = tid / UPR + i * DROW;
        const bool in = tid < UNITS && row < n;
#pragma unroll
        for (int w = 0; w < W; ++w) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (ES == 4) {
              const int c = col + 4 * w + k;
              r[i][w][k] = __builtin_amdgcn_raw_buffer_load_b32(rsrc, in && c < width ? row * step + c * 4 : kBufOOB, 0, 0);
            } else {
              const int c = col + 2 * k;
              const uint32_t lo = static_cast<uint16_t>(
                  __builtin_amdgcn_raw_buffer_load_b16(rsrc, in && c < width ? row * step + c * 2 : kBufOOB, 0, 0));
              const uint32_t hi = static_cast<uint16_t>(
                  __builtin_amdgcn_raw_buffer_load_b16(rsrc, in && c + 1 < width ? row * step + c * 2 + 2 : kBufOOB, 0, 0));
              r[i][w][k] = lo | hi << 16;
            }
          }
        }
      }
    }
  }
  // Whether any element is an infinity or a NaN (all bits of its exponent are set).
  __device__ __forceinline__ bool odd() const {
    constexpr uint32_t X = std::is_same_v<E, F32> ? 0x7f800000u : std::is_same_v<E, BF16> ? 0x7f807f80u : 0x7c007c00u;
    constexpr uint32_t ONE = std::is_same_v<E, F32> ? 0x00800000u : std::is_same_v<E, BF16> ? 0x00800080u : 0x04000400u;
    uint32_t any = 0;  // one more in a full exponent carries into the sign
#pragma unroll
    for (int i = 0; i < PER; ++i) {
#pragma unroll
      for (int w = 0; w < W; ++w) {
#pragma unroll
        for (int k = 0; k < 4; ++k) any |= (r[i][w][k] & X) + ONE;
      }
    }
    return (any & (std::is_same_v<E, F32> ? 0x80000000u : 0x80008000u)) != 0;
  }
  // negated: with the other sign (16-bit tiles).
  __device__ __forceinline__ void store(typename ET<M>::raw* tile, int tid, bool negated = false) const {
    if (UNITS < THREADS && tid >= UNITS) return;
    const uint32_t flip = sizeof(typename ET<M>::raw) == 2 && negated ? 0x80008000u : 0u;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      typename ET<M>::raw* p = tile + at + i * DROW * T::STRIDE;
      if constexpr (ES == sizeof(typename ET<M>::raw)) {
#pragma unroll
        for (int w = 0; w < W; ++w) reinterpret_cast<u32x4*>(p)[w] = r[i][w] ^ flip;
      } else {
        const U8<E> e = __builtin_bit_cast(U8<E>, r[i][0]);
#pragma unroll
        for (int w = 0; w < 2; ++w)
          reinterpret_cast<float4*>(p)[w] = make_float4(ET<E>::to_f(e.e[4 * w]), ET<E>::to_f(e.e[4 * w + 1]),
                                                        ET<E>::to_f(e.e[4 * w + 2]), ET<E>::to_f(e.e[4 * w + 3]));
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

// The state's update acc = decay acc + sum_t weight_t x_t[p] k_t^T, 32 tokens at a time.  weight_t x_t is a float32
// number, kept whole as three bfloat16 parts: the state is carried over thousands of tokens, where a
// rounding to fewer bits would add up.
template <class M>
__device__ __forceinline__ void weigh_frag(const Frag8<M>& x, f32x4 w0, f32x4 w1, Frag8<M> (&part)[SelShape<M>::PARTS]) {
  float v[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = ET<M>::to_f(x.e[e]) * w0[e];
    v[4 + e] = ET<M>::to_f(x.e[4 + e]) * w1[e];
  }
  split_frag<M, SelShape<M>::PARTS>(v, part);
}
template <class M, int NT>
__device__ __forceinline__ void update_step(f32x4 (&acc)[NT], const Frag8<M> (&kf)[NT],
                                            const Frag8<M> (&part)[SelShape<M>::PARTS]) {
#pragma unroll
  for (int p = SelShape<M>::PARTS - 1; p >= 0; --p) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc[nt] = mfma8(kf[nt], part[p], acc[nt]);
  }
}
template <class T, class M, int NT>
__device__ __forceinline__ void key_frags(Frag8<M> (&kf)[NT], const typename ET<M>::raw* k, int t0) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) kf[nt] = col_frag<T, M>(k, t0, nt * 16);
}
// Keeps what stands before it before it: reads issued ahead stay ahead.
__device__ __forceinline__ void hold_order() { __builtin_amdgcn_sched_barrier(0); }

// A 16- or 8-byte store, past the caches where `stream`.
template <class T>
__device__ __forceinline__ void store_as(T* p, T v, bool stream) {
  if (stream) __builtin_nontemporal_store(v, p);
  else *p = v;
}

// A lane's tiles hold four columns of one row, 64 bytes of each of 16 rows a store.  Two tiles' halves are exchanged
// between lanes eight apart first, so that a store covers 128 bytes, a whole line, of each of eight rows (reverse walk of
// 8 x 2048 tokens x 32 heads 97 -> 84 us, the forward with its states 137 -> 119).  `sign`: 1 or -1, a factor.
template <int NT>
__device__ __forceinline__ void state_store(const f32x4 (&acc)[NT], float* s, int p0, int P, int N, float sign = 1.f) {
  static_assert(NT % 2 == 0, "tiles in pairs");
  int lane = lane_id();
  asm volatile("" : "+v"(lane));  // no address made from it is kept in registers between stores
  const int p = lane & 15, low = p & 8;
  if ((N & 3) == 0) {
    const __amdgpu_buffer_rsrc_t rsrc = make_rsrc(s, static_cast<uint32_t>(P * N * 4));
#pragma unroll
    for (int nt = 0; nt < NT; nt += 2) {
      const int n = nt * 16 + 2 * low + 4 * (lane >> 4);
      f32x4 v[2];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float give = low ? acc[nt][r] : acc[nt + 1][r];
        const float take = __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(give), 0x128, 0xf, 0xf, true));
        v[0][r] = low ? take : acc[nt][r];
        v[1][r] = low ? acc[nt + 1][r] : take;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        const int row = p0 + 8 * u + (p & 7), at = row < P && n < N ? (row * N + n) * 4 : kBufOOB;
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v[u] * sign), rsrc, at, 0, 0);
      }
      hold_order();
    }
  } else if (p0 + p < P) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = nt * 16 + 4 * (lane >> 4) + r;
        if (n < N) s[static_cast<int64_t>(p0 + p) * N + n] = sign * acc[nt][r];
      }
    }
  }
}

// Host side: f(E, M, NP, VEC) with one of the compiled forms.
template <class F>
void sel_with_form(int dtype, int64_t N, bool vec, F f) {
  auto by_vec = [&](auto e, auto m, auto np) {
    if (vec) f(e, m, np, std::true_type{});
    else f(e, m, np, std::false_type{});
  };
  auto by_width = [&](auto e, auto m) {
    if (N <= 32) by_vec(e, m, std::integral_constant<int, 32>{});
    else if (N <= 64) by_vec(e, m, std::integral_constant<int, 64>{});
    else by_vec(e, m, std::integral_constant<int, 128>{});
  };
  if (dtype == GRM_HIP_BF16) by_width(BF16{}, BF16{});
  else if (dtype == GRM_HIP_F16) by_width(F16{}, F32{});
  else by_width(F32{}, F32{});
}
inline int64_t sel_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }
// More than the eight 4 MB L2 caches hold is stored past them: what would be written back at the kernel's end leaves
// during it: the step of 64 sequences x 32 heads 33.8 -> 33.3 us, back to back; the scan of 8 x 2048 tokens x 32 heads the same
// either way.
inline int sel_streams(int64_t bytes) { return bytes > (int64_t{32} << 20); }
int sel_check(const struct grm_hip_selective_args* u, const char* what, bool step = false);
SelArgs sel_args(const struct grm_hip_selective_args* u);
// Tokens of a backward chunk, and time parts of a walk: part_tokens set to a multiple of it.
int64_t sel_block(int dtype);
int sel_parts(int64_t seqs, int64_t T, int dtype, int64_t* part_tokens);
// The state walk alone (selective_scan.hip): part-local sums, or the reverse walk of the backward.
int launch_state_pass(const SelArgs& a, int dtype, bool reverse, bool local, hipStream_t stream, const char* what);

}  // namespace grmhip
