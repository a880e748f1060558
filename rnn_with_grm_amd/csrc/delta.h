// Pieces shared by the delta rule's kernels (delta_scan.hip, delta_bwd.hip).
//
//   u_t = b_t (v_t - a_t M_{t-1} k_t),  M_t = a_t M_{t-1} + u_t k_t^T,  h_t = M_t q_t,  a_t = exp(g_t)
//
// A chunk of 64 tokens from state S, with c the running sum of g, D_i = e^{c_i}, W_ij = e^{c_i - c_j} (j <= i),
// E_j = e^{c_63 - c_j} and diag(b) written b:
//   m = v - a M k solves (I + A b) m = V - D K S^T with A_ij = W_ij k_i.k_j (j < i); u = b m
//   H = D Q S^T + (W * Q K^T) b m,   S' = e^{c_63} S + (E b m)^T K
// The inverse of I + A b and the weights W * Q K^T hang on no state: a launch of their own forms them for all chunks side
// by side (delta_prep_kernel) and leaves them in the order in which matrix products read them.
//
// Numbers.  States, m and everything that reaches them are float32.  Products run on the bf16 MFMA: a float32
// number is the sum of three bfloat16 parts, a float16 one of two, a bfloat16 one is itself, and the pairs of parts whose
// product reaches 2^-24 of the whole are multiplied (six of nine; three where one side is bfloat16).  That costs 3/16 to
// 6/16 of the float32 MFMA's cycles.
// What only reaches a 16-bit output takes two parts, and their three larger products: 2^-16 of a term is lost where the output's
// rounding loses 2^-9 or 2^-12.  These are the state and m as queries read them, W * Q K^T, and X, Y of the keys' and queries'
// gradients; the state itself and all that a later token reads keep their 24 bits.  With three parts there, bfloat16 outputs differ
// from a float32 form's by 3.7e-5 of their norm instead of 1.2e-4 (neighbours in the last rounding), the error against float64
// is the same (1.7e-3; float16 2.1e-4), and calls take longer: 8 x 2048 bf16 tokens x 16 heads of 128 x 128 180 -> 199 us, with
// gradients 953 -> 988, 32768 tokens 638 -> 681, 5 x 777 x 12 heads float16 63 -> 66.
#pragma once

#include "selective.h"

namespace grmhip {

constexpr int kDTokens = 64;   // tokens of a chunk
constexpr int kDCols = 64;     // value columns of a walk's workgroup, 16 a wave
constexpr int kDFrags = 6;     // 16 x 32 fragments of a triangular 64 x 64 matrix
constexpr int kDFragElems = 512;
constexpr int kDScal = 208;    // floats kept of a chunk: D, E (forward: E b), b, first odd token

// Parts of an input, and of a float32 number that only reaches outputs of type E.
template <class E> struct DParts;
template <> struct DParts<BF16> { static constexpr int IN = 1, OUT = 2; };
template <> struct DParts<F16> { static constexpr int IN = 2, OUT = 2; };
template <> struct DParts<F32> { static constexpr int IN = 3, OUT = 3; };

typedef Frag8<BF16> B8;

struct DeltaArgs {
  const void *keys, *values, *queries;  // [B, T, G, N], [B, T, H, P], [B, T, G, N]
  const void *strengths, *decays;       // [B, T, H]; decays may be null
  const int64_t* lengths;               // [B] or null
  const float* memory;                  // [B, H, P, N] or null
  void* hidden;                         // [B, T, H, P]
  float* memory_out;                    // [B, H, P, N]
  float* states;                        // [B, C, H, P, N] or null: the state before every chunk
  float* miss;                          // [B, T, H, P] or null: m
  char* work;                           // what delta_prep_kernel leaves, [B, H, C]
  float* part_state;                    // [parts - 1, B, H, P, N]: what a part leaves of a zero state, then the state behind it
  float* part_map;                      // [parts - 1, B, H, N, N]: what a part makes of the identity, without values
  int64_t kb, kt, vb, vt, qb, qt, sb, st, db, dt;
  int64_t T;
  int B, H, P, G, N, C, PT;
  int parts, part_chunks, NT;           // time parts, their chunks, tiles of 64 rows of a part's map
  int mirror;                           // parts are numbered from the last one
  int s_f32, d_f32, vec;
};

// Bytes of a chunk of a head in the workspace: the inverse in three parts, the weights in PP parts, scalars.
constexpr int64_t delta_chunk_bytes(int pp) { return (3 + pp) * kDFrags * kDFragElems * 2 + kDScal * 4; }

// Fragment of row tile `t` and reduction step `s` among the six of a lower triangular matrix (columns up to the
// row), and of an upper triangular one (from the row on).
__host__ __device__ constexpr int lower_frag(int t, int s) { return t == 0 ? 0 : t == 1 ? 1 : t == 2 ? 2 + s : 4 + s; }
__host__ __device__ constexpr int upper_frag(int t, int s) { return t == 0 ? s : t == 1 ? 2 + s : t == 2 ? 4 : 5; }

__device__ __forceinline__ int64_t delta_length(const DeltaArgs& a, int b) {
  return a.lengths == nullptr ? a.T : max_i64(0, min_i64(a.lengths[b], a.T));
}

// Float32 values as parts whose sum they are: each the rounded remainder of the ones before.  (An infinity's further
// parts are NaN, and so is what it reaches.)
template <int PARTS>
__device__ __forceinline__ void split8(const float (&v)[8], B8 (&out)[PARTS]) {
  float rest[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) rest[e] = v[e];
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      u[e] = pack2<BF16>(rest[2 * e], rest[2 * e + 1]);
      if (p + 1 < PARTS) {
        rest[2 * e] -= __uint_as_float(u[e] << 16);
        rest[2 * e + 1] -= __uint_as_float(u[e] & 0xffff0000u);
      }
    }
    out[p] = __builtin_bit_cast(B8, make_uint4(u[0], u[1], u[2], u[3]));
  }
}
// Two accumulators (tokens 0-15 and 16-31 of a step) as one fragment's parts.
template <int PARTS>
__device__ __forceinline__ void split2(f32x4 lo, f32x4 hi, B8 (&out)[PARTS]) {
  const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  split8<PARTS>(v, out);
}

// acc += sum of a[i] b[j] over the pairs with i + j < LIM, the smaller products first.
template <int LIM, int NA, int NB>
__device__ __forceinline__ f32x4 mma_parts(const B8 (&a)[NA], const B8 (&b)[NB], f32x4 acc) {
#pragma unroll
  for (int d = LIM - 1; d >= 0; --d) {
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int j = d - i;
      if (j >= 0 && j < NB) acc = mfma8(a[i], b[j], acc);
    }
  }
  return acc;
}

// The same for several accumulators that share b (ROWS: a[t] is the left operand; else the right one): consecutive
// products hang on different accumulators.
template <int LIM, bool ROWS, int C, int NA, int NB>
__device__ __forceinline__ void mma_many(const B8 (&a)[C][NA], const B8 (&b)[NB], f32x4 (&acc)[C]) {
#pragma unroll
  for (int d = LIM - 1; d >= 0; --d) {
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int j = d - i;
      if (j < 0 || j >= NB) continue;
#pragma unroll
      for (int t = 0; t < C; ++t) acc[t] = ROWS ? mfma8(a[t][i], b[j], acc[t]) : mfma8(b[j], a[t][i], acc[t]);
    }
  }
}

// Products of a triangular 64 x 64 matrix, whose six fragments are f, with b's two steps of tokens: acc[t] += rows of tile t.
// LOWER: tile t meets steps up to its own, else from its own on.  ROWS as above.
template <int LIM, bool LOWER, bool ROWS, int NA, int NB>
__device__ __forceinline__ void mma_triangle(const B8 (&f)[kDFrags][NA], const B8 (&b)[2][NB], f32x4 (&acc)[4]) {
#pragma unroll
  for (int d = LIM - 1; d >= 0; --d) {
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int j = d - i;
      if (j < 0 || j >= NB) continue;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          if (LOWER ? s > t / 2 : s < t / 2) continue;
          const B8& x = f[LOWER ? lower_frag(t, s) : upper_frag(t, s)][i];
          acc[t] = ROWS ? mfma8(x, b[s][j], acc[t]) : mfma8(b[s][j], x, acc[t]);
        }
      }
    }
  }
}

// Tiles nt and nt + 1 of a wave's 16 value rows of a state to memory, as state_store does (which takes all at once where rows
// are not of whole 16-byte units).  The walk stores them between the products that read them (8 x 2048 bf16 tokens x 16 heads of
// 128 x 128: 216 us behind the chunk's last product, 207 here); its mirror, whose output waves load and store more in
// that half, behind the last one (207-211 us; 220 between the products).
template <bool WHOLE, int NT>
__device__ __forceinline__ void state_out(const f32x4 (&acc)[NT], int nt, float* s, int p0, int P, int N) {
  if constexpr (!WHOLE) {
    if (nt == 0) state_store<NT>(acc, s, p0, P, N);
  } else {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    int lane = lane_id();
    asm volatile("" : "+v"(lane));  // no address made from it is kept in registers between stores
    const int low = lane & 8;
    const __amdgpu_buffer_rsrc_t rsrc = make_rsrc(s, static_cast<uint32_t>(P * N * 4));
    {  // (halves exchanged between lanes eight apart: whole 128-byte lines)
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
        const int row = p0 + 8 * u + (lane & 7);
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v[u]), rsrc, row < P && n < N ? (row * N + n) * 4 : kBufOOB, 0, 0);
      }
    }
  }
}

// Four rows of a lane's column as a row's four columns, among the four lanes of a quad: rows leave in 16 bytes.
__device__ __forceinline__ f32x4 quad_turn(f32x4 v) {
  const int lane = lane_id();
  auto swap = [](float mine, float other, bool second, auto ctrl) {  // (second: `mine` is handed over, else `other`)
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(second ? mine : other), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  const bool odd = lane & 1, high = lane & 2;
  constexpr std::integral_constant<int, 0xb1> by1{};  // lanes 1 0 3 2
  constexpr std::integral_constant<int, 0x4e> by2{};  // lanes 2 3 0 1
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const float t = swap(v[i], v[i + 1], odd, by1);
    v[i] = odd ? t : v[i];
    v[i + 1] = odd ? v[i + 1] : t;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float t = swap(v[i], v[i + 2], high, by2);
    v[i] = high ? t : v[i];
    v[i + 2] = high ? v[i + 2] : t;
  }
  return v;
}

// A column of 16 x 4 float32 accumulators (tokens 16 t + 4 g + r, value p0 + n) to rows of `step` bytes; WHOLE: in 16 bytes
// (a quarter of the stores).
template <bool WHOLE>
__device__ __forceinline__ void rows_out(const f32x4 (&acc)[4], __amdgpu_buffer_rsrc_t to, int step, int64_t rows, int p0, int P) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const int g = lane_id() >> 4, n = lane_id() & 15;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if constexpr (WHOLE) {
      const int tok = 16 * t + 4 * g + (n & 3), col = p0 + (n & 12);
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, quad_turn(acc[t])), to, tok < rows && col < P ? tok * step + col * 4 : kBufOOB, 0, 0);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int tok = 16 * t + 4 * g + r;
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(acc[t][r]), to, tok < rows && p0 + n < P ? tok * step + (p0 + n) * 4 : kBufOOB, 0, 0);
      }
    }
  }
}

// Eight elements of type E as their parts.
template <class E, int NI>
__device__ __forceinline__ void input_parts(const U8<E>& u, B8 (&f)[NI]) {
  if constexpr (std::is_same_v<E, BF16>) {
    f[0] = __builtin_bit_cast(B8, u);
  } else {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = ET<E>::to_f(u.e[e]);
    split8<NI>(v, f);
  }
}

// A loaded tile into LDS as NI tiles of parts, `part` elements apart; rows from `rows` on become zeros.
template <class T, int NI, class E, class L>
__device__ __forceinline__ void store_parts(const L& l, uint16_t* tile, int part, int rows, int tid) {
  constexpr int UPR = L::UPR, PER = L::PER, DROW = L::DROW;
  if (L::UNITS < DROW * UPR && tid >= L::UNITS) return;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int row = tid / UPR + i * DROW;
    U8<E> u;
    __builtin_memcpy(&u, &l.r[i][0], sizeof(u));
    if (row >= rows) zero_u8<E>(u);
    B8 f[NI];
    input_parts<E, NI>(u, f);
#pragma unroll
    for (int p = 0; p < NI; ++p)
      *reinterpret_cast<uint4*>(tile + p * part + l.at + i * DROW * T::STRIDE) = __builtin_bit_cast(uint4, f[p]);
  }
}

// The parts of a fragment from tiles `part` elements apart.
template <class T, int NI>
__device__ __forceinline__ void row_parts_t(const uint16_t* tile, int part, int row, int col, B8 (&f)[NI]) {
#pragma unroll
  for (int p = 0; p < NI; ++p) f[p] = row_frag_t<T, BF16>(tile + p * part, row, col);
}
template <class T, int NI>
__device__ __forceinline__ void col_parts(const uint16_t* tile, int part, int t0, int col, B8 (&f)[NI]) {
#pragma unroll
  for (int p = 0; p < NI; ++p) f[p] = col_frag<T, BF16>(tile + p * part, t0, col);
}

// A fragment's parts as delta_prep_kernel leaves them.
template <int NP>
__device__ __forceinline__ void stored_parts(const uint16_t* m, int frag, B8 (&f)[NP], int lane) {
#pragma unroll
  for (int p = 0; p < NP; ++p)
    f[p] = __builtin_bit_cast(B8, *reinterpret_cast<const uint4*>(m + (frag * NP + p) * kDFragElems + 8 * lane));
}

template <int NP>
__device__ __forceinline__ void stored_triangle(const uint16_t* m, B8 (&f)[kDFrags][NP], int lane) {
#pragma unroll
  for (int i = 0; i < kDFrags; ++i) stored_parts<NP>(m, i, f[i], lane);
}

int delta_check(const struct grm_hip_delta_args* u, const char* what, bool step);
DeltaArgs delta_args(const struct grm_hip_delta_args* u);
// The chunks' inverses and weights into a.work; `back`: in the reverse walk's form.
int launch_delta_prep(const DeltaArgs& a, int dtype, bool back, hipStream_t stream, const char* what);
// The parts' first states of part_state and part_map, for parts above two.
int launch_delta_join(const DeltaArgs& a, hipStream_t stream, const char* what);
// Time parts of the walk over C chunks and of its mirror, and a part's chunks.
int delta_time_parts(int64_t seqs, int64_t P, int64_t N, int64_t C, int dtype, bool mirror, int64_t* part_chunks);

// Host side: f(E, NK, VEC) with one of the compiled forms.
template <class F>
void delta_with_form(int dtype, int64_t N, bool vec, F f) {
  auto by_vec = [&](auto e, auto nk) {
    if (vec) f(e, nk, std::true_type{});
    else f(e, nk, std::false_type{});
  };
  auto by_width = [&](auto e) {
    if (N <= 64) by_vec(e, std::integral_constant<int, 64>{});
    else by_vec(e, std::integral_constant<int, 128>{});
  };
  if (dtype == GRM_HIP_BF16) by_width(BF16{});
  else if (dtype == GRM_HIP_F16) by_width(F16{});
  else by_width(F32{});
}

}  // namespace grmhip
