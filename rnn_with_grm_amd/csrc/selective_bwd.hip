// Gradients of the selective state scan, gfx950.
//
// Over a block of L tokens from state S at its start, with the adjoint G of the state at its end,
// c_i the summed log decays, E_ij = e^{c_i - c_j} (j <= i), K_ij = q_i . k_j and W_ij = dy_i . x_j:
//   dx_j = d_j (sum_i E_ij K_ij dy_i + e^{c_L - c_j} G k_j) + D dy_j
//   dq_i = sum_j E_ij d_j W_ij k_j + e^{c_i} S^T dy_i          summed over the heads of a group
//   dk_j = sum_i E_ij d_j W_ij q_i + d_j e^{c_L - c_j} G^T x_j  likewise
//   G'   = e^{c_L} G + sum_i e^{c_i} dy_i q_i^T                 the adjoint at the block's start
// and for the step sizes, with Q_ij = E_ij d_j K_ij W_ij, t1_i = e^{c_i} q_i . S^T dy_i and t2_j = e^{c_L - c_j} k_j . G^T x_j,
//   dl_t = sum_{j < t <= i} Q_ij + sum_{i >= t} t1_i + sum_{j < t} d_j t2_j + e^{c_L} <G, S>   (l_t = d_t A, the log decay)
//   dd_t = A dl_t + sum_i E_it K_it W_it + t2_t,   dA = sum_t d_t dl_t,   dD = sum_t W_tt
//
// Steps.  The forward has left S before every block; the reverse walk (selective_pass_kernel)
// leaves G behind every block, and selective_token_kernel every token's decays; then all blocks run side by
// side, one workgroup for a block and some of a group's heads, whose dk and dq it sums in registers.  It leaves the
// sums of Q, t1 and t2 by token, of which selective_steps_kernel makes the step sizes' gradients, one wave a head and block.
// Where more than one workgroup shares a group, their sums are added in a fixed order by a last
// kernel: no atomics, the same bits on every run.
//
// The step sizes' gradients stay float32: K and W are sums of exact products, and S and G enter t1 and t2 as three
// bfloat16 parts (24 bits; with two, 2^-17, each token's gradient was off by 4.5e-7 where it is now by 1.7e-7, for 25 us).
// dl_t is summed without taking large sums off each other (at selective_steps_kernel).
// dx, dk and dq are rounded to 16 bits in the end; their weights E K and E d W, and G where it meets k, are two bfloat16
// parts, which lose 2^-16 of a term (8 x 2048 tokens x 32 heads, forward and backward: 489 us, 494 with the signs in turn below; with one part,
// whose 2^-8 is seen in the outputs, 458).
#include <stdint.h>

#include "selective.h"

namespace grmhip {
namespace {

constexpr int kGradThreads = 512;

// A head's numbers by token, planes of LB in `tokens`: log2 decay from the block's start through the token in two
// floats, step size, e^c, e^{c_L - c}, and decays inside 16-token tiles: from the end of the tile before
// through the token, and from the token through its tile's end times the step size.
enum { HI, LO, DD, EC, EE, RB, TD, kPlanes };
// A head's sums by token that the step sizes' gradients are made of: its row of Q in earlier 16-token tiles, its row less
// its column inside its own tile, its column in later tiles, its row and its column in tiles that are not next to its
// own, t1, d t2, and du . x.
enum { ROW, TILE, COL, FAR_ROW, FAR_COL, T1, T2, DUX, kSums };

struct GradArgs {
  SelArgs s;              // the forward's inputs; states: S before every block
  const void* dy;         // [B, T, H, P]
  const float* adj;       // [B, nsave, H, P, N]: G behind every block
  float* tokens;          // [B, nsave, H, kPlanes, LB]
  float* diffs;           // [B, nsave, H * PT, shares, kSums, LB]
  float* dots;            // [B, nsave, H * PT, 8, 2]: <G, S> and sum W_jj, a part a wave
  void* dx;               // [B, T, H, P]
  void* dk;               // [B, T, G, N]
  void* dq;               // [B, T, G, N]
  void* dsteps;           // [B, T, H]
  float* rows_part;       // [splits][2][B, T, G, N] or null: dk and dq of each share of the heads
  float* head_part;       // [B * nsave, H, 3]: dA, dD and the step bias's gradient
  int splits;
};

template <class M, int NP>
struct GradLds {
  using S = SelShape<M>;
  using KT = SelTile<M, NP, true>;          // keys, queries, states: columns, and rows in 16-byte pieces
  using XT = SelTile<M, kSelRows, false>;   // values and their gradients: rows in 8-byte pieces
  static constexpr int LB = S::LB;
  static constexpr int SPARTS = S::kHalf ? 3 : 1;             // parts of S and G in LDS: two of their own,
  static constexpr int STATE = kSelRows * KT::STRIDE;
  static constexpr int OWN = S::kHalf ? 2 : 1;                 // the third where the values lay
  static_assert(SPARTS == OWN || STATE <= LB * XT::STRIDE, "the third part's room");
  static constexpr int TILES = LB * (2 * KT::STRIDE + 2 * XT::STRIDE) + OWN * STATE;
  static constexpr int TOK = LB / 16;                          // token tiles
  static constexpr int CS = 8 / TOK;                           // waves that share one, a share of the columns each
  static constexpr size_t bytes = TILES * sizeof(typename ET<M>::raw) + kPlanes * LB * sizeof(float);
  static_assert(bytes <= 160 * 1024, "one CU's LDS");
};

template <int ROT>
__device__ __forceinline__ float row_rot(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + ROT, 0xf, 0xf, true));
}
// Sum over the 16 lanes of a row, in all of them.
__device__ __forceinline__ float row_sum(float x) {
  x += row_rot<8>(x);
  x += row_rot<4>(x);
  x += row_rot<2>(x);
  x += row_rot<1>(x);
  return x;
}
// x of the lane ROT further in the row, 0 past its end.
template <int ROT>
__device__ __forceinline__ float dpp_shl(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x100 + ROT, 0xf, 0xf, true));
}
// x of the lane ROT before in the row, 0 past its start.
template <int ROT>
__device__ __forceinline__ float dpp_shr(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x110 + ROT, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_f32(float x, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}
// Sum over the four lane groups.
__device__ __forceinline__ float group_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

template <class E>
__device__ __forceinline__ void store_row4(typename ET<E>::raw* p, int left, bool vec, f32x4 v) {
  if (vec) {
    if (left > 0) store4_raw<E>(p, v);
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (r < left) p[r] = ET<E>::from_f(v[r]);
    }
  }
}

// A 64 x NP float32 state by 512 threads: from memory into registers (zeros outside [rows, N]), then into LDS as
// bfloat16 parts or as it is.
template <class M, int NP>
struct StateLoad {
  using KT = SelTile<M, NP, true>;
  static constexpr int PER = kSelRows * NP / 4 / kGradThreads, PARTS = GradLds<M, NP>::SPARTS;
  static constexpr int DROW = kGradThreads * 4 / NP;
  static_assert(PER >= 1 && PER * kGradThreads * 4 == kSelRows * NP, "states split evenly");
  f32x4 r[PER];
  __device__ __forceinline__ void load(const float* base, int rows, int N, int tid) {
    const __amdgpu_buffer_rsrc_t rsrc = make_rsrc(base, static_cast<uint32_t>((rows < kSelRows ? rows : kSelRows) * N * 4));
    const int row = tid / (NP / 4), n = tid % (NP / 4) * 4;
    if ((N & 3) == 0) {
      // (The whole offset in the vector register, where the range check sees it: rows past the state read zeros.)
      const uint32_t off = n < N ? (row * N + n) * 4 : kBufOOB;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        r[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, off + static_cast<uint32_t>(i * DROW * N * 4), 0, 0));
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          r[i][e] = buf_load1<F32>(rsrc, n + e < N ? ((row + i * DROW) * N + n + e) * 4 : kBufOOB);
      }
    }
  }
  // Parts FIRST to LAST - 1 of `sign` (1 or -1) times the state, part 2 into `third`.
  template <int FIRST, int LAST>
  __device__ __forceinline__ void store(typename ET<M>::raw* tile, typename ET<M>::raw* third, int tid, float sign) const {
    const int at = KT::at(tid / (NP / 4), tid % (NP / 4) * 4);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      f32x4 rest = r[i] * sign;
#pragma unroll
      for (int s = 0; s < PARTS && s < LAST; ++s) {
        if (s >= FIRST) store4_raw<M>((s == 2 ? third : tile + s * GradLds<M, NP>::STATE) + at + i * DROW * KT::STRIDE, rest);
        if (s + 1 < PARTS) {
#pragma unroll
          for (int e = 0; e < 4; ++e) rest[e] -= ET<M>::to_f(ET<M>::from_f(rest[e]));
        }
      }
    }
  }
};

// One wave a head and block: every token's decays (PL tokens a lane).
template <class E, int LB>
__global__ __launch_bounds__(256) void selective_token_kernel(GradArgs a) {
  constexpr int PL = LB / 64;
  const SelArgs& f = a.s;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (id >= static_cast<int64_t>(f.B) * f.nsave * f.H) return;
  const int h = static_cast<int>(id % f.H), lane = lane_id();
  const int64_t blk = id / f.H % f.nsave, t0 = blk * LB;
  const int b = static_cast<int>(id / f.H / f.nsave);
  const int64_t len = sel_length(f, b);
  if (t0 >= len) return;
  const float rate = f.rates[h];
  float d[PL];
  double cum[PL], sum = 0.0;
#pragma unroll
  for (int k = 0; k < PL; ++k) {
    const int64_t t = t0 + lane * PL + k;
    d[k] = t < len ? step_size(f, raw_step<E>(f, b, t, h)) : 0.f;
    double l = t < len ? static_cast<double>(d[k]) * static_cast<double>(rate) : 0.0;
    l = l < -200.0 ? -200.0 : l;
    sum += l * 1.4426950408889634;
    cum[k] = sum;
  }
  const double scan = wave_prefix(sum), before = scan - sum, total = lane_value(scan, 63);
#pragma unroll
  for (int k = 0; k < PL; ++k) cum[k] += before;
  constexpr int LPT = 16 / PL;  // lanes of a tile
  const int first = lane / LPT * LPT;
  const double tile_end = __shfl(cum[PL - 1], first + LPT - 1), up = __shfl(cum[PL - 1], first > 0 ? first - 1 : 0);
  const double tile_start = first > 0 ? up : 0.0;
  float* o = a.tokens + id * kPlanes * LB + lane * PL;
#pragma unroll
  for (int k = 0; k < PL; ++k) {
    const float top = static_cast<float>(cum[k]);
    o[HI * LB + k] = top;
    o[LO * LB + k] = static_cast<float>(cum[k] - top);
    o[DD * LB + k] = d[k];
    o[EC * LB + k] = exp2_d(cum[k]);
    o[EE * LB + k] = exp2_d(total - cum[k]);
    o[RB * LB + k] = exp2_d(cum[k] - tile_start);
    o[TD * LB + k] = d[k] * exp2_d(tile_end - cum[k]);
  }
}

// Sum over the later (earlier) lanes of this lane's group of W, W = 8 or 16: shifted first, so that nothing is taken off again.
template <int W, int ROT>
__device__ __forceinline__ float later_lane(float x) {
  const float y = dpp_shl<ROT>(x);
  return (lane_id() & (W - 1)) + ROT < W ? y : 0.f;
}
template <int W, int ROT>
__device__ __forceinline__ float earlier_lane(float x) {
  const float y = dpp_shr<ROT>(x);
  return (lane_id() & (W - 1)) >= ROT ? y : 0.f;
}
template <int W>
__device__ __forceinline__ float sum_later(float x) {
  x = later_lane<W, 1>(x);
  x += later_lane<W, 1>(x);
  x += later_lane<W, 2>(x);
  x += later_lane<W, 4>(x);
  if constexpr (W > 8) x += later_lane<W, 8>(x);
  return x;
}
template <int W>
__device__ __forceinline__ float sum_earlier(float x) {
  x = earlier_lane<W, 1>(x);
  x += earlier_lane<W, 1>(x);
  x += earlier_lane<W, 2>(x);
  x += earlier_lane<W, 4>(x);
  if constexpr (W > 8) x += earlier_lane<W, 8>(x);
  return x;
}

// One wave a head and block: the step sizes' gradients, dd_t = A dl_t + du_t . x_t.  dl_t could be summed as rows less
// columns of Q from t on, but where the decay is strong the pairs across t are few and small, and their sum would drown in
// the rounding of all later pairs.  So they are taken by where they lie.  Of the pairs (i, j) across token t of tile I
//   both in I:              rows less columns inside the tile, from t to its end;
//   i in I, j before it:    rows in earlier tiles, from t to the tile's end;     i behind I, j in it: columns before t;
//   i behind I, j before:   a difference again, but of whole tiles' sums over pairs with a tile between them.
// (As rows less columns throughout, the sums for the rates and the step bias, which cancel over the tokens, were off by
// 3.5e-6 of their norm in bf16, 1.4e-6 in float32; now by 1e-7 to 5e-7.)
template <class E, int LB, int CS>
__global__ __launch_bounds__(256) void selective_steps_kernel(GradArgs a) {
  constexpr int PL = LB / 64;
  const SelArgs& f = a.s;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (id >= static_cast<int64_t>(f.B) * f.nsave * f.H) return;
  const int h = static_cast<int>(id % f.H), lane = lane_id();
  const int64_t blk = id / f.H % f.nsave, t0 = blk * LB;
  const int b = static_cast<int>(id / f.H / f.nsave);
  const int64_t len = sel_length(f, b);
  float da = 0.f, db = 0.f, dskip = 0.f, dz[PL];
#pragma unroll
  for (int k = 0; k < PL; ++k) dz[k] = 0.f;
  if (t0 < len) {
    const float* tk = a.tokens + id * kPlanes * LB + lane * PL;
    constexpr int W = 16 / PL, TOK = LB / 16;  // lanes of a tile, tiles
    float sums[kSums][PL], d[PL], gdot = 0.f;
#pragma unroll
    for (int k = 0; k < PL; ++k) {
      d[k] = tk[DD * LB + k];
#pragma unroll
      for (int n = 0; n < kSums; ++n) sums[n][k] = 0.f;
    }
    for (int pt = 0; pt < f.PT; ++pt) {
      const int64_t hp = id * f.PT + pt;
#pragma unroll
      for (int c = 0; c < CS; ++c) {
#pragma unroll
        for (int n = 0; n < kSums; ++n) {
#pragma unroll
          for (int k = 0; k < PL; ++k) sums[n][k] += a.diffs[((hp * CS + c) * kSums + n) * LB + lane * PL + k];
        }
      }
      const float2 v = *reinterpret_cast<const float2*>(a.dots + (hp * 8 + (lane & 7)) * 2);
      gdot += lane < 8 ? v.x : 0.f;
      dskip += lane < 8 ? v.y : 0.f;
    }
    const float total = lane_f32(tk[HI * LB + PL - 1], 63), rest = lane_f32(tk[LO * LB + PL - 1], 63);
    gdot = group_sum(row_sum(gdot));
    dskip = group_sum(row_sum(dskip));
    // From each token to its tile's end (t1 too), and before it in its tile; then a tile's own totals.
    float rows = 0.f, both = 0.f, t1 = 0.f, cols = 0.f, t2 = 0.f, far_rows = 0.f, far_cols = 0.f, in_tile[PL];
#pragma unroll
    for (int k = 0; k < PL; ++k) {
      far_rows += sums[FAR_ROW][k];
      far_cols += sums[FAR_COL][k];
      cols += sums[COL][k];
      t2 += sums[T2][k];
    }
#pragma unroll
    for (int k = PL - 1; k >= 0; --k) {
      rows += sums[ROW][k];
      both += sums[TILE][k];
      t1 += sums[T1][k];
      in_tile[k] = (rows + both) + t1;
    }
    const float rows_later = sum_later<W>(rows), both_later = sum_later<W>(both), t1_later = sum_later<W>(t1);
    const float cols_before = sum_earlier<W>(cols), t2_before = sum_earlier<W>(t2);
    const float rows_tile = far_rows + sum_later<W>(far_rows), t1_tile = t1 + t1_later;        // in a tile's first lane
    const float cols_tile = far_cols + sum_earlier<W>(far_cols), t2_tile = t2 + t2_before;     // in its last
    float across = 0.f, others = 0.f, crossing = 0.f;
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
      // Pairs round tile i: those round i - 1, less the rows of i, and the columns of i - 1.
      if (i > 0) crossing += lane_f32(cols_tile, i * W - 1) - lane_f32(rows_tile, i * W);
      across = lane / W == i ? crossing : across;
      const float behind = lane_f32(t1_tile, i * W), ahead = lane_f32(t2_tile, i * W + W - 1);
      others += lane / W < i ? behind : lane / W > i ? ahead : 0.f;
    }
    const float end = exp2_f(total) * exp2_f(rest) * gdot;
    const float all = ((rows_later + both_later) + (t1_later + others)) + (across + end);
    float before = cols_before + t2_before;
    const float rate = f.rates[h];
#pragma unroll
    for (int k = 0; k < PL; ++k) {
      const int64_t t = t0 + lane * PL + k;
      const float dl = in_tile[k] + before + all;
      before += sums[COL][k] + sums[T2][k];
      if (t < len) {
        float slope = 1.f;
        if (f.softplus) {
          const float z = raw_step<E>(f, b, t, h);
          slope = z > 20.f ? 1.f : __builtin_amdgcn_rcpf(1.f + __expf(-z));
        }
        dz[k] = fmaf(rate, dl, sums[DUX][k]) * slope;
        da = fmaf(d[k], dl, da);
        db += dz[k];
      }
    }
    da = group_sum(row_sum(da));
    db = group_sum(row_sum(db));
  }
#pragma unroll
  for (int k = 0; k < PL; ++k) {
    const int64_t t = t0 + lane * PL + k;
    if (t < f.T) st_state<E>(a.dsteps, (b * f.T + t) * f.H + h, f.steps_f32 != 0, dz[k]);
  }
  if (lane < 3) a.head_part[id * 3 + lane] = lane == 0 ? da : lane == 1 ? dskip : db;
}

template <class E, class M, int NP, bool VEC>
__global__ __launch_bounds__(kGradThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void selective_grad_kernel(GradArgs a) {
  using S = SelShape<M>;
  using Lds = GradLds<M, NP>;
  using raw = typename ET<M>::raw;
  using eraw = typename ET<E>::raw;
  using KT = typename Lds::KT;
  using XT = typename Lds::XT;
  constexpr int LB = S::LB, TOK = Lds::TOK, CS = Lds::CS, SP = Lds::SPARTS;
  constexpr int NK = NP / 32, NT = NP / 16 / CS, PW = kSelRows / 16 / CS;
  constexpr int WP = Lds::OWN;  // parts of the weights E K and E d W, and of G where it meets k
  constexpr int NPL = (kPlanes * LB + kGradThreads - 1) / kGradThreads;
  extern __shared__ __align__(16) unsigned char smem[];
  raw* kt = reinterpret_cast<raw*>(smem);
  raw* qt = kt + LB * KT::STRIDE;
  raw* xt = qt + LB * KT::STRIDE;
  raw* yt = xt + LB * XT::STRIDE;
  raw* st = yt + LB * XT::STRIDE;
  float* sc = reinterpret_cast<float*>(st + Lds::OWN * Lds::STATE);

  const SelArgs& f = a.s;
  uint32_t v = xcd_order(blockIdx.x, gridDim.x);
  const int split = static_cast<int>(v % a.splits);
  v /= a.splits;
  const int gi = static_cast<int>(v % f.G);
  v /= f.G;
  const int blk = static_cast<int>(v % f.nsave), b = static_cast<int>(v / f.nsave);
  const int tid = static_cast<int>(threadIdx.x);
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tile = wave % TOK, cs = wave / TOK;
  const int64_t t0 = static_cast<int64_t>(blk) * LB;
  const int live = static_cast<int>(max_i64(0, min_i64(sel_length(f, b) - t0, LB)));
  const int in_block = static_cast<int>(min_i64(LB, f.T - t0));
  const bool nvec = VEC && (f.N & 3) == 0, pvec = VEC && (f.P & 3) == 0;
  const int heads = f.H / f.G * f.PT;  // (head, value tile) pairs of the group
  const int h_lo = static_cast<int>(static_cast<int64_t>(heads) * split / a.splits),
            h_hi = static_cast<int>(static_cast<int64_t>(heads) * (split + 1) / a.splits);
  const int64_t row_b = static_cast<int64_t>(b) * f.T + t0;  // the block's first token
  const int64_t blocks = static_cast<int64_t>(b) * f.nsave + blk;
  int h = gi * (f.H / f.G) + h_lo / f.PT, pt = h_lo % f.PT;  // the head and its value tile

  // The bf16 matrix products round a sum down a little more often than up (by 0.3% of their error's spread; the float32 ones do
  // not).  The step sizes' gradients add up thousands of W and S^T dy and G^T x times keys, queries and values that are mostly
  // of one sign, and cancel, so that in the sums for `rates` this was what was seen of their error: 7e-7 to 1.6e-6 of their norm, now
  // 1e-7 to 5e-7.  So in every other block x and S, and with them W, S^T dy and G^T x, carry the other sign.
  const float sg = S::kHalf && ((b + blk) & 1) ? -1.f : 1.f;

  f32x4 dk[NT], dq[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) dk[i] = dq[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (live == 0) {  // behind the sequence's length: zeros
    for (int hp = h_lo; hp < h_hi; ++hp) {
      const int p0 = pt * kSelRows, cols = f.P - p0 < kSelRows ? f.P - p0 : kSelRows, lane = lane_id();
      eraw* dxp = static_cast<eraw*>(a.dx) + (row_b * f.H + h) * f.P + p0;
      for (int t = wave; t < in_block; t += 8) {
        if (lane < cols) dxp[static_cast<int64_t>(t) * f.H * f.P + lane] = ET<E>::from_f(0.f);
      }
      if (++pt == f.PT) pt = 0, ++h;
    }
  } else {
    TileLoad<E, XT, M, VEC, LB, kSelRows, kGradThreads> xr, yr;
    float pr[NPL];
    auto ask_rows = [&](int hn, int pn, int tid) {
      const int p0 = pn * kSelRows, cols = f.P - p0 < kSelRows ? f.P - p0 : kSelRows;
      xr.init(f.vt, cols, tid);
      xr.load(static_cast<const eraw*>(f.values) + b * f.vb + t0 * f.vt + hn * f.P + p0, live, tid);
      yr.init(static_cast<int64_t>(f.H) * f.P, cols, tid);
      yr.load(static_cast<const eraw*>(a.dy) + (row_b * f.H + hn) * f.P + p0, live, tid);
      const __amdgpu_buffer_rsrc_t rsrc = make_rsrc(a.tokens + (blocks * f.H + hn) * kPlanes * LB, kPlanes * LB * 4);
#pragma unroll
      for (int i = 0; i < NPL; ++i) pr[i] = buf_load1<F32>(rsrc, (tid + i * kGradThreads) * 4);
    };
    ask_rows(h, pt, tid);
    {
      TileLoad<E, KT, M, VEC, LB, NP, kGradThreads> r;
      r.init(f.kt, f.N, tid);
      r.load(static_cast<const eraw*>(f.keys) + b * f.kb + t0 * f.kt + gi * f.N, live, tid);
      r.store(kt, tid);
      r.init(f.qt, f.N, tid);
      r.load(static_cast<const eraw*>(f.queries) + b * f.qb + t0 * f.qt + gi * f.N, live, tid);
      r.store(qt, tid);
    }

    for (int hp = h_lo; hp < h_hi; ++hp) {
      // The lane's number anew for every head, so that the hundreds of LDS addresses made from it are not kept in
      // registers from head to head.
      int lane = lane_id();
      asm volatile("" : "+v"(lane));
      const int tid = wave * 64 + lane;
      const int g = lane >> 4, n16 = lane & 15, tok = tile * 16 + n16;  // this lane's token in both orders
      const int p0 = pt * kSelRows, pw = f.P - p0;
      const float skip = f.skip == nullptr ? 0.f : f.skip[h];
      const int64_t sat = ((blocks * f.H + h) * f.P + p0) * f.N;
      const int64_t pair = (blocks * f.H + h) * f.PT + pt;
      xr.at = yr.at = XT::at(tid / (kSelRows / 8), tid % (kSelRows / 8) * 8);
      xr.store(xt, tid, sg < 0.f);
      yr.store(yt, tid);
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        if (kPlanes * LB % kGradThreads == 0 || tid + i * kGradThreads < kPlanes * LB) sc[tid + i * kGradThreads] = pr[i];
      }
      StateLoad<M, NP> sr, gr;
      sr.load(f.states + sat, pw, f.N, tid);
      __syncthreads();

      // Columns j of this wave's tile: dx and dk from the rows i >= j, two tiles of rows at a time.
      f32x4 dx[PW];
#pragma unroll
      for (int p = 0; p < PW; ++p) dx[p] = f32x4{0.f, 0.f, 0.f, 0.f};
      Frag8<M> xf[2], yf[2], kf[NK];
#pragma unroll
      for (int k = 0; k < 2; ++k) xf[k] = row_frag_t<XT, M>(xt, tile * 16, k * 32, lane);
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) kf[kk] = row_frag<KT, M>(kt, tile * 16, kk * 32, lane);
      const float hj = sc[HI * LB + tok], lj = sc[LO * LB + tok], djs = sg * sc[DD * LB + tok];
      float near = 0.f, next = 0.f, far = 0.f, kw_diag = 0.f, w_diag = 0.f;
      auto columns = [&](int dp, auto diag) {
        // The second tile past the block is the first again, with weights of zero.
        const int i0 = tile + dp, i1 = i0 + 1 < TOK ? i0 + 1 : i0;
        f32x4 ek[2], ew[2], w[2], k2[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          w[u] = k2[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < 2; ++k) w[u] = mfma8(row_frag_t<XT, M>(yt, (u ? i1 : i0) * 16, k * 32, lane), xf[k], w[u]);
#pragma unroll
          for (int kk = 0; kk < NK; ++kk) k2[u] = mfma8(row_frag<KT, M>(qt, (u ? i1 : i0) * 16, kk * 32, lane), kf[kk], k2[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int it = u ? i1 : i0, ti = it * 16 + 4 * g;
          if (decltype(diag)::value && u == 0) {  // on the diagonal, pair by pair
            const f32x4 hv = *reinterpret_cast<const f32x4*>(sc + HI * LB + ti), lv = *reinterpret_cast<const f32x4*>(sc + LO * LB + ti);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const bool in = ti + r >= tok, own = ti + r == tok;
              const float e = exp2_f(in ? (hv[r] - hj) + (lv[r] - lj) : -INFINITY), wr = in ? w[u][r] : 0.f;
              ek[u][r] = e * (in ? k2[u][r] : 0.f);
              ew[u][r] = e * djs * wr;
              near = fmaf(ek[u][r], own ? 0.f : wr, near);
              kw_diag = fmaf(ek[u][r], own ? wr : 0.f, kw_diag);
              w_diag += own ? wr : 0.f;
            }
          } else {  // e^{c_i - c_j} through the end of the tile before i's: one exponential a lane, one product a pair
            const bool on = u == 0 || i1 != i0;
            const f32x4 rv = *reinterpret_cast<const f32x4*>(sc + RB * LB + ti);
            const int before = on ? it * 16 - 1 : 0;
            const float c = on ? exp2_f((sc[HI * LB + before] - hj) + (sc[LO * LB + before] - lj)) : 0.f, cd = c * djs;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              ek[u][r] = rv[r] * c * k2[u][r];
              ew[u][r] = rv[r] * cd * w[u][r];
              float& to = decltype(diag)::value ? next : far;
              to = fmaf(ek[u][r], w[u][r], to);
            }
          }
        }
        Frag8<M> ekf[WP], ewf[WP];
        split_pair<M>(ek[0], ek[1], ekf);
#pragma unroll
        for (int p = 0; p < PW; ++p) {
          const Frag8<M> yc = col_frag2<XT, M>(yt, i0 * 16, i1 * 16, (cs * PW + p) * 16, lane);
#pragma unroll
          for (int s = WP - 1; s >= 0; --s) dx[p] = mfma8(yc, ekf[s], dx[p]);
          if (p & 1) hold_order();
        }
        hold_order();
        split_pair<M>(ew[0], ew[1], ewf);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const Frag8<M> qc = col_frag2<KT, M>(qt, i0 * 16, i1 * 16, (cs * NT + nt) * 16, lane);
#pragma unroll
          for (int s = WP - 1; s >= 0; --s) dk[nt] = mfma8(qc, ewf[s], dk[nt]);
        }
      };
      columns(0, std::true_type{});
#pragma unroll 1
      for (int dp = 2; dp < TOK - tile; dp += 2) columns(dp, std::false_type{});

      // What the step sizes' gradients want of this wave's tokens, as soon as it is there: little is held meanwhile.
      const __amdgpu_buffer_rsrc_t dfr = make_rsrc(a.diffs + (pair * CS + cs) * LB * kSums, LB * kSums * 4);
      auto by_token = [&](int what, float x) { buf_store1<F32>(dfr, g == 0 ? (what * LB + tok) * 4 : kBufOOB, x); };
      const __amdgpu_buffer_rsrc_t dtr = make_rsrc(a.dots + (pair * 8 + wave) * 2, 8);
      const bool one = cs == 0;
      float near_col, dux;
      {
        const float nr = group_sum(near), far_col = group_sum(far), fr = group_sum(next) + far_col;
        const float wsum = group_sum(row_sum(sg * w_diag));
        near_col = djs * nr;
        dux = one ? sg * (group_sum(kw_diag) + (nr + fr)) : 0.f;
        by_token(COL, one ? djs * fr : 0.f);
        by_token(FAR_COL, one ? djs * far_col : 0.f);
        buf_store1<F32>(dtr, lane == 0 ? 4 : kBufOOB, one ? wsum : 0.f);
      }

      // Rows i of this wave's tile: dq from the columns j <= i, and the rows' sums.
      const float e_i = sg * sc[EC * LB + tok];
      float row_near = 0.f, row_next = 0.f, row_far = 0.f;
      Frag8<M> qf[NK];
#pragma unroll
      for (int k = 0; k < 2; ++k) yf[k] = row_frag_t<XT, M>(yt, tile * 16, k * 32, lane);
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) qf[kk] = row_frag<KT, M>(qt, tile * 16, kk * 32, lane);
      gr.load(a.adj + sat, pw, f.N, tid);
      auto rows = [&](int dp, auto diag) {
        const int j0 = tile - dp, j1 = j0 > 0 ? j0 - 1 : 0;
        f32x4 ew[2], w[2], k2[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          w[u] = k2[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < 2; ++k) w[u] = mfma8(row_frag_t<XT, M>(xt, (u ? j1 : j0) * 16, k * 32, lane), yf[k], w[u]);
#pragma unroll
          for (int kk = 0; kk < NK; ++kk) k2[u] = mfma8(row_frag<KT, M>(kt, (u ? j1 : j0) * 16, kk * 32, lane), qf[kk], k2[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int jt = u ? j1 : j0, tj = jt * 16 + 4 * g;
          if (decltype(diag)::value && u == 0) {
            const f32x4 hv = *reinterpret_cast<const f32x4*>(sc + HI * LB + tj), lv = *reinterpret_cast<const f32x4*>(sc + LO * LB + tj),
                        dv = *reinterpret_cast<const f32x4*>(sc + DD * LB + tj);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const bool in = tj + r <= tok;
              ew[u][r] = exp2_f(in ? (hj - hv[r]) + (lj - lv[r]) : -INFINITY) * (in ? sg * dv[r] * w[u][r] : 0.f);
              row_near = fmaf(ew[u][r], tj + r < tok ? k2[u][r] : 0.f, row_near);
            }
          } else {  // through the end of j's tile
            const bool on = u == 0 || j0 > 0;
            const f32x4 dv = *reinterpret_cast<const f32x4*>(sc + TD * LB + tj);
            const float c = on ? sg * exp2_f((hj - sc[HI * LB + jt * 16 + 15]) + (lj - sc[LO * LB + jt * 16 + 15])) : 0.f;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              ew[u][r] = c * dv[r] * w[u][r];
              float& to = decltype(diag)::value ? row_next : row_far;
              to = fmaf(ew[u][r], k2[u][r], to);
            }
          }
        }
        Frag8<M> ewf[WP];
        split_pair<M>(ew[0], ew[1], ewf);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const Frag8<M> kc = col_frag2<KT, M>(kt, j0 * 16, j1 * 16, (cs * NT + nt) * 16, lane);
#pragma unroll
          for (int s = WP - 1; s >= 0; --s) dq[nt] = mfma8(kc, ewf[s], dq[nt]);
        }
      };
      rows(0, std::true_type{});
#pragma unroll 1
      for (int dp = 2; dp <= tile; dp += 2) rows(dp, std::false_type{});
      sr.template store<0, 2>(st, xt, tid, sg);
#pragma unroll
      for (int k = 0; k < 2; ++k) xf[k] = row_frag_t<XT, M>(xt, tile * 16, k * 32, lane);
      const float far_row = group_sum(row_far);
      by_token(ROW, one ? group_sum(row_next) + far_row : 0.f);
      by_token(FAR_ROW, one ? far_row : 0.f);
      by_token(TILE, one ? group_sum(row_near) - near_col : 0.f);
      __syncthreads();
      if constexpr (SP == 3) {  // the values' fragments are in registers: their room is free
        sr.template store<2, 3>(st, xt, tid, sg);
        __syncthreads();
      }

      // From the state: dq.
      float dot1 = 0.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        f32x4 r = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = SP - 1; s >= 0; --s) {
#pragma unroll
          for (int k = 0; k < 2; ++k) r = mfma8(col_frag<KT, M>(s == 2 ? xt : st + s * Lds::STATE, k * 32, (cs * NT + nt) * 16, lane), yf[k], r);
        }
        const f32x4 qv = lds_row4<M>(qt + KT::at(tok, (cs * NT + nt) * 16 + 4 * g));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          dot1 = fmaf(qv[e], r[e], dot1);
          dq[nt][e] = fmaf(e_i, r[e], dq[nt][e]);
        }
        if (nt & 1) hold_order();
      }
      by_token(T1, e_i * group_sum(dot1));
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < StateLoad<M, NP>::PER; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) dot = fmaf(gr.r[i][e], sr.r[i][e], dot);
      }
      dot = group_sum(row_sum(dot));
      __syncthreads();
      gr.template store<0, 3>(st, xt, tid, 1.f);
      const bool wrap = pt + 1 == f.PT;
      const int hn = h + (wrap ? 1 : 0), pn = wrap ? 0 : pt + 1;
      if (hp + 1 < h_hi) ask_rows(hn, pn, tid);
      __syncthreads();

      // From the adjoint: dk and dx.
      const float e_t = sc[EE * LB + tok];
      float dot2 = 0.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        f32x4 r = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = SP - 1; s >= 0; --s) {
#pragma unroll
          for (int k = 0; k < 2; ++k) r = mfma8(col_frag<KT, M>(s == 2 ? xt : st + s * Lds::STATE, k * 32, (cs * NT + nt) * 16, lane), xf[k], r);
        }
        const f32x4 kv = lds_row4<M>(kt + KT::at(tok, (cs * NT + nt) * 16 + 4 * g));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          dot2 = fmaf(kv[e], r[e], dot2);
          dk[nt][e] = fmaf(djs * e_t, r[e], dk[nt][e]);
        }
        if (nt & 1) hold_order();
      }
      {
        // (Buffer stores: with no branch round them the compiler knows how many stand behind the next head's loads.)
        const int64_t wide = static_cast<int64_t>(f.H) * f.P;
        const __amdgpu_buffer_rsrc_t dxr = make_rsrc(static_cast<eraw*>(a.dx) + row_b * wide + h * f.P + p0, 0x7fffff00u);
        const int dx_at = tok * static_cast<int>(wide);
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) kf[kk] = row_frag<KT, M>(kt, tile * 16, kk * 32, lane);
        const float dj = sg * djs;
#pragma unroll
        for (int p = 0; p < PW; ++p) {
          f32x4 u = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = WP - 1; s >= 0; --s) {
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) u = mfma8(row_frag<KT, M>(st + s * Lds::STATE, (cs * PW + p) * 16, kk * 32, lane), kf[kk], u);
          }
          const int c = (cs * PW + p) * 16 + 4 * g;
          const f32x4 yv = lds_row4<M>(yt + XT::at(tok, c));
          f32x4 o;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = tok < live ? fmaf(dj, fmaf(e_t, u[e], dx[p][e]), skip * yv[e]) : 0.f;
          out4<E>(dxr, dx_at + c, tok < in_block ? pw - c : 0, pvec, o);
        }
      }
      const float s2 = sg * e_t * group_sum(dot2);
      by_token(T2, sg * djs * s2);
      by_token(DUX, dux + s2);
      buf_store1<F32>(dtr, lane == 0 ? 0 : kBufOOB, dot);
      __syncthreads();
      h = hn;
      pt = pn;
    }
  }

  // dk and dq of this workgroup's heads.
  const int lane = lane_id(), g = lane >> 4, tok = tile * 16 + (lane & 15);
  const int64_t all = static_cast<int64_t>(f.B) * f.T * f.G * f.N;
  const int64_t at = (row_b + tok) * f.G * f.N + static_cast<int64_t>(gi) * f.N;
  if (tok < in_block) {
    const bool on = tok < live;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int c = (cs * NT + nt) * 16 + 4 * g;
      const f32x4 none = {0.f, 0.f, 0.f, 0.f}, ko = on ? dk[nt] : none, qo = on ? dq[nt] : none;
      if (a.rows_part != nullptr) {
        float* p = a.rows_part + static_cast<int64_t>(split) * 2 * all + at + c;
        store_row4<F32>(p, f.N - c, (f.N & 3) == 0, ko);
        store_row4<F32>(p + all, f.N - c, (f.N & 3) == 0, qo);
      } else {
        store_row4<E>(static_cast<eraw*>(a.dk) + at + c, f.N - c, nvec, ko);
        store_row4<E>(static_cast<eraw*>(a.dq) + at + c, f.N - c, nvec, qo);
      }
    }
  }
}

// The first blocks: dk and dq as the sums of their shares, in order (n elements each, `parts` shares of both).  The
// last H blocks: dA, dD and the step bias's gradient of a head, its blocks' sums in a fixed order.
template <class E>
__global__ __launch_bounds__(256) void selective_sum_kernel(const float* part, int parts, void* dk, void* dq, int64_t n,
                                                            const float* heads, int64_t blocks, int H, float* da, float* dskip,
                                                            float* dbias) {
  const int tid = static_cast<int>(threadIdx.x), row_blocks = static_cast<int>(gridDim.x) - H;
  if (static_cast<int>(blockIdx.x) < row_blocks) {
    const int64_t step = static_cast<int64_t>(row_blocks) * 256;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + tid; i < 2 * n; i += step) {
      float s = part[i];
      for (int p = 1; p < parts; ++p) s += part[p * 2 * n + i];
      if (i < n) st_state<E>(dk, i, false, s);
      else st_state<E>(dq, i - n, false, s);
    }
    return;
  }
  __shared__ float sums[3][4];
  const int h = static_cast<int>(blockIdx.x) - row_blocks;
  float s[3] = {0.f, 0.f, 0.f};
  for (int64_t i = tid; i < blocks; i += 256) {
    const float* p = heads + (i * H + h) * 3;
#pragma unroll
    for (int k = 0; k < 3; ++k) s[k] += p[k];
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const float x = group_sum(row_sum(s[k]));
    if ((tid & 63) == 0) sums[k][tid >> 6] = x;
  }
  __syncthreads();
  if (tid == 0) {
    float* out[3] = {da, dskip, dbias};
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      if (out[k] != nullptr) out[k][h] = (sums[k][0] + sums[k][1]) + (sums[k][2] + sums[k][3]);
    }
  }
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Workspace: the adjoint behind every block, its walk's parts, the tokens' numbers and the shares' sums.
struct BwdPlan {
  int64_t nsave, part_tokens, wgs;
  int parts, splits, PT;
  int64_t adj, part_state, part_log, tokens, diffs, dots, rows, heads, bytes;  // byte offsets
};

BwdPlan bwd_plan(int64_t B, int64_t T, int64_t H, int64_t P, int64_t G, int64_t N, int dtype) {
  BwdPlan p{};
  auto up = [](int64_t n) { return sel_ceil(n, 256) * 256; };
  const int64_t LB = sel_block(dtype), CS = 128 / LB;
  p.PT = static_cast<int>(sel_ceil(P, kSelRows));
  p.nsave = sel_ceil(T, LB);
  p.parts = sel_parts(B * H * p.PT, T, dtype, &p.part_tokens);
  // A workgroup for each of 256 CUs; the heads of a group are shared no further, since every share reads
  // the keys and queries and writes a float32 copy of dk and dq (selective_grad_kernel at 4 x 1000 float32 tokens x 8
  // heads in 2 groups: 39 us in two shares, 66 us in one).
  p.wgs = B * p.nsave * G;
  const int64_t heads = H / G * p.PT;
  int64_t splits = p.wgs > 0 ? sel_ceil(256, p.wgs) : 1;
  if (splits > heads) splits = heads;
  p.splits = static_cast<int>(splits);
  const int64_t state = H * P * N * 4, pairs = B * p.nsave * H * p.PT;
  int64_t at = 0;
  p.adj = at; at += up(B * p.nsave * state);
  p.part_state = at; at += p.parts > 1 ? up(p.parts * B * state) : 0;
  p.part_log = at; at += p.parts > 1 ? up(p.parts * B * H * 8) : 0;
  p.tokens = at; at += up(B * p.nsave * H * kPlanes * LB * 4);
  p.diffs = at; at += up(pairs * CS * LB * kSums * 4);
  p.dots = at; at += up(pairs * 16 * 4);
  p.rows = at; at += p.splits > 1 ? up(p.splits * 2 * B * T * G * N * 4) : 0;
  p.heads = at; at += up(B * p.nsave * H * 12);
  p.bytes = at;
  return p;
}

}  // namespace
}  // namespace grmhip

using namespace grmhip;

extern "C" int64_t grm_hip_selective_scan_bwd_workspace(int64_t batch, int64_t seq_len, int64_t heads, int64_t value_dim,
                                                        int64_t groups, int64_t key_dim, int dtype) {
  if (batch <= 0 || seq_len < 0 || heads <= 0 || value_dim <= 0 || groups <= 0 || heads % groups != 0 || key_dim <= 0 ||
      dtype < 0 || dtype > 2)
    return 0;
  return bwd_plan(batch, seq_len, heads, value_dim, groups, key_dim, dtype).bytes;
}

extern "C" int grm_hip_selective_scan_bwd(const grm_hip_selective_args* u, const float* states, const void* grad_hidden,
                                          const float* grad_memory_out, void* grad_keys, void* grad_values,
                                          void* grad_queries, void* grad_steps, float* grad_rates, float* grad_memory,
                                          float* grad_skip, float* grad_step_bias, void* workspace,
                                          int64_t workspace_bytes, void* stream) {
  const char* what = "selective_scan backward";
  if (int rc = sel_check(u, what)) return rc;
  if (grad_rates == nullptr || (u->batch > 0 && grad_memory == nullptr) || !aligned(states) || !aligned(grad_memory_out) ||
      !aligned(grad_memory) ||
      (u->batch > 0 && u->seq_len > 0 &&
       (states == nullptr || grad_hidden == nullptr || grad_keys == nullptr || grad_values == nullptr ||
        grad_queries == nullptr || grad_steps == nullptr))) {
    set_error("%s: every gradient but those of skip and step_bias is required, states 16-byte aligned", what);
    return GRM_HIP_EINVAL;
  }
  const BwdPlan p = bwd_plan(u->batch > 0 ? u->batch : 0, u->seq_len, u->heads, u->value_dim, u->groups, u->key_dim, u->dtype);
  if (u->batch > 0 && (workspace == nullptr || !aligned(workspace) || workspace_bytes < p.bytes)) {
    set_error("%s: workspace missing, misaligned or too small", what);
    return GRM_HIP_EINVAL;
  }
  const int64_t waves4 = sel_ceil(u->batch * p.nsave * u->heads, 4);
  if (p.wgs * p.splits * kGradThreads > UINT32_MAX || waves4 * 256 > UINT32_MAX) {  // a grid dimension has fewer than 2^32 threads
    set_error("%s: too many blocks for one launch", what);
    return GRM_HIP_EUNSUPPORTED;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  const int64_t rows = u->heads * u->value_dim;
  if (u->batch > 0) {
    // The adjoint's walk, from the gradient of the final state to that of the first.
    SelArgs r = sel_args(u);
    r.vec = r.vec && aligned(grad_hidden);
    r.keys = u->queries; r.kb = u->queries_batch_stride; r.kt = u->queries_token_stride;
    r.values = grad_hidden; r.vb = u->seq_len * rows; r.vt = rows;
    r.memory = grad_memory_out; r.memory_out = grad_memory;
    r.states = reinterpret_cast<float*>(ws + p.adj); r.nsave = p.nsave;
    r.parts = p.parts; r.part_tokens = p.part_tokens;
    r.part_state = reinterpret_cast<float*>(ws + p.part_state);
    r.part_log = reinterpret_cast<double*>(ws + p.part_log);
    if (p.parts > 1) {
      if (int rc = launch_state_pass(r, u->dtype, true, true, s, what)) return rc;
    }
    if (int rc = launch_state_pass(r, u->dtype, true, false, s, what)) return rc;
  }
  int rc = GRM_HIP_OK;
  if (p.wgs > 0) {
    GradArgs a{};
    a.s = sel_args(u);
    a.s.states = const_cast<float*>(states);
    a.s.nsave = p.nsave;
    a.s.vec = a.s.vec && aligned(grad_hidden) && aligned(grad_keys) && aligned(grad_values) && aligned(grad_queries);
    a.dy = grad_hidden; a.adj = reinterpret_cast<const float*>(ws + p.adj);
    a.dx = grad_values; a.dk = grad_keys; a.dq = grad_queries; a.dsteps = grad_steps;
    a.tokens = reinterpret_cast<float*>(ws + p.tokens);
    a.diffs = reinterpret_cast<float*>(ws + p.diffs);
    a.dots = reinterpret_cast<float*>(ws + p.dots);
    a.rows_part = p.splits > 1 ? reinterpret_cast<float*>(ws + p.rows) : nullptr;
    a.head_part = reinterpret_cast<float*>(ws + p.heads);
    a.splits = p.splits;
    const dim3 waves(static_cast<uint32_t>(waves4));
    sel_with_form(u->dtype, u->key_dim, a.s.vec != 0, [&](auto e, auto m, auto np, auto vec) {
      using E = decltype(e);
      using M = decltype(m);
      constexpr int NP = decltype(np)::value;
      using Lds = GradLds<M, NP>;
      auto kernel = selective_grad_kernel<E, M, NP, decltype(vec)::value>;
      const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Lds::bytes));
      if (err != hipSuccess) {
        set_error("%s: %s", what, hipGetErrorString(err));
        rc = static_cast<int>(err);
        return;
      }
      selective_token_kernel<E, Lds::LB><<<waves, dim3(256), 0, s>>>(a);
      if ((rc = check_launch(what)) != GRM_HIP_OK) return;
      kernel<<<dim3(static_cast<uint32_t>(p.wgs * p.splits)), dim3(kGradThreads), Lds::bytes, s>>>(a);
      if ((rc = check_launch(what)) != GRM_HIP_OK) return;
      selective_steps_kernel<E, Lds::LB, Lds::CS><<<waves, dim3(256), 0, s>>>(a);
      rc = check_launch(what);
    });
    if (rc != GRM_HIP_OK) return rc;
  }
  const int64_t n = p.splits > 1 ? u->batch * u->seq_len * u->groups * u->key_dim : 0, blocks = sel_ceil(2 * n, 256);
  const dim3 grid(static_cast<uint32_t>((blocks < 4096 ? blocks : 4096) + u->heads));
  auto sum = [&](auto e) {
    selective_sum_kernel<decltype(e)><<<grid, dim3(256), 0, s>>>(
        reinterpret_cast<const float*>(ws + p.rows), p.splits, grad_keys, grad_queries, n,
        reinterpret_cast<const float*>(ws + p.heads), u->batch * p.nsave, static_cast<int>(u->heads), grad_rates, grad_skip,
        grad_step_bias);
  };
  if (u->dtype == GRM_HIP_F32) sum(F32{});
  else if (u->dtype == GRM_HIP_F16) sum(F16{});
  else sum(BF16{});
  return check_launch(what);
}
