// The gated delta rule on MI355X: the chunks' inverses and weights, the walk over a sequence's chunks, and the single
// token.  The mathematics is in delta.h.
#include "delta.h"
#include "delta_limits.h"

namespace grmhip {
namespace {

constexpr int kPrepThreads = 256;
constexpr int kWalkThreads = 256;
constexpr int kStepThreads = 256;
constexpr int kTriStride = 68;  // floats of a row of a 64 x 64 float32 matrix in LDS

// acc += X Y of two 16 x 16 float32 tiles in LDS, in float32.
__device__ __forceinline__ f32x4 mm16(const float* x, const float* y, f32x4 acc) {
  const int g = lane_id() >> 4, n = lane_id() & 15;
#pragma unroll
  for (int s = 0; s < 4; ++s)
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[n * kTriStride + 4 * s + g], y[(4 * s + g) * kTriStride + n], acc, 0, 0, 0);
  return acc;
}
__device__ __forceinline__ void put16(float* y, f32x4 v) {
  const int g = lane_id() >> 4, n = lane_id() & 15;
#pragma unroll
  for (int r = 0; r < 4; ++r) y[(4 * g + r) * kTriStride + n] = v[r];
}

// LDS of a chunk's preparation: A, and in one place the keys' fragments and then the inverse.
template <class E, int NK>
struct PrepLds {
  static constexpr int NI = DParts<E>::IN, S = NK / 32, frags = 4 * S * NI;
  static constexpr size_t a = 0, m = 64 * kTriStride * 4, keys = frags * kDFragElems * 2,
                          cum = m + (keys > 64 * kTriStride * 4 ? keys : 64 * kTriStride * 4), b = cum + 64 * 8, odd = b + 64 * 4,
                          bytes = odd + 4 * 4;
};

// One workgroup a chunk of a head.  Forward: the inverse of I + A b and the weights (W * Q K^T) b, both lower
// triangular, by rows.  BACK: the inverse of I + b A and W * Q K^T, transposed (the reverse walk multiplies by their transposes).
// The inverse: forward substitution inside the four 16 x 16 blocks of the diagonal, then two rounds of
// -T2 (A21 T1) in float32 products.  Substitution does not cancel where keys lie close to each other, as a product of
// powers of A would.  Wave w holds token tile w; the other tiles' keys come as fragments through LDS.
// Bound by the substitution's chain and by what it writes (31 KB a chunk with 2 parts of the weights), so four workgroups share a
// CU (fewer: 63 us): 55 us for 8 x 2048 bf16 tokens x 16 heads of 128 keys, 2.3 TB/s written; transposed 66 (37 KB a chunk).
template <class E, int NK, bool VEC, bool BACK>
__global__ __launch_bounds__(kPrepThreads, 4) void delta_prep_kernel(DeltaArgs a) {
  using raw = typename ET<E>::raw;
  using L = PrepLds<E, NK>;
  constexpr int NI = DParts<E>::IN, PP = BACK ? 3 : DParts<E>::OUT, S = NK / 32, ES = static_cast<int>(sizeof(raw));
  extern __shared__ __attribute__((aligned(16))) char lds[];
  float* A = reinterpret_cast<float*>(lds + L::a);
  float* M = reinterpret_cast<float*>(lds + L::m);
  uint16_t* keys = reinterpret_cast<uint16_t*>(lds + L::m);
  double* cum_s = reinterpret_cast<double*>(lds + L::cum);
  float* b_s = reinterpret_cast<float*>(lds + L::b);
  int* odd_s = reinterpret_cast<int*>(lds + L::odd);
  const int lane = lane_id(), w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, n = lane & 15;
  const uint32_t at = xcd_order(blockIdx.x, gridDim.x);
  const int h = static_cast<int>(at % a.H), c = static_cast<int>(at / a.H % a.C), b = static_cast<int>(at / a.H / a.C);
  const int64_t len = delta_length(a, b), t0 = static_cast<int64_t>(c) * kDTokens;
  if (t0 >= len) return;
  const int rows = static_cast<int>(min_i64(kDTokens, len - t0)), gi = h / (a.H / a.G);

  // Keys and queries of this wave's tile, with no load behind a branch.
  U8<E> ku[S], qu[S];
  {
    const __amdgpu_buffer_rsrc_t kr = make_rsrc(static_cast<const raw*>(a.keys) + b * a.kb + t0 * a.kt + static_cast<int64_t>(gi) * a.N, 0x7ffffff0u),
                                 qr = make_rsrc(static_cast<const raw*>(a.queries) + b * a.qb + t0 * a.qt + static_cast<int64_t>(gi) * a.N, 0x7ffffff0u);
    const int tok = 16 * w + n, ko = tok * static_cast<int>(a.kt), qo = tok * static_cast<int>(a.qt);
    auto load = [&](__amdgpu_buffer_rsrc_t r, int off, int s) {
      const int col = 32 * s + 8 * g;
      if constexpr (VEC) {
        return buf_load8<E>(r, tok < rows && col < a.N ? (off + col) * ES : kBufOOB);
      } else {
        U8<E> u;
#pragma unroll
        for (int e = 0; e < 8; ++e) u.e[e] = buf_load1<E>(r, tok < rows && col + e < a.N ? (off + col + e) * ES : kBufOOB);
        return u;
      }
    };
#pragma unroll
    for (int s = 0; s < S; ++s) {
      ku[s] = load(kr, ko, s);
      qu[s] = load(qr, qo, s);
    }
  }
  // Scalars, lane = token, in every wave.
  float bt = 0.f, gt = 0.f;
  if (lane < rows) {
    const int64_t i = b * a.sb + (t0 + lane) * a.st + h, j = b * a.db + (t0 + lane) * a.dt + h;
    bt = a.s_f32 ? static_cast<const float*>(a.strengths)[i] : ET<E>::to_f(static_cast<const raw*>(a.strengths)[i]);
    if (a.decays != nullptr)
      gt = a.d_f32 ? static_cast<const float*>(a.decays)[j] : ET<E>::to_f(static_cast<const raw*>(a.decays)[j]);
  }
  // The first token whose key, strength or decay is no number (the walk takes it from there).
  const float inf = __builtin_inff();
  int odd = 64;
  if (!BACK) {
    float zero = 0.f;  // (a product with zero is zero or NaN)
#pragma unroll
    for (int s = 0; s < S; ++s) {
#pragma unroll
      for (int e = 0; e < 8; ++e) zero = fmaf(ET<E>::to_f(ku[s].e[e]), 0.f, zero);
    }
    const uint64_t mask = __ballot(zero != 0.f);
    const uint32_t m16 = static_cast<uint32_t>((mask | mask >> 16 | mask >> 32 | mask >> 48) & 0xffff);
    const uint64_t scal = __ballot(!(fabsf(bt) < inf) || !(gt < inf));
    if (m16 != 0) odd = 16 * w + __builtin_ctz(m16);
    if (scal != 0 && __builtin_ctzll(scal) < odd) odd = __builtin_ctzll(scal);
    if (lane == 0) odd_s[w] = odd;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) odd = odd_s[i] < odd ? odd_s[i] : odd;
    if (lane >= odd) bt = gt = 0.f;
  }
  // Log decays in log2 units and float64, as differences of running sums stay exact; a token's is held to -200 (a
  // factor of 1e-60, nothing beside the 2^-24 of a term), so that sums stay numbers.
  double l = static_cast<double>(gt) * 1.4426950408889634;
  l = l < -200.0 ? -200.0 : l;
  const double cum = wave_prefix(l), total = lane_value(cum, 63);
  char* out = a.work + ((static_cast<int64_t>(b) * a.H + h) * a.C + c) * delta_chunk_bytes(PP);
  uint16_t* tf = reinterpret_cast<uint16_t*>(out);
  uint16_t* pf = tf + 3 * kDFrags * kDFragElems;
  float* sc = reinterpret_cast<float*>(pf + PP * kDFrags * kDFragElems);
  if (w == 0) {
    cum_s[lane] = cum;
    b_s[lane] = bt;
    sc[lane] = exp2_d(cum);
    sc[64 + lane] = exp2_d(total - cum) * (BACK ? 1.f : bt);
    sc[128 + lane] = bt;
    if (lane == 0) reinterpret_cast<int*>(sc)[192] = odd;
  }
  B8 ki[S][NI], qi[S][NI];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if (!BACK && 16 * w + n >= odd) zero_u8<E>(ku[s]);
    input_parts<E, NI>(ku[s], ki[s]);
    input_parts<E, NI>(qu[s], qi[s]);
#pragma unroll
    for (int p = 0; p < NI; ++p)
      *reinterpret_cast<uint4*>(keys + ((w * S + s) * NI + p) * kDFragElems + 8 * lane) = __builtin_bit_cast(uint4, ki[s][p]);
  }
  __syncthreads();

  const int i = 16 * w + n;
  const double ci = cum_s[i];
  const float bi = b_s[i];
  float y[4][4];
#pragma unroll
  for (int tj = 0; tj < 4; ++tj) {
    f32x4 kk = {0.f, 0.f, 0.f, 0.f}, qk = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 4; ++r) y[tj][r] = 0.f;
    if (tj > w) continue;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      B8 kj[NI];
#pragma unroll
      for (int p = 0; p < NI; ++p)
        kj[p] = __builtin_bit_cast(B8, *reinterpret_cast<const uint4*>(keys + ((tj * S + s) * NI + p) * kDFragElems + 8 * lane));
      kk = mma_parts<3>(kj, ki[s], kk);                  // column i = 16 w + n, rows j = 16 tj + 4 g + r
      if (BACK) qk = mma_parts<3>(qi[s], kj, qk);        // column j = 16 tj + n, rows i = 16 w + 4 g + r
      else qk = mma_parts<3>(kj, qi[s], qk);
    }
    float x[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int j = 16 * tj + 4 * g + r;
      const float bj = b_s[j], wt = j <= i ? exp2_f(static_cast<float>(ci - cum_s[j])) : 0.f;
      x[r] = j < i ? wt * kk[r] * (BACK ? bi : bj) : 0.f;
      if (BACK) {
        const int i2 = 16 * w + 4 * g + r, j2 = 16 * tj + n;
        y[tj][r] = j2 <= i2 ? exp2_f(static_cast<float>(cum_s[i2] - cum_s[j2])) * qk[r] : 0.f;
      } else {
        y[tj][r] = j <= i ? wt * qk[r] * bj : 0.f;
      }
    }
    *reinterpret_cast<float4*>(&A[i * kTriStride + 16 * tj + 4 * g]) = make_float4(x[0], x[1], x[2], x[3]);
  }
  // The weights: forward a step of a fragment is two tiles of this wave; backward its halves come from two waves.
  if constexpr (!BACK) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s > w / 2) continue;
      const float v[8] = {y[2 * s][0], y[2 * s][1], y[2 * s][2], y[2 * s][3], y[2 * s + 1][0], y[2 * s + 1][1], y[2 * s + 1][2], y[2 * s + 1][3]};
      B8 f[PP];
      split8<PP>(v, f);
      const int frag = w < 2 ? w : 2 * w - 2 + s;  // lower_frag(w, s)
#pragma unroll
      for (int p = 0; p < PP; ++p)
        *reinterpret_cast<uint4*>(pf + (frag * PP + p) * kDFragElems + 8 * lane) = __builtin_bit_cast(uint4, f[p]);
    }
  } else {
#pragma unroll
    for (int tj = 0; tj < 4; ++tj) {
      if (tj > w) continue;
      const int frag = tj < 2 ? 2 * tj + (w >> 1) : tj + 2, half = w & 1;  // upper_frag(tj, w / 2)
      float v[8] = {y[tj][0], y[tj][1], y[tj][2], y[tj][3], 0.f, 0.f, 0.f, 0.f};
      B8 f[PP];
      split8<PP>(v, f);
#pragma unroll
      for (int p = 0; p < PP; ++p) {
        const uint4 u = __builtin_bit_cast(uint4, f[p]);
        uint16_t* to = pf + (frag * PP + p) * kDFragElems + 8 * lane;
        *reinterpret_cast<uint2*>(to + 4 * half) = make_uint2(u.x, u.y);
        if (tj == w && half == 1) *reinterpret_cast<uint2*>(to) = make_uint2(0u, 0u);  // (beyond the diagonal)
      }
    }
  }
  __syncthreads();

  // Diagonal blocks, column n of block w in the registers of lane n (four times over); A's rows in whole reads.
  auto tile = [](float* m, int i, int j) { return m + 16 * i * kTriStride + 16 * j; };
  {
    const float* d = tile(A, w, w);
    float x[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float v = r == n ? 1.f : 0.f, u = 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (4 * q >= r) continue;
        const float4 e = *reinterpret_cast<const float4*>(d + r * kTriStride + 4 * q);
        const float ee[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (4 * q + k < r) (k & 1 ? u : v) = fmaf(-ee[k], x[4 * q + k], k & 1 ? u : v);
      }
      x[r] = v + u;
    }
    float* m = tile(M, w, w);
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if ((r >> 2) == g) m[r * kTriStride + n] = x[r];
  }
  __syncthreads();
  // The products wait in the tiles of A above the diagonal.
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  if (w < 2) put16(tile(A, 2 * w, 2 * w + 1), mm16(tile(A, 2 * w + 1, 2 * w), tile(M, 2 * w, 2 * w), zero));
  __syncthreads();
  if (w < 2) put16(tile(M, 2 * w + 1, 2 * w), -mm16(tile(M, 2 * w + 1, 2 * w + 1), tile(A, 2 * w, 2 * w + 1), zero));
  __syncthreads();
  {
    const int ti = 2 + (w >> 1), tj = w & 1;
    f32x4 v = mm16(tile(A, ti, 1), tile(M, 1, tj), zero);
    if (tj == 0) v = mm16(tile(A, ti, 0), tile(M, 0, 0), v);
    put16(tile(A, tj, ti), v);
    __syncthreads();
    f32x4 z = mm16(tile(M, ti, 2), tile(A, tj, 2), zero);
    if (ti == 3) z = mm16(tile(M, 3, 3), tile(A, tj, 3), z);
    put16(tile(M, ti, tj), -z);
  }
  __syncthreads();
  // Into fragments: forward rows i with slots over j, backward rows j with slots over i.
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if (BACK ? s < w / 2 : s > w / 2) continue;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = 32 * s + (e < 4 ? 4 * g + e : 16 + 4 * g + e - 4);
      const float u = BACK ? M[k * kTriStride + i] : M[i * kTriStride + k];
      v[e] = (BACK ? k >= i : k <= i) ? u : 0.f;
    }
    B8 f[3];
    split8<3>(v, f);
    const int frag = BACK ? (w < 2 ? 2 * w + s : w + 2) : (w < 2 ? w : 2 * w - 2 + s);
#pragma unroll
    for (int p = 0; p < 3; ++p)
      *reinterpret_cast<uint4*>(tf + (frag * 3 + p) * kDFragElems + 8 * lane) = __builtin_bit_cast(uint4, f[p]);
  }
}

// Zeros for the tokens (columns) from `rows` on: a query of zeros alone gives NaN of a state that is no number, and what is
// NaN from a live token on stays so to the chunk's end.
__device__ __forceinline__ void clear_rows(f32x4 (&o)[4], int64_t rows) {
#pragma unroll
  for (int t = 0; t < 4; ++t)
    if (16 * t + (lane_id() & 15) >= rows) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
}

// LDS of a walk: keys and queries as their parts, values, the chunk's scalars.
template <class E, int NK>
struct WalkLds {
  using KT = SelTile<BF16, NK, true>;
  using QT = SelTile<BF16, NK, false>;
  using VT = SelTile<E, kDCols, true>;
  static constexpr int NI = DParts<E>::IN;
  static constexpr int kpart = kDTokens * KT::STRIDE, qpart = kDTokens * QT::STRIDE;
  static constexpr size_t k = 0, q = k + NI * kpart * 2, v = q + NI * qpart * 2,
                          s = v + kDTokens * VT::STRIDE * sizeof(typename ET<E>::raw), bytes = s + 128 * 4;
};

// One workgroup walks 64 value columns of a head over the whole sequence; a wave holds 16 of them, its state in
// accumulators (the state's columns never meet: each wave's chain is its own).  Accumulators of K S^T, of m and of the state
// lie as the next product's operand wants them, so nothing but the inputs passes through LDS.
// For float16 and float32 keys wider than 64 only, whose stages for delta_pair_kernel do not fit, and in one time part.  8 x 2048
// tokens x 16 heads of 128 x 128, whole calls: 316 us in float16, 529 in float32 (bfloat16 by the other kernel 180-230); a
// sequence of 32768 tokens x 16 heads, which its 32 workgroups walk alone, 3.7 and 5.7 ms (0.66).
template <class E, int NK, bool VEC>
__global__ __launch_bounds__(kWalkThreads, 1) void delta_walk_kernel(DeltaArgs a) {
  using raw = typename ET<E>::raw;
  using L = WalkLds<E, NK>;
  using KT = typename L::KT;
  using QT = typename L::QT;
  using VT = typename L::VT;
  constexpr int NI = L::NI, NO = DParts<E>::OUT, S = NK / 32, NT = NK / 16;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  uint16_t* kt = reinterpret_cast<uint16_t*>(lds + L::k);
  uint16_t* qt = reinterpret_cast<uint16_t*>(lds + L::q);
  raw* vt = reinterpret_cast<raw*>(lds + L::v);
  float* sc = reinterpret_cast<float*>(lds + L::s);
  const int tid = threadIdx.x, lane = lane_id(), w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, n = lane & 15;
  const uint32_t at = xcd_order(blockIdx.x, gridDim.x);
  const int pt = static_cast<int>(at % a.PT), h = static_cast<int>(at / a.PT % a.H), b = static_cast<int>(at / a.PT / a.H);
  const int64_t len = delta_length(a, b);
  const int col0 = pt * kDCols, p0 = col0 + 16 * w, gi = h / (a.H / a.G);
  const int chunks = static_cast<int>((len + kDTokens - 1) / kDTokens);
  const float inf = __builtin_inff();

  const raw* kp = static_cast<const raw*>(a.keys) + b * a.kb + static_cast<int64_t>(gi) * a.N;
  const raw* qp = static_cast<const raw*>(a.queries) + b * a.qb + static_cast<int64_t>(gi) * a.N;
  const raw* vp = static_cast<const raw*>(a.values) + b * a.vb + static_cast<int64_t>(h) * a.P + col0;
  const char* work = a.work + (static_cast<int64_t>(b) * a.H + h) * a.C * delta_chunk_bytes(NO);
  TileLoad<E, KT, BF16, VEC, kDTokens, NK, kWalkThreads> kl;
  TileLoad<E, QT, BF16, VEC, kDTokens, NK, kWalkThreads> ql;
  TileLoad<E, VT, E, VEC, kDTokens, kDCols, kWalkThreads> vl;
  kl.init(a.kt, a.N, tid);
  ql.init(a.qt, a.N, tid);
  vl.init(a.vt, a.P - col0 < kDCols ? a.P - col0 : kDCols, tid);
  float sreg = 0.f;
  int odd_next = 64;
  auto fetch = [&](int c) {
    const int64_t t0 = static_cast<int64_t>(c) * kDTokens;
    kl.load(kp + t0 * a.kt, len - t0, tid);
    ql.load(qp + t0 * a.qt, len - t0, tid);
    vl.load(vp + t0 * a.vt, len - t0, tid);
    const float* s = reinterpret_cast<const float*>(work + c * delta_chunk_bytes(NO) + (3 + NO) * kDFrags * kDFragElems * 2);
    sreg = s[tid & 127];
    odd_next = reinterpret_cast<const int*>(s)[192];
  };

  f32x4 st[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) st[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int64_t head = static_cast<int64_t>(b) * a.H + h, cells = static_cast<int64_t>(a.P) * a.N;
  if (a.memory != nullptr) state_add<NT>(st, a.memory + head * cells, p0, a.P, a.N, 1.f);
  // The triangular matrices' fragments, loaded a chunk ahead as soon as the last ones are done with.
  B8 tf[kDFrags][3], pf[kDFrags][NO];
  if (chunks > 0) {
    fetch(0);
    stored_triangle<3>(reinterpret_cast<const uint16_t*>(work), tf, lane);
    stored_triangle<NO>(reinterpret_cast<const uint16_t*>(work) + 3 * kDFrags * kDFragElems, pf, lane);
  }

  for (int c = 0; c < chunks; ++c) {
    const int64_t t0 = static_cast<int64_t>(c) * kDTokens;
    const int odd_key = odd_next;
    __syncthreads();
    store_parts<KT, NI, E>(kl, kt, L::kpart, odd_key, tid);
    store_parts<QT, NI, E>(ql, qt, L::qpart, kDTokens, tid);
    vl.store(vt, tid);
    if (tid < 128) sc[tid] = sreg;
    __syncthreads();
    // Loads ahead stand behind no branch (behind the last chunk it is loaded again): a wait then counts them exactly.
    const int next = c + 1 < chunks ? c + 1 : c;
    fetch(next);
    if (a.states != nullptr)
      state_store<NT>(st, a.states + ((static_cast<int64_t>(b) * a.C + c) * a.H + h) * cells, p0, a.P, a.N);

    // K S^T (a token a row, a value a column) and Q S^T (transposed, as its rows are stored).
    B8 sp[S][3];
#pragma unroll
    for (int s = 0; s < S; ++s) split2<3>(st[2 * s], st[2 * s + 1], sp[s]);
    f32x4 x[4], o[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) x[t] = o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < S; ++s) {
      B8 kf[4][NI], qf[4][NI], so[NO];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        row_parts_t<KT, NI>(kt, L::kpart, 16 * t, 32 * s, kf[t]);
        row_parts_t<QT, NI>(qt, L::qpart, 16 * t, 32 * s, qf[t]);
      }
#pragma unroll
      for (int p = 0; p < NO; ++p) so[p] = sp[s][p];
      mma_many<3, true>(kf, sp[s], x);
      mma_many<NO, false>(qf, so, o);
    }
    // V - D K S^T.
    f32x4 rt[4];
    bool any = false;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const Frag8<E> vf = col_frag<VT, E>(vt, 32 * s, 16 * w);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 d = *reinterpret_cast<const float4*>(sc + 32 * s + 16 * i + 4 * g);
        const float dd[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float v = fmaf(-dd[r], x[2 * s + i][r], ET<E>::to_f(vf.e[4 * i + r]));
          rt[2 * s + i][r] = v;
          any |= !(fabsf(v) < inf);
        }
      }
    }
    // A value, key or state that is no number: from its token on the column is NaN.  Its rows stay out of the products,
    // whose zeros would not keep them out of earlier tokens' sums.
    int cut = 64;
    if (__any(any) || odd_key < 64) {
      auto first = [&](const f32x4 (&y)[4]) {
        int f = 64;
#pragma unroll
        for (int t = 3; t >= 0; --t) {
#pragma unroll
          for (int r = 3; r >= 0; --r)
            if (!(fabsf(y[t][r]) < inf)) f = 16 * t + 4 * g + r;
        }
        const int f1 = __shfl_xor(f, 16), f2 = f < f1 ? f : f1, f3 = __shfl_xor(f2, 32);
        return f2 < f3 ? f2 : f3;
      };
      cut = first(rt);
      cut = cut < odd_key ? cut : odd_key;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (16 * t + 4 * g + r >= cut) rt[t][r] = 0.f;
      }
    }
    // m.
    f32x4 m[4];
    {
      B8 rp[2][3];
#pragma unroll
      for (int s = 0; s < 2; ++s) split2<3>(rt[2 * s], rt[2 * s + 1], rp[s]);
#pragma unroll
      for (int t = 0; t < 4; ++t) m[t] = f32x4{0.f, 0.f, 0.f, 0.f};
      mma_triangle<3, true, true>(tf, rp, m);
    }
    stored_triangle<3>(reinterpret_cast<const uint16_t*>(work + next * delta_chunk_bytes(NO)), tf, lane);
    if (a.miss != nullptr && p0 + n < a.P) {
      float* to = a.miss + ((static_cast<int64_t>(b) * a.T + t0) * a.H + h) * a.P + p0 + n;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int tok = 16 * t + 4 * g + r;
          if (t0 + tok < len) to[static_cast<int64_t>(tok) * a.H * a.P] = m[t][r];
        }
      }
    }
    // H^T = S Q^T D + m^T P^T.
    {
      B8 mp[2][NO];
#pragma unroll
      for (int s = 0; s < 2; ++s) split2<NO>(m[2 * s], m[2 * s + 1], mp[s]);
#pragma unroll
      for (int t = 0; t < 4; ++t) o[t] *= sc[16 * t + n];
      mma_triangle<NO, true, false>(pf, mp, o);
    }
    stored_triangle<NO>(reinterpret_cast<const uint16_t*>(work + next * delta_chunk_bytes(NO)) + 3 * kDFrags * kDFragElems, pf, lane);
    if (__any(cut < 64)) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int f = __shfl(cut, 4 * g + r);
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (16 * t + n >= f) o[t][r] = __builtin_nanf("");
      }
    }
    if (t0 + kDTokens > len) clear_rows(o, len - t0);
    {
      const int p = p0 + 4 * g, row = a.H * a.P * static_cast<int>(sizeof(raw));
      const int64_t left = a.T - t0;
      const __amdgpu_buffer_rsrc_t to =
          make_rsrc(static_cast<raw*>(a.hidden) + ((static_cast<int64_t>(b) * a.T + t0) * a.H + h) * a.P, 0x7ffffff0u);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int tok = 16 * t + n;
        if (VEC) {
          buf_store4<E>(to, tok < left && p < a.P ? tok * row + p * static_cast<int>(sizeof(raw)) : kBufOOB, o[t]);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            buf_store1<E>(to, tok < left && p + r < a.P ? tok * row + (p + r) * static_cast<int>(sizeof(raw)) : kBufOOB, o[t][r]);
        }
      }
    }
    // S' = e^{c_63} S + (E b m)^T K.
    {
      const float keep = sc[63];
#pragma unroll
      for (int i = 0; i < NT; ++i) st[i] *= keep;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        f32x4 em[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 e = *reinterpret_cast<const float4*>(sc + 64 + 32 * s + 16 * i + 4 * g);
          em[i] = f32x4{m[2 * s + i][0] * e.x, m[2 * s + i][1] * e.y, m[2 * s + i][2] * e.z, m[2 * s + i][3] * e.w};
        }
        B8 ep[3];
        split2<3>(em[0], em[1], ep);
        B8 kf[NT][NI];
#pragma unroll
        for (int i = 0; i < NT; ++i) col_parts<KT, NI>(kt, L::kpart, 32 * s, 16 * i, kf[i]);
        mma_many<3, true>(kf, ep, st);
      }
    }
    if (cut < 64) {
#pragma unroll
      for (int i = 0; i < NT; ++i) st[i] = f32x4{1.f, 1.f, 1.f, 1.f} * __builtin_nanf("");
    }
  }
  state_store<NT>(st, a.memory_out + head * cells, p0, a.P, a.N);
  // Rows behind the last chunk.
  for (int64_t t = static_cast<int64_t>(chunks) * kDTokens + tid / 16; t < a.T; t += kWalkThreads / 16) {
    raw* row = static_cast<raw*>(a.hidden) + ((b * a.T + t) * a.H + h) * a.P + col0;
    for (int p = tid % 16; p < kDCols && col0 + p < a.P; p += 16) row[p] = 0;
  }
}

// LDS of the walk in two halves: two stages of a chunk, where they fit, else of its keys alone.
template <class E, int NK>
struct PairLds {
  // Keys are read by rows and by columns; rows 4 banks apart (2 clocks a row read, 4 a column read) take 140 us for 8 x 2048
  // tokens x 16 heads where rows 8 banks apart (4 and 2) took 148: the row reads stand in the chain.
  using KT = SelTile<BF16, NK, false>;
  using QT = SelTile<BF16, NK, false>;
  using VT = SelTile<E, kDCols, true>;
  static constexpr int NI = DParts<E>::IN, NO = DParts<E>::OUT, SCAL = 132;
  static constexpr int kpart = kDTokens * KT::STRIDE, qpart = kDTokens * QT::STRIDE;
  static constexpr int state = NK / 32 * NO * kDFragElems;  // a wave's state as fragments
  static constexpr int qstage = NI * qpart, vstage = kDTokens * VT::STRIDE;
  static constexpr size_t kbytes = 2 * NI * kpart * 2, qvbytes = qstage * 2 + vstage * sizeof(typename ET<E>::raw),
                          other = 4 * state * 2 + 4 * 4 * 64 * 16 + 2 * SCAL * 4 + 64 * 4;
  static constexpr int QV = kbytes + 2 * qvbytes + other <= 160 * 1024 ? 2 : 1;  // stages of queries and values
  static constexpr size_t k = 0, q = kbytes, v = q + QV * qstage * 2, s = v + QV * vstage * sizeof(typename ET<E>::raw),
                          m = s + 4 * state * 2, sc = m + 4 * 4 * 64 * 16, cut = sc + 2 * SCAL * 4, bytes = cut + 64 * 4;
  static constexpr bool fits = bytes <= 160 * 1024;
};
// Of the parts' walk without outputs: three stages of keys and two of both halves' values.
template <class E, int NK>
struct LocalLds : PairLds<E, NK> {
  using L = PairLds<E, NK>;
  static constexpr size_t k = 0, v = 3 * L::NI * L::kpart * 2, sc = v + 4 * L::vstage * sizeof(typename ET<E>::raw),
                          bytes = sc + 3 * L::SCAL * 4;
  static_assert(!L::fits || bytes <= 160 * 1024, "three stages");
};

// The walk over a sequence's chunks, 64 value columns of a head a workgroup.  Four state waves hold 16 columns each, in
// accumulators, and run the chain that a chunk hangs on: K S^T, m, the next state.  Four output waves, one beside each
// on its SIMD, load the chunks ahead into LDS and form what hangs on no later chunk: Q S^T while m is formed, then
// the weights' product with m, and the stores.  A state's columns never meet, so a state wave's chain is its own;
// accumulators of K S^T, of m and of the state lie as the next product's operand wants them.  Two barriers a chunk:
// m is there, the next state is there.
// Bound by the chain: 8 x 2048 bf16 tokens x 16 heads of 128 x 128 take 140 us, 4.4 a chunk.  Of the busy cycles a SIMD's matrix
// products are 35% and a CU's LDS accesses 44% (four waves that did all of it took 130 us more).
// SAVE: the states before every chunk and m are kept for the backward.
// Sequences in time parts: a first launch (LOCAL) walks all parts but the last side by side and without outputs.  Rows of a
// state never meet, and without values each passes through a part as a row of a matrix product; so beside the value rows of a
// part, from a zero state, go the N rows of the identity without values, whose end is the part's map.  delta_join_kernel makes
// the parts' first states of both, and the second launch walks every part from its own.  Without outputs all eight waves hold
// states, 128 columns of value rows and then identity a workgroup, so that two chains share a SIMD; they load the keys
// together, three stages, one barrier a chunk (7 parts of 64 chunks x 16 heads of 128 x 128: 340 us; 446 with a chain a SIMD).
template <class E, int NK, bool VEC, bool SAVE, bool LOCAL>
__global__ __launch_bounds__(2 * kWalkThreads, 2) void delta_pair_kernel(DeltaArgs a) {
  using raw = typename ET<E>::raw;
  using L = std::conditional_t<LOCAL, LocalLds<E, NK>, PairLds<E, NK>>;
  using KT = typename L::KT;
  using QT = typename L::QT;
  using VT = typename L::VT;
  constexpr int NI = L::NI, NO = L::NO, S = NK / 32, NT = NK / 16, QV = LOCAL ? 2 : L::QV;
  constexpr int KLOADERS = (LOCAL ? 2 : 1) * kWalkThreads;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  uint16_t* kt = reinterpret_cast<uint16_t*>(lds + L::k);
  uint16_t* qt = reinterpret_cast<uint16_t*>(lds + L::q);
  raw* vt = reinterpret_cast<raw*>(lds + L::v);
  float* sc = reinterpret_cast<float*>(lds + L::sc);
  int* cuts = reinterpret_cast<int*>(lds + L::cut);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3;
  const int lane = lane_id(), g = lane >> 4, n = lane & 15;
  const uint32_t at = xcd_order(blockIdx.x, gridDim.x);
  const int tiles = LOCAL ? (a.PT + a.NT + 1) / 2 : a.PT, parts = LOCAL ? a.parts - 1 : a.parts;
  const int half = LOCAL ? wave >> 2 : 0;
  const int pt = static_cast<int>(at % tiles) * (LOCAL ? 2 : 1) + half, part = static_cast<int>(at / tiles % parts);
  const int h = static_cast<int>(at / tiles / parts % a.H), b = static_cast<int>(at / tiles / parts / a.H);
  const bool map = LOCAL && pt >= a.PT;  // rows of the identity
  if (LOCAL && pt - half >= a.PT && part == 0) return;  // (the first part starts from the sequence's own state)
  const int64_t len = delta_length(a, b);
  const int col0 = (map ? pt - a.PT : pt) * kDCols, p0 = col0 + 16 * w, gi = h / (a.H / a.G), prows = map ? a.N : a.P;
  const int first = part * a.part_chunks, have = static_cast<int>((len + kDTokens - 1) / kDTokens);
  const int chunks = have < first + a.part_chunks ? (have > first ? have : first) : first + a.part_chunks;  // this part's end
  const int64_t head = static_cast<int64_t>(b) * a.H + h, cells = static_cast<int64_t>(a.P) * a.N, all = static_cast<int64_t>(a.B) * a.H;
  const char* work = a.work + head * a.C * delta_chunk_bytes(NO);
  uint16_t* sf = reinterpret_cast<uint16_t*>(lds + L::s) + w * L::state + 8 * lane;
  f32x4* mf = reinterpret_cast<f32x4*>(lds + L::m) + w * 256 + lane;

  const int tid = static_cast<int>(threadIdx.x) - (LOCAL ? 0 : kWalkThreads), vtid = tid % kWalkThreads;  // of the loading waves
  const raw* kp = static_cast<const raw*>(a.keys) + b * a.kb + static_cast<int64_t>(gi) * a.N;
  const raw* qp = static_cast<const raw*>(a.queries) + b * a.qb + static_cast<int64_t>(gi) * a.N;
  const raw* vp = static_cast<const raw*>(a.values) + b * a.vb + static_cast<int64_t>(h) * a.P + (map ? 0 : col0);
  TileLoad<E, KT, BF16, VEC, kDTokens, NK, KLOADERS> kl;
  TileLoad<E, QT, BF16, VEC, kDTokens, NK, kWalkThreads> ql;
  TileLoad<E, VT, E, VEC, kDTokens, kDCols, kWalkThreads> vl;
  float sreg = 0.f, warm = 0.f;
  int oreg = 64;
  auto fetch = [&](int want) {
    const int c = want < chunks ? want : chunks - 1;
    const int64_t t0 = static_cast<int64_t>(c) * kDTokens;
    const float* s = reinterpret_cast<const float*>(work + c * delta_chunk_bytes(NO) + (3 + NO) * kDFrags * kDFragElems * 2);
    sreg = s[tid & 127];
    oreg = reinterpret_cast<const int*>(s)[192];
    kl.load(kp + t0 * a.kt, len - t0, tid);
    if constexpr (!LOCAL) ql.load(qp + t0 * a.qt, len - t0, tid);
    vl.load(vp + t0 * a.vt, map ? 0 : len - t0, vtid);  // (a map's rows have no values)
  };
  auto place_qv = [&](int c) {
    if constexpr (!LOCAL) store_parts<QT, NI, E>(ql, qt + (c & (QV - 1)) * L::qstage, L::qpart, kDTokens, tid);
    vl.store(vt + (2 * half + (c & (QV - 1))) * L::vstage, vtid);
  };
  auto stage = [](int c) { return LOCAL ? c % 3 : c & 1; };
  auto place_k = [&](int c) {
    store_parts<KT, NI, E>(kl, kt + stage(c) * NI * L::kpart, L::kpart, oreg, tid);
    float* to = sc + stage(c) * L::SCAL;
    if (tid < 128) to[tid] = sreg;
    if (tid == 128) reinterpret_cast<int*>(to)[128] = oreg;
  };
  // One word of every line of a later chunk's matrices, so that they lie in the L2 when they are called for.
  auto warm_up = [&](int want) {
    const int c = want < chunks ? want : chunks - 1;
    asm volatile("" ::"v"(warm));
    constexpr int lines = static_cast<int>((LOCAL ? 3 * kDFrags * kDFragElems * 2 : delta_chunk_bytes(NO)) / 128);
    for (int i = tid; i < lines; i += KLOADERS) warm = *reinterpret_cast<const float*>(work + c * delta_chunk_bytes(NO) + 128 * i);
  };
  auto begin = [&] {
    kl.init(a.kt, a.N, tid);
    if constexpr (!LOCAL) ql.init(a.qt, a.N, tid);
    const int cols = prows - col0;
    vl.init(a.vt, cols > kDCols ? kDCols : cols > 0 ? cols : 0, vtid);
    if (chunks > first) {
      fetch(first);
      place_k(first);
      place_qv(first);
      fetch(first + 1);
    }
  };

  if (LOCAL || wave < 4) {
    if constexpr (LOCAL) begin();
    else __builtin_amdgcn_s_setprio(2);
    const float inf = __builtin_inff();
    f32x4 st[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) st[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (map) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int r = 0; r < 4; ++r) st[i][r] = p0 + n == 16 * i + 4 * g + r && p0 + n < a.N ? 1.f : 0.f;
      }
    } else if (part > 0 && !LOCAL) {
      state_add<NT>(st, a.part_state + ((part - 1) * all + head) * cells, p0, a.P, a.N, 1.f);
    } else if (part == 0 && a.memory != nullptr) {
      state_add<NT>(st, a.memory + head * cells, p0, a.P, a.N, 1.f);
    }
    // The triangular matrix's fragments, loaded a chunk ahead as soon as the last ones are done with.
    B8 tf[kDFrags][3], sp[S][3];
    if (chunks > first) stored_triangle<3>(reinterpret_cast<const uint16_t*>(work + first * delta_chunk_bytes(NO)), tf, lane);
    auto publish = [&](int s) {
      split2<3>(st[2 * s], st[2 * s + 1], sp[s]);
      if constexpr (LOCAL) return;
#pragma unroll
      for (int p = 0; p < NO; ++p)
        *reinterpret_cast<uint4*>(sf + (s * NO + p) * kDFragElems) = __builtin_bit_cast(uint4, sp[s][p]);
    };
    auto keep_state = [&](int c, int s) {
      if constexpr (SAVE) state_out<VEC>(st, 2 * s, a.states + ((static_cast<int64_t>(b) * a.C + c) * a.H + h) * cells, p0, a.P, a.N);
    };
    B8 kr[2][4][NI];  // keys by rows, [step & 1][tile]
    auto row_keys = [&](const uint16_t* from, int s) {
#pragma unroll
      for (int t = 0; t < 4; ++t) row_parts_t<KT, NI>(from, L::kpart, 16 * t, 32 * s, kr[s & 1][t]);
    };
#pragma unroll
    for (int s = 0; s < S; ++s) publish(s);
    __syncthreads();
    if (chunks > first) row_keys(kt + stage(first) * NI * L::kpart, 0);
    for (int c = first; c < chunks; ++c) {
      const uint16_t* kc = kt + stage(c) * NI * L::kpart;
      const float* scc = sc + stage(c) * L::SCAL;
      const int next = c + 1 < chunks ? c + 1 : c;
      const raw* vc = vt + (2 * half + (c & (QV - 1))) * L::vstage;
      // (Read ahead of the products, which they wait for.)
      Frag8<E> vf[2];
      float4 dd[4];
#pragma unroll
      for (int s = 0; s < 2; ++s) vf[s] = col_frag<VT, E>(vc, 32 * s, 16 * w);
#pragma unroll
      for (int t = 0; t < 4; ++t) dd[t] = *reinterpret_cast<const float4*>(scc + 16 * t + 4 * g);
      const int odd_key = __builtin_amdgcn_readfirstlane(reinterpret_cast<const int*>(scc)[128]);
      if constexpr (LOCAL) {  // (the stages of the keys two chunks ago and of the last chunk's values)
        place_k(c + 1);
        place_qv(c + 1);
        warm_up(c + 3);
        fetch(c + 2);
      }
      hold_order();
      // K S^T: a token a row, a value a column.
      f32x4 x[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) x[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (s + 1 < S) row_keys(kc, s + 1);
        mma_many<3, true>(kr[s & 1], sp[s], x);
        keep_state(c, s);
        hold_order();
      }
      // V - D K S^T.
      float odd = 0.f;  // (a product with zero is zero or NaN)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float d[4] = {dd[t].x, dd[t].y, dd[t].z, dd[t].w};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[t][r] = fmaf(-d[r], x[t][r], ET<E>::to_f(vf[t / 2].e[4 * (t & 1) + r]));
          odd = fmaf(x[t][r], 0.f, odd);
        }
      }
      // A value, key or state that is no number: from its token on the column is NaN.  Its rows stay out of the products,
      // whose zeros would not keep them out of earlier tokens' sums.
      int cut = 64;
      if (__any(odd != 0.f) || odd_key < 64) {
        int f = odd_key;
#pragma unroll
        for (int t = 3; t >= 0; --t) {
#pragma unroll
          for (int r = 3; r >= 0; --r) {
            const int tok = 16 * t + 4 * g + r;
            if (!(fabsf(x[t][r]) < inf) && tok < f) f = tok;
          }
        }
        const int f1 = __shfl_xor(f, 16), f2 = f < f1 ? f : f1, f3 = __shfl_xor(f2, 32);
        cut = f2 < f3 ? f2 : f3;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (16 * t + 4 * g + r >= cut) x[t][r] = 0.f;
        }
      }
      f32x4 m[4];
      {
        B8 rp[2][3];
#pragma unroll
        for (int s = 0; s < 2; ++s) split2<3>(x[2 * s], x[2 * s + 1], rp[s]);
#pragma unroll
        for (int t = 0; t < 4; ++t) m[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        mma_triangle<3, true, true>(tf, rp, m);
      }
      if constexpr (!LOCAL) {
#pragma unroll
        for (int t = 0; t < 4; ++t) mf[64 * t] = m[t];
        if (g == 0) cuts[16 * w + n] = cut;
      }
      B8 kf[2][2][2][NI];  // [pair & 1][step][tile of the pair]
      auto pair_keys = [&](int j) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
          for (int i = 0; i < 2; ++i) col_parts<KT, NI>(kc, L::kpart, 32 * s, 16 * (2 * j + i), kf[j & 1][s][i]);
        }
      };
      pair_keys(0);
      __syncthreads();
      // S' = e^{c_63} S + (E b m)^T K, two tiles of keys at a time: while one pair's products run, the last pair's sums
      // are split for the next chunk and a share of its triangular matrix is called for (all at once the loads would wait for
      // each other).  Loads ahead stand behind no branch (behind the last chunk it is loaded again): a wait then counts
      // them exactly.
      const float keep = scc[63];
      const uint16_t* tn = reinterpret_cast<const uint16_t*>(work + next * delta_chunk_bytes(NO));
      B8 ep[2][3];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        f32x4 em[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 e = *reinterpret_cast<const float4*>(scc + 64 + 32 * s + 16 * i + 4 * g);
          em[i] = f32x4{m[2 * s + i][0] * e.x, m[2 * s + i][1] * e.y, m[2 * s + i][2] * e.z, m[2 * s + i][3] * e.w};
        }
        split2<3>(em[0], em[1], ep[s]);
      }
#pragma unroll
      for (int j = 0; j < S; ++j) {
        if (j + 1 < S) pair_keys(j + 1);
        f32x4 y[2] = {st[2 * j] * keep, st[2 * j + 1] * keep};
#pragma unroll
        for (int s = 0; s < 2; ++s) mma_many<3, true>(kf[j & 1][s], ep[s], y);
        st[2 * j] = y[0];
        st[2 * j + 1] = y[1];
        constexpr int per = (kDFrags + S - 1) / S;
#pragma unroll
        for (int f = j * per; f < (j + 1) * per; ++f)
          if (f < kDFrags) stored_parts<3>(tn, f, tf[f], lane);
        if (j > 0) publish(j - 1);
        hold_order();
      }
      if (cut < 64) {
#pragma unroll
        for (int i = 0; i < NT; ++i) st[i] = f32x4{1.f, 1.f, 1.f, 1.f} * __builtin_nanf("");
      }
      if (__any(cut < 64)) {
#pragma unroll
        for (int s = 0; s + 1 < S; ++s) publish(s);
      }
      publish(S - 1);
      row_keys(kt + stage(c + 1) * NI * L::kpart, 0);  // (there since the chunk's first barrier)
      if constexpr (!LOCAL) __syncthreads();
    }
    if (map) state_store<NT>(st, a.part_map + (part * all + head) * a.N * a.N, p0, a.N, a.N);
    else if (LOCAL) state_store<NT>(st, a.part_state + (part * all + head) * cells, p0, a.P, a.N);
    else if (part == a.parts - 1) state_store<NT>(st, a.memory_out + head * cells, p0, a.P, a.N);
  } else {
    B8 pf[kDFrags][NO];
    auto weights = [&](int want) {
      const int c = want < chunks ? want : chunks - 1;
      stored_triangle<NO>(reinterpret_cast<const uint16_t*>(work + c * delta_chunk_bytes(NO)) + 3 * kDFrags * kDFragElems, pf, lane);
    };
    begin();
    __syncthreads();
    const int p = p0 + 4 * g, row = a.H * a.P * static_cast<int>(sizeof(raw));
    for (int c = first; c < chunks; ++c) {
      const int64_t t0 = static_cast<int64_t>(c) * kDTokens;
      // (Loads are dealt to both halves of a chunk: the state waves call for their matrix in the second one.)
      weights(c);
      place_k(c + 1);
      if constexpr (QV == 2) place_qv(c + 1);
      warm_up(c + 3);
      const uint16_t* qc = qt + (c & (QV - 1)) * L::qstage;
      // S Q^T: a value a row, a token a column, as rows are stored.
      f32x4 o[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < S; ++s) {
        B8 qf[4][NI], so[NO];
#pragma unroll
        for (int i = 0; i < NO; ++i) so[i] = __builtin_bit_cast(B8, *reinterpret_cast<const uint4*>(sf + (s * NO + i) * kDFragElems));
#pragma unroll
        for (int t = 0; t < 4; ++t) row_parts_t<QT, NI>(qc, L::qpart, 16 * t, 32 * s, qf[t]);
        mma_many<NO, false>(qf, so, o);
      }
      const float* scc = sc + (c & 1) * L::SCAL;
#pragma unroll
      for (int t = 0; t < 4; ++t) o[t] *= scc[16 * t + n];
      __syncthreads();
      f32x4 m[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) m[t] = mf[64 * t];
      const int cut = cuts[16 * w + n];
      {
        B8 mp[2][NO];
#pragma unroll
        for (int s = 0; s < 2; ++s) split2<NO>(m[2 * s], m[2 * s + 1], mp[s]);
        mma_triangle<NO, true, false>(pf, mp, o);
      }
      if constexpr (QV == 1) place_qv(c + 1);
      fetch(c + 2);
      if (__any(cut < 64)) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int f = __shfl(cut, 4 * g + r);
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (16 * t + n >= f) o[t][r] = __builtin_nanf("");
        }
      }
      if (t0 + kDTokens > len) clear_rows(o, len - t0);
      const int64_t left = a.T - t0;
      const __amdgpu_buffer_rsrc_t to =
          make_rsrc(static_cast<raw*>(a.hidden) + ((static_cast<int64_t>(b) * a.T + t0) * a.H + h) * a.P, 0x7ffffff0u);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int tok = 16 * t + n;
        if (VEC) {
          buf_store4<E>(to, tok < left && p < a.P ? tok * row + p * static_cast<int>(sizeof(raw)) : kBufOOB, o[t]);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            buf_store1<E>(to, tok < left && p + r < a.P ? tok * row + (p + r) * static_cast<int>(sizeof(raw)) : kBufOOB, o[t][r]);
        }
      }
      if constexpr (SAVE) {
        const __amdgpu_buffer_rsrc_t ms =
            make_rsrc(a.miss + ((static_cast<int64_t>(b) * a.T + t0) * a.H + h) * a.P, 0x7ffffff0u);
        rows_out<VEC>(m, ms, a.H * a.P * 4, len - t0, p0, a.P);
      }
      __syncthreads();
    }
    // Rows of this part behind the last chunk.
    const int64_t end = min_i64(a.T, (static_cast<int64_t>(first) + a.part_chunks) * kDTokens);
    for (int64_t t = static_cast<int64_t>(chunks) * kDTokens + tid / 16; t < end; t += kWalkThreads / 16) {
      raw* to = static_cast<raw*>(a.hidden) + ((b * a.T + t) * a.H + h) * a.P + col0;
      for (int i = tid % 16; i < kDCols && col0 + i < a.P; i += 16) to[i] = 0;
    }
  }
}

// The state before every part but the first: M_{p+1} = M_p F_p + D_p with the parts' maps F and what they leave of a zero
// state D (of the first, of the sequence's own state: M_1).  A workgroup takes 16 value rows through all parts; each wave
// holds 32 of the keys, and they hand each other the state's fragments.  The map hangs on no state and is loaded a part
// ahead.  A chain of loads: 26-29 us for 7 parts of 16 heads of 128 x 128 (155 with a wave for all keys and no loads ahead).
// A part behind a sequence's length hands its state on as it is: the product with the identity would make NaN of a row with
// an infinity, and of numbers that round to one in 16 bits.
template <int NK>
__global__ __launch_bounds__(2 * NK) void delta_join_kernel(DeltaArgs a) {
  constexpr int S = NK / 32;
  __shared__ __attribute__((aligned(16))) uint16_t frags[S * 3 * kDFragElems];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = lane_id(), g = lane >> 4, n = lane & 15;
  const int tiles = (a.P + 15) / 16, p0 = static_cast<int>(blockIdx.x % tiles) * 16;
  const int64_t head = blockIdx.x / tiles, cells = static_cast<int64_t>(a.P) * a.N, all = static_cast<int64_t>(a.B) * a.H;
  float map[2][S][8];
  auto fetch = [&](int want) {
    const int p = want < a.parts - 1 ? want : a.parts - 2;
    const __amdgpu_buffer_rsrc_t r = make_rsrc(a.part_map + (p * all + head) * a.N * a.N, static_cast<uint32_t>(a.N * a.N * 4));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int s = 0; s < S; ++s) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int from = 32 * s + (e < 4 ? 4 * g + e : 12 + 4 * g + e), to = 32 * w + 16 * i + n;
          map[i][s][e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, from < a.N && to < a.N ? (from * a.N + to) * 4 : kBufOOB, 0, 0));
        }
      }
    }
  };
  // This wave's tiles of a state: value row p0 + n, keys 32 w + 16 i + 4 g + r.
  auto where = [&](int i, int r) {
    const int key = 32 * w + 16 * i + 4 * g + r;
    return p0 + n < a.P && key < a.N ? ((p0 + n) * a.N + key) * 4 : kBufOOB;
  };
  auto rsrc = [&](int p) { return make_rsrc(a.part_state + (p * all + head) * cells, static_cast<uint32_t>(cells * 4)); };
  f32x4 st[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int r = 0; r < 4; ++r) st[i][r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rsrc(0), where(i, r), 0, 0));
  }
  fetch(1);
  const int have = static_cast<int>((delta_length(a, static_cast<int>(head / a.H)) + kDTokens - 1) / kDTokens);
  for (int p = 1; p < a.parts - 1; ++p) {
    if ((a.mirror ? a.parts - 1 - p : p) * a.part_chunks >= have) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int r = 0; r < 4; ++r) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(st[i][r]), rsrc(p), where(i, r), 0, 0);
      }
      fetch(p + 1);
      continue;
    }
    B8 sp[3], f[2][S][3];
    split2<3>(st[0], st[1], sp);
#pragma unroll
    for (int q = 0; q < 3; ++q) *reinterpret_cast<uint4*>(frags + (w * 3 + q) * kDFragElems + 8 * lane) = __builtin_bit_cast(uint4, sp[q]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) st[i][r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rsrc(p), where(i, r), 0, 0));
#pragma unroll
      for (int s = 0; s < S; ++s) split8<3>(map[i][s], f[i][s]);
    }
    fetch(p + 1);
    __syncthreads();
#pragma unroll
    for (int s = 0; s < S; ++s) {
      B8 m[3], fs[2][3];
#pragma unroll
      for (int q = 0; q < 3; ++q) {
        m[q] = __builtin_bit_cast(B8, *reinterpret_cast<const uint4*>(frags + (s * 3 + q) * kDFragElems + 8 * lane));
        fs[0][q] = f[0][s][q];
        fs[1][q] = f[1][s][q];
      }
      mma_many<3, true>(fs, m, st);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(st[i][r]), rsrc(p), where(i, r), 0, 0);
    }
  }
}

// One token.  LPR lanes share a state row, which is read and written once: its product with k is summed over them, the row moves
// by u k in their registers, and its product with q is summed.  Bound by those bytes: 27.7 us for 64 sequences x 16 heads of
// 128 x 128 (134 MB, 4.9 TB/s, what a large copy reaches).
template <class E, int LPR>
__global__ __launch_bounds__(kStepThreads) void delta_step_kernel(DeltaArgs a) {
  using raw = typename ET<E>::raw;
  constexpr int RPW = 64 / LPR, U = 4;
  const int lane = lane_id(), wave = static_cast<int>(threadIdx.x) >> 6;
  const uint32_t head = blockIdx.x;
  const int h = static_cast<int>(head % a.H), b = static_cast<int>(head / a.H), gi = h / (a.H / a.G);
  const int col = 4 * (lane % LPR);
  const bool whole = (a.N & 3) == 0;
  float k[4], q[4];
  const raw* kp = static_cast<const raw*>(a.keys) + b * a.kb + static_cast<int64_t>(gi) * a.N;
  const raw* qp = static_cast<const raw*>(a.queries) + b * a.qb + static_cast<int64_t>(gi) * a.N;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const bool in = col + r < a.N;
    k[r] = in ? ET<E>::to_f(kp[col + r]) : 0.f;
    q[r] = in ? ET<E>::to_f(qp[col + r]) : 0.f;
  }
  const int64_t is = b * a.sb + h, id = b * a.db + h;
  const float bt = a.s_f32 ? static_cast<const float*>(a.strengths)[is] : ET<E>::to_f(static_cast<const raw*>(a.strengths)[is]);
  float keep = 1.f;
  if (a.decays != nullptr)
    keep = expf(a.d_f32 ? static_cast<const float*>(a.decays)[id] : ET<E>::to_f(static_cast<const raw*>(a.decays)[id]));
  const raw* xp = static_cast<const raw*>(a.values) + b * a.vb + static_cast<int64_t>(h) * a.P;
  const float* mp = a.memory + static_cast<int64_t>(head) * a.P * a.N;
  float* op = a.memory_out + static_cast<int64_t>(head) * a.P * a.N;
  raw* hp = static_cast<raw*>(a.hidden) + static_cast<int64_t>(head) * a.P;
  const int stride = static_cast<int>(gridDim.y) * 4 * RPW * U;
  for (int p0 = (static_cast<int>(blockIdx.y) * 4 + wave) * RPW * U; p0 < a.P; p0 += stride) {
    f32x4 m[U];
    float x[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int p = p0 + i * RPW + lane / LPR;
      m[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      x[i] = p < a.P ? ET<E>::to_f(xp[p]) : 0.f;
      if (p < a.P && col < a.N) {
        const float* s = mp + static_cast<int64_t>(p) * a.N + col;
        if (whole) {
          m[i] = *reinterpret_cast<const f32x4*>(s);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) m[i][r] = col + r < a.N ? s[r] : 0.f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int p = p0 + i * RPW + lane / LPR;
#pragma unroll
      for (int r = 0; r < 4; ++r) m[i][r] *= keep;
      float mk = fmaf(m[i][0], k[0], fmaf(m[i][1], k[1], fmaf(m[i][2], k[2], m[i][3] * k[3])));
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) mk += __shfl_xor(mk, o);
      const float u = bt * (x[i] - mk);
#pragma unroll
      for (int r = 0; r < 4; ++r) m[i][r] = fmaf(u, k[r], m[i][r]);
      float y = fmaf(m[i][0], q[0], fmaf(m[i][1], q[1], fmaf(m[i][2], q[2], m[i][3] * q[3])));
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) y += __shfl_xor(y, o);
      if (p < a.P && col < a.N) {
        float* s = op + static_cast<int64_t>(p) * a.N + col;
        if (whole) {
          *reinterpret_cast<f32x4*>(s) = m[i];
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (col + r < a.N) s[r] = m[i][r];
        }
      }
      if (p < a.P && lane % LPR == 0) hp[p] = ET<E>::from_f(y);
    }
  }
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int set_lds(const void* kernel, size_t bytes, const char* what) {
  const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e != hipSuccess) {
    set_error("%s: %s", what, hipGetErrorString(e));
    return static_cast<int>(e);
  }
  return GRM_HIP_OK;
}

int out_parts(int dtype) { return dtype == GRM_HIP_F32 ? 3 : 2; }
int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }

struct Work {
  int64_t states, maps, bytes;
};
Work work_of(int64_t B, int64_t T, int64_t H, int64_t P, int64_t N, int dtype, int* parts, int64_t* part_chunks) {
  const int64_t C = (T + kDTokens - 1) / kDTokens;
  *parts = delta_time_parts(B * H, P, N, C, dtype, false, part_chunks);
  Work w{};
  w.states = up16(B * H * C * delta_chunk_bytes(out_parts(dtype)));
  w.maps = w.states + up16((*parts - 1) * B * H * P * N * 4);
  w.bytes = w.maps + (*parts - 1) * B * H * N * N * 4;
  return w;
}

}  // namespace

// Time parts of a sequence.  256 CUs hold a workgroup each; a part costs its chunks once more, for the value rows and for
// the N rows of its map, so parts are taken where they shorten the longest line of chunks behind each other (in quarters of
// a chunk's time; one of the first walk, with two chains a SIMD, takes five, of the mirror's four, a launch and a join a
// few chunks).  32768 bf16 tokens x 16 heads of 128 x 128: 1900 us in one part, 640 in eight.  The prices are those of bfloat16
// keys of 128, and are taken for every form; where sequences have 13 to 30 chunks (4 x 1000 float32 tokens x 8 heads of 64 x 64 take
// one part) they have not been set against times of parts.
int delta_time_parts(int64_t seqs, int64_t P, int64_t N, int64_t C, int dtype, bool mirror, int64_t* part_chunks) {
  *part_chunks = C;
  if ((dtype != GRM_HIP_BF16 && N > 64) || seqs > 4096) return 1;  // (delta_walk_kernel and delta_reverse_kernel take whole sequences)
  const int64_t PT = (P + kDCols - 1) / kDCols, NT = (N + kDCols - 1) / kDCols;
  auto rounds = [](int64_t wgs) { return (wgs + 255) / 256; };
  int64_t best = 4 * C * rounds(seqs * PT), parts = 1;
  for (int64_t r = 2; r <= 64 && r <= C / 4; ++r) {
    const int64_t per = (C + r - 1) / r, n = (C + per - 1) / per;
    const int64_t first = mirror ? 4 * rounds(seqs * (PT + NT) * (n - 1)) : 5 * rounds(seqs * ((PT + NT + 1) / 2) * (n - 1));
    const int64_t cost = per * (4 * rounds(seqs * PT * n) + first) + 8 * n + 24;
    if (cost < best) best = cost, parts = n, *part_chunks = per;
  }
  return static_cast<int>(parts);
}

int delta_check(const grm_hip_delta_args* u, const char* what, bool step) {
  auto bad = [&](const char* why) {
    set_error("%s: %s", what, why);
    return GRM_HIP_EINVAL;
  };
  if (u == nullptr) return bad("no arguments");
  if (u->batch < 0 || u->seq_len < 0 || u->heads < 1 || u->value_dim < 1 || u->groups < 1 || u->key_dim < 1)
    return bad("batch and seq_len must be >= 0, the other sizes >= 1");
  if (u->heads % u->groups != 0) return bad("heads must be a multiple of groups");
  if (u->dtype < 0 || u->dtype > 2 || (u->strengths_dtype != u->dtype && u->strengths_dtype != GRM_HIP_F32) ||
      (u->decays_dtype != u->dtype && u->decays_dtype != GRM_HIP_F32)) {
    set_error("%s: keys, values and queries must be float32, float16 or bfloat16, strengths and log_decays the same or float32", what);
    return GRM_HIP_EUNSUPPORTED;
  }
  if (u->key_dim > 128) {
    set_error("%s: key_dim must be <= 128, got %lld", what, static_cast<long long>(u->key_dim));
    return GRM_HIP_EUNSUPPORTED;
  }
  if (const char* limit = delta_limit(u->batch, u->seq_len, u->heads, u->value_dim, u->groups, u->key_dim, step)) {
    set_error("%s: %s", what, limit);
    return GRM_HIP_EUNSUPPORTED;
  }
  const int64_t most = int64_t{1} << 21;
  if (u->keys_token_stride < 0 || u->keys_token_stride > most || u->values_token_stride < 0 || u->values_token_stride > most ||
      u->queries_token_stride < 0 || u->queries_token_stride > most) {
    set_error("%s: token strides and row widths must be at most 2^21 elements", what);
    return GRM_HIP_EUNSUPPORTED;
  }
  if (u->seq_len > 1 && (u->keys_token_stride < u->groups * u->key_dim || u->queries_token_stride < u->groups * u->key_dim ||
                         u->values_token_stride < u->heads * u->value_dim))
    return bad("token strides must not be below a row's width");
  if (u->batch > 0 && u->seq_len > 0 &&
      (u->keys == nullptr || u->values == nullptr || u->queries == nullptr || u->strengths == nullptr))
    return bad("keys, values, queries and strengths are required");
  if (!aligned(u->memory)) return bad("memory must be 16-byte aligned");
  return GRM_HIP_OK;
}

DeltaArgs delta_args(const grm_hip_delta_args* u) {
  DeltaArgs a{};
  a.keys = u->keys; a.values = u->values; a.queries = u->queries;
  a.strengths = u->strengths; a.decays = u->log_decays; a.lengths = u->lengths; a.memory = u->memory;
  a.kb = u->keys_batch_stride; a.kt = u->keys_token_stride;
  a.vb = u->values_batch_stride; a.vt = u->values_token_stride;
  a.qb = u->queries_batch_stride; a.qt = u->queries_token_stride;
  a.sb = u->strengths_batch_stride; a.st = u->strengths_token_stride;
  a.db = u->decays_batch_stride; a.dt = u->decays_token_stride;
  a.T = u->seq_len;
  a.B = static_cast<int>(u->batch); a.H = static_cast<int>(u->heads); a.P = static_cast<int>(u->value_dim);
  a.G = static_cast<int>(u->groups); a.N = static_cast<int>(u->key_dim);
  a.C = static_cast<int>((u->seq_len + kDTokens - 1) / kDTokens);
  a.PT = static_cast<int>((u->value_dim + kDCols - 1) / kDCols);
  a.NT = static_cast<int>((u->key_dim + kDCols - 1) / kDCols);
  a.parts = 1;
  a.part_chunks = a.C;
  a.s_f32 = u->strengths_dtype == GRM_HIP_F32;
  a.d_f32 = u->decays_dtype == GRM_HIP_F32;
  // Whole 16-byte loads where every row of 8-element units allows them.
  a.vec = u->value_dim % 8 == 0 && u->key_dim % 8 == 0 && aligned(u->keys) && aligned(u->values) &&
          aligned(u->queries) && (u->keys_batch_stride | u->keys_token_stride | u->values_batch_stride |
                                  u->values_token_stride | u->queries_batch_stride | u->queries_token_stride) % 8 == 0;
  return a;
}

int launch_delta_prep(const DeltaArgs& a, int dtype, bool back, hipStream_t stream, const char* what) {
  int rc = GRM_HIP_OK;
  delta_with_form(dtype, a.N, a.vec != 0, [&](auto e, auto nk, auto vec) {
    using E = decltype(e);
    constexpr int NK = decltype(nk)::value;
    constexpr bool VEC = decltype(vec)::value;
    auto go = [&](auto kernel) {
      constexpr size_t lds = PrepLds<E, NK>::bytes;
      if ((rc = set_lds(reinterpret_cast<const void*>(kernel), lds, what)) != GRM_HIP_OK) return;
      kernel<<<dim3(static_cast<uint32_t>(a.B) * a.H * a.C), dim3(kPrepThreads), lds, stream>>>(a);
      rc = check_launch(what);
    };
    if (back) go(delta_prep_kernel<E, NK, VEC, true>);
    else go(delta_prep_kernel<E, NK, VEC, false>);
  });
  return rc;
}

int launch_delta_join(const DeltaArgs& a, hipStream_t stream, const char* what) {
  if (a.parts <= 2) return GRM_HIP_OK;  // (the first part's end is the second one's start)
  const dim3 grid(static_cast<uint32_t>(a.B) * a.H * ((a.P + 15) / 16));
  if (a.N <= 64) delta_join_kernel<64><<<grid, dim3(128), 0, stream>>>(a);
  else delta_join_kernel<128><<<grid, dim3(256), 0, stream>>>(a);
  return check_launch(what);
}

}  // namespace grmhip

using namespace grmhip;

extern "C" int64_t grm_hip_delta_scan_workspace(int64_t batch, int64_t seq_len, int64_t heads, int64_t value_dim, int64_t key_dim,
                                                int dtype) {
  if (batch <= 0 || seq_len <= 0 || heads <= 0 || value_dim <= 0 || key_dim <= 0 || dtype < 0 || dtype > 2) return 0;
  int parts = 1;
  int64_t part_chunks = 0;
  return work_of(batch, seq_len, heads, value_dim, key_dim, dtype, &parts, &part_chunks).bytes;
}

extern "C" int grm_hip_delta_scan_fwd(const grm_hip_delta_args* u, void* hidden, float* memory_out, float* states,
                                      float* miss, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "delta_scan";
  if (int rc = delta_check(u, what, false)) return rc;
  if (u->batch == 0) return GRM_HIP_OK;
  const int64_t state_bytes = u->batch * u->heads * u->value_dim * u->key_dim * 4;
  if (memory_out == nullptr || (u->seq_len > 0 && hidden == nullptr) || !aligned(memory_out) || !aligned(states)) {
    set_error("%s: hidden and memory_out are required, memory_out and states 16-byte aligned", what);
    return GRM_HIP_EINVAL;
  }
  if ((states == nullptr) != (miss == nullptr)) {
    set_error("%s: states and miss are given both or neither", what);
    return GRM_HIP_EINVAL;
  }
  if (ranges_overlap(u->memory, state_bytes, memory_out, state_bytes)) {
    set_error("%s: memory_out may not overlap memory", what);
    return GRM_HIP_EINVAL;
  }
  DeltaArgs a = delta_args(u);
  a.hidden = hidden; a.memory_out = memory_out; a.states = states; a.miss = miss;
  a.work = static_cast<char*>(workspace);
  if (a.C > 0) {
    int64_t part_chunks = 0;
    const Work wk = work_of(u->batch, u->seq_len, u->heads, u->value_dim, u->key_dim, u->dtype, &a.parts, &part_chunks);
    a.part_chunks = static_cast<int>(part_chunks);
    a.part_state = reinterpret_cast<float*>(a.work + wk.states);
    a.part_map = reinterpret_cast<float*>(a.work + wk.maps);
    if (workspace == nullptr || !aligned(workspace) || workspace_bytes < wk.bytes) {
      set_error("%s: workspace missing, misaligned or too small", what);
      return GRM_HIP_EINVAL;
    }
    if (int rc = launch_delta_prep(a, u->dtype, false, static_cast<hipStream_t>(stream), what)) return rc;
  }
  int rc = GRM_HIP_OK;
  delta_with_form(u->dtype, a.N, a.vec != 0 && aligned(hidden), [&](auto e, auto nk, auto vec) {
    using E = decltype(e);
    constexpr int NK = decltype(nk)::value;
    const uint32_t heads = static_cast<uint32_t>(a.B) * a.H;
    if constexpr (PairLds<E, NK>::fits) {
      constexpr bool V = decltype(vec)::value;
      auto go = [&](auto kernel, uint32_t grid, size_t lds) {
        if ((rc = set_lds(reinterpret_cast<const void*>(kernel), lds, what)) != GRM_HIP_OK) return;
        kernel<<<dim3(grid), dim3(2 * kWalkThreads), lds, static_cast<hipStream_t>(stream)>>>(a);
        rc = check_launch(what);
      };
      if (a.parts > 1) {
        go(delta_pair_kernel<E, NK, V, false, true>, heads * ((a.PT + a.NT + 1) / 2) * (a.parts - 1), LocalLds<E, NK>::bytes);
        if (rc != GRM_HIP_OK) return;
        if ((rc = launch_delta_join(a, static_cast<hipStream_t>(stream), what)) != GRM_HIP_OK) return;
      }
      if (states != nullptr) go(delta_pair_kernel<E, NK, V, true, false>, heads * a.PT * a.parts, PairLds<E, NK>::bytes);
      else go(delta_pair_kernel<E, NK, V, false, false>, heads * a.PT * a.parts, PairLds<E, NK>::bytes);
    } else {
      auto kernel = delta_walk_kernel<E, NK, decltype(vec)::value>;
      constexpr size_t lds = WalkLds<E, NK>::bytes;
      if ((rc = set_lds(reinterpret_cast<const void*>(kernel), lds, what)) != GRM_HIP_OK) return;
      kernel<<<dim3(heads * a.PT), dim3(kWalkThreads), lds, static_cast<hipStream_t>(stream)>>>(a);
      rc = check_launch(what);
    }
  });
  return rc;
}

extern "C" int grm_hip_delta_step(const grm_hip_delta_args* u, void* hidden, float* memory_out, void* stream) {
  const char* what = "delta_step";
  if (int rc = delta_check(u, what, true)) return rc;
  if (u->seq_len != 1 || u->lengths != nullptr) {
    set_error("%s: seq_len must be 1, without lengths", what);
    return GRM_HIP_EINVAL;
  }
  if (u->batch == 0) return GRM_HIP_OK;
  if (u->memory == nullptr || hidden == nullptr || memory_out == nullptr || !aligned(memory_out)) {
    set_error("%s: memory, hidden and memory_out are required, memory_out 16-byte aligned", what);
    return GRM_HIP_EINVAL;
  }
  const int64_t state_bytes = u->batch * u->heads * u->value_dim * u->key_dim * 4;
  if (memory_out != u->memory && ranges_overlap(u->memory, state_bytes, memory_out, state_bytes)) {
    set_error("%s: memory_out must be memory itself or not overlap it", what);
    return GRM_HIP_EINVAL;
  }
  DeltaArgs a = delta_args(u);
  a.hidden = hidden; a.memory_out = memory_out;
  auto go = [&](auto e, auto lpr) {
    constexpr int LPR = decltype(lpr)::value, rows = 4 * (64 / LPR) * 4;  // of a workgroup at a time
    const int64_t tiles = (a.P + rows - 1) / rows, most = 65535;  // a grid's second dimension; the kernel goes round
    delta_step_kernel<decltype(e), LPR>
        <<<dim3(static_cast<uint32_t>(a.B) * a.H, static_cast<uint32_t>(tiles < most ? tiles : most)), dim3(kStepThreads), 0,
           static_cast<hipStream_t>(stream)>>>(a);
  };
  auto by_width = [&](auto e) {
    if (a.N <= 16) go(e, std::integral_constant<int, 4>{});
    else if (a.N <= 32) go(e, std::integral_constant<int, 8>{});
    else if (a.N <= 64) go(e, std::integral_constant<int, 16>{});
    else go(e, std::integral_constant<int, 32>{});
  };
  if (u->dtype == GRM_HIP_F32) by_width(F32{});
  else if (u->dtype == GRM_HIP_F16) by_width(F16{});
  else by_width(BF16{});
  return check_launch(what);
}
