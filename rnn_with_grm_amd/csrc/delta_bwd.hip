// Gradients of the gated delta rule.  With the states S before every chunk and m from the forward (delta.h), and G the gradient
// of the state behind a chunk:
//   z  = (W * Q K^T)^T dH + E K G^T,  du = (I + b A)^-T z       (du: of what a token writes, u = b m)
//   G0 = e^{c_63} G + (D dH)^T Q - (D b du)^T K,  dV = b du,  db = sum_p du m
//   Y  = W b_j (dH m^T)  (j <= i),  X = -W b_i b_j (du m^T)  (j < i)
//   dQ = D dH S + Y K,  dK = -D b du S + E b m G + Y^T Q + (X + X^T) K
// and for the log decays, with T = X * K K^T + Y * Q K^T and e_j = k_j.(E b m G)_j, dc_i = row sums less column sums of T (j < i)
// + q_i.(D dH S)_i - k_i.(D b du S)_i - e_i; dg_t = sum_{i >= t} dc_i + sum_j e_j + e^{c_63} <G, S>.  (The column sums are
// b m.du less e, and the rows' dh.h - dv.(v - m) in all, without a sum over pairs; but those are rounded apart from each other and
// leave 8e-7 to 2e-6 of dg's norm where decays are weak, the sums over pairs 1e-7 to 4e-7.)
// The walk over the chunks from the last to the first leaves du and G (delta_reverse_kernel); all else is done for all chunks
// side by side (delta_grad_kernel).  No atomics: sums are taken in a fixed order.
#include "delta.h"

namespace grmhip {
namespace {

constexpr int kThreads = 256;
constexpr int kGradThreads = 512;
constexpr int kGradWaves = 2;  // a SIMD

struct DeltaBwdArgs {
  DeltaArgs f;
  const void* dhidden;    // [B, T, H, P]
  const float* dmemory;   // [B, H, P, N] or null: of memory_out
  float* gstates;         // [B, C, H, P, N]: G behind every chunk
  float* du;              // [B, T, H, P]
  void *dk, *dv, *dq, *ds, *dd;
  float* dm;              // [B, H, P, N]
  float* part;            // [2, shares, B, T, G, N] or null: dk and dq of a share of a group's heads
  int shares, per;        // shares of a group's heads, heads of a share
  int whole;              // four keys' gradients leave in one store
};

template <class E, int NK>
struct ReverseLds {
  using KT = SelTile<BF16, NK, true>;
  using VT = SelTile<E, kDCols, true>;
  static constexpr int NI = DParts<E>::IN, kpart = kDTokens * KT::STRIDE;
  static constexpr size_t k = 0, q = k + NI * kpart * 2, v = q + NI * kpart * 2,
                          s = v + kDTokens * VT::STRIDE * sizeof(typename ET<E>::raw), bytes = s + 192 * 4;
};

// Two accumulators scaled by what sc holds for their tokens (row tiles t0 and t0 + 1 of 16), in three parts.
__device__ __forceinline__ void scaled_pair(const f32x4& lo, const f32x4& hi, const float* sc, int g, B8 (&out)[3]) {
  const float4 a = *reinterpret_cast<const float4*>(sc + 4 * g), b = *reinterpret_cast<const float4*>(sc + 16 + 4 * g);
  split2<3>(f32x4{lo[0] * a.x, lo[1] * a.y, lo[2] * a.z, lo[3] * a.w},
                      f32x4{hi[0] * b.x, hi[1] * b.y, hi[2] * b.z, hi[3] * b.w}, out);
}

// The same where two stages of keys do not fit into LDS (float16 and float32 keys wider than 64): four waves that do all of it, in
// one time part.  8 x 2048 tokens x 16 heads of 128 x 128 with gradients, whole calls: 1.38 ms in float16, 1.90 in float32 (bfloat16
// by the other kernel 0.95-0.98); 16384 tokens x 16 heads 5.7 and 8.3 (1.36).
template <class E, int NK, bool VEC>
__global__ __launch_bounds__(kThreads) void delta_reverse_kernel(DeltaBwdArgs ba) {
  using raw = typename ET<E>::raw;
  using L = ReverseLds<E, NK>;
  using KT = typename L::KT;
  using VT = typename L::VT;
  constexpr int NI = L::NI, S = NK / 32, NT = NK / 16;
  const DeltaArgs& a = ba.f;
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

  const raw* kp = static_cast<const raw*>(a.keys) + b * a.kb + static_cast<int64_t>(gi) * a.N;
  const raw* qp = static_cast<const raw*>(a.queries) + b * a.qb + static_cast<int64_t>(gi) * a.N;
  const int64_t row = static_cast<int64_t>(a.H) * a.P;
  const raw* vp = static_cast<const raw*>(ba.dhidden) + b * a.T * row + static_cast<int64_t>(h) * a.P + col0;
  const char* work = a.work + (static_cast<int64_t>(b) * a.H + h) * a.C * delta_chunk_bytes(3);
  TileLoad<E, KT, BF16, VEC, kDTokens, NK, kThreads> kl, ql;
  TileLoad<E, VT, E, VEC, kDTokens, kDCols, kThreads> vl;
  kl.init(a.kt, a.N, tid);
  ql.init(a.qt, a.N, tid);
  vl.init(row, a.P - col0 < kDCols ? a.P - col0 : kDCols, tid);
  float sreg = 0.f;
  auto fetch = [&](int c) {
    const int64_t t0 = static_cast<int64_t>(c) * kDTokens;
    kl.load(kp + t0 * a.kt, len - t0, tid);
    ql.load(qp + t0 * a.qt, len - t0, tid);
    vl.load(vp + t0 * row, len - t0, tid);
    if (tid < 192)
      sreg = reinterpret_cast<const float*>(work + c * delta_chunk_bytes(3) + 6 * kDFrags * kDFragElems * 2)[tid];
  };
  f32x4 st[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) st[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int64_t head = static_cast<int64_t>(b) * a.H + h, cells = static_cast<int64_t>(a.P) * a.N;
  if (ba.dmemory != nullptr) state_add<NT>(st, ba.dmemory + head * cells, p0, a.P, a.N, 1.f);
  if (chunks > 0) fetch(chunks - 1);

  for (int c = chunks - 1; c >= 0; --c) {
    const int64_t t0 = static_cast<int64_t>(c) * kDTokens;
    __syncthreads();
    store_parts<KT, NI, E>(kl, kt, L::kpart, kDTokens, tid);
    store_parts<KT, NI, E>(ql, qt, L::kpart, kDTokens, tid);
    vl.store(vt, tid);
    if (tid < 192) sc[tid] = sreg;
    __syncthreads();
    if (c > 0) fetch(c - 1);
    const uint16_t* tf = reinterpret_cast<const uint16_t*>(work + c * delta_chunk_bytes(3));
    const uint16_t* pf = tf + 3 * kDFrags * kDFragElems;
    state_store<NT>(st, ba.gstates + ((static_cast<int64_t>(b) * a.C + c) * a.H + h) * cells, p0, a.P, a.N);

    // z = E K G^T + (W * Q K^T)^T dH.
    f32x4 z[4], dh[4];
    {
      B8 gp[S][3];
#pragma unroll
      for (int s = 0; s < S; ++s) split2<3>(st[2 * s], st[2 * s + 1], gp[s]);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        z[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < S; ++s) {
          B8 kf[NI];
          row_parts_t<KT, NI>(kt, L::kpart, 16 * t, 32 * s, kf);
          z[t] = mma_parts<3>(kf, gp[s], z[t]);
        }
        const float4 e = *reinterpret_cast<const float4*>(sc + 64 + 16 * t + 4 * g);
        z[t] = f32x4{z[t][0] * e.x, z[t][1] * e.y, z[t][2] * e.z, z[t][3] * e.w};
      }
    }
    {
      B8 hp[2][NI];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const Frag8<E> f = col_frag<VT, E>(vt, 32 * s, 16 * w);
        input_parts<E, NI>(__builtin_bit_cast(U8<E>, f), hp[s]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          dh[2 * s][r] = ET<E>::to_f(f.e[r]);
          dh[2 * s + 1][r] = ET<E>::to_f(f.e[4 + r]);
        }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int s = t / 2; s < 2; ++s) {
          B8 f[3];
          stored_parts<3>(pf, upper_frag(t, s), f, lane);
          z[t] = mma_parts<3>(f, hp[s], z[t]);
        }
      }
    }
    f32x4 du[4];
    {
      B8 zp[2][3];
#pragma unroll
      for (int s = 0; s < 2; ++s) split2<3>(z[2 * s], z[2 * s + 1], zp[s]);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        du[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = t / 2; s < 2; ++s) {
          B8 f[3];
          stored_parts<3>(tf, upper_frag(t, s), f, lane);
          du[t] = mma_parts<3>(f, zp[s], du[t]);
        }
      }
    }
    if (p0 + n < a.P) {
      float* to = ba.du + (b * a.T + t0) * row + static_cast<int64_t>(h) * a.P + p0 + n;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int tok = 16 * t + 4 * g + r;
          if (t0 + tok < len) to[tok * row] = du[t][r];
        }
      }
    }
    // G0.
    const float keep = sc[63];
#pragma unroll
    for (int i = 0; i < NT; ++i) st[i] *= keep;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      B8 hp[3], up[3];
      scaled_pair(dh[2 * s], dh[2 * s + 1], sc + 32 * s, g, hp);
      const float4 b0 = *reinterpret_cast<const float4*>(sc + 128 + 32 * s + 4 * g),
                   b1 = *reinterpret_cast<const float4*>(sc + 144 + 32 * s + 4 * g);
      scaled_pair(f32x4{-du[2 * s][0] * b0.x, -du[2 * s][1] * b0.y, -du[2 * s][2] * b0.z, -du[2 * s][3] * b0.w},
                  f32x4{-du[2 * s + 1][0] * b1.x, -du[2 * s + 1][1] * b1.y, -du[2 * s + 1][2] * b1.z, -du[2 * s + 1][3] * b1.w},
                  sc + 32 * s, g, up);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        B8 kf[NI], qf[NI];
        col_parts<KT, NI>(qt, L::kpart, 32 * s, 16 * i, qf);
        col_parts<KT, NI>(kt, L::kpart, 32 * s, 16 * i, kf);
        st[i] = mma_parts<3>(qf, hp, st[i]);
        st[i] = mma_parts<3>(kf, up, st[i]);
      }
    }
  }
  state_store<NT>(st, ba.dm + head * cells, p0, a.P, a.N);
}

// LDS of the mirror walk in two halves.
template <class E, int NK>
struct MirrorLds {
  using KT = SelTile<BF16, NK, false>;  // read by rows and by columns
  using QT = SelTile<BF16, NK, true>;   // read by columns
  using VT = SelTile<E, kDCols, true>;
  static constexpr int NI = DParts<E>::IN, kpart = kDTokens * KT::STRIDE, qpart = kDTokens * QT::STRIDE, SCAL = 192, NT = NK / 16;
  static constexpr size_t k = 0, q = k + 2 * NI * kpart * 2, v = q + NI * qpart * 2,
                          z = v + kDTokens * VT::STRIDE * sizeof(typename ET<E>::raw), u = z + 4 * 4 * 64 * 16,
                          c = u + 4 * 4 * 64 * 16, s = c + 4 * NT * 64 * 16, bytes = s + 2 * SCAL * 4;
  static constexpr bool fits = bytes <= 160 * 1024;
};

// The walk's mirror: 64 value columns of the gradient's state a workgroup, chunks from the last to the first.  Four state
// waves run the chain that the next chunk hangs on (K G^T, du, the state's update by the keys); four output waves, one beside
// each on its SIMD, load the chunks ahead, form what hangs on no state, (W * Q K^T)^T dH and (D dH)^T Q, one chunk ahead, and
// store du.  Two barriers a chunk: du is there, the next state is there.
// Time parts as the walk's: a first launch (LOCAL) takes all parts but a sequence's first one from their ends to their
// beginnings, from a zero state and, without rows of values, from the identity's rows; the second each from its own
// (16384 bf16 tokens x 8 heads of 128 x 128: 1046 us in one part, in nine 129 and 163 with a join of 29 between).
// Bound by the chain, like the walk: 207-234 us for 8 x 2048 bf16 tokens x 16 heads of 128 x 128, 400 MB of states and du written.
template <class E, int NK, bool VEC, bool LOCAL>
__global__ __launch_bounds__(2 * kThreads, 2) void delta_mirror_kernel(DeltaBwdArgs ba) {
  using raw = typename ET<E>::raw;
  using L = MirrorLds<E, NK>;
  using KT = typename L::KT;
  using QT = typename L::QT;
  using VT = typename L::VT;
  constexpr int NI = L::NI, S = NK / 32, NT = NK / 16;
  const DeltaArgs& a = ba.f;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  uint16_t* kt = reinterpret_cast<uint16_t*>(lds + L::k);
  uint16_t* qt = reinterpret_cast<uint16_t*>(lds + L::q);
  raw* vt = reinterpret_cast<raw*>(lds + L::v);
  float* sc = reinterpret_cast<float*>(lds + L::s);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3;
  const int lane = lane_id(), g = lane >> 4, n = lane & 15;
  const uint32_t at = xcd_order(blockIdx.x, gridDim.x);
  const int tiles = LOCAL ? a.PT + a.NT : a.PT, parts = LOCAL ? a.parts - 1 : a.parts;
  const int pt = static_cast<int>(at % tiles), turn = static_cast<int>(at / tiles % parts);  // (the last part is the first in turn)
  const int h = static_cast<int>(at / tiles / parts % a.H), b = static_cast<int>(at / tiles / parts / a.H);
  const bool map = LOCAL && pt >= a.PT;  // rows of the identity
  if (map && turn == 0) return;
  const int64_t len = delta_length(a, b);
  const int col0 = (map ? pt - a.PT : pt) * kDCols, p0 = col0 + 16 * w, gi = h / (a.H / a.G), prows = map ? a.N : a.P;
  const int part = a.parts - 1 - turn, first = part * a.part_chunks, have = static_cast<int>((len + kDTokens - 1) / kDTokens);
  const int chunks = have < first + a.part_chunks ? (have > first ? have : first) : first + a.part_chunks;  // this part's end
  const int64_t all = static_cast<int64_t>(a.B) * a.H;
  const int64_t head = static_cast<int64_t>(b) * a.H + h, cells = static_cast<int64_t>(a.P) * a.N, row = static_cast<int64_t>(a.H) * a.P;
  const char* work = a.work + head * a.C * delta_chunk_bytes(3);
  f32x4* zf = reinterpret_cast<f32x4*>(lds + L::z) + w * 256 + lane;
  f32x4* uf = reinterpret_cast<f32x4*>(lds + L::u) + w * 256 + lane;
  f32x4* cf = reinterpret_cast<f32x4*>(lds + L::c) + w * NT * 64 + lane;

  if (wave < 4) {
    __builtin_amdgcn_s_setprio(2);
    f32x4 st[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) st[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (map) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int r = 0; r < 4; ++r) st[i][r] = p0 + n == 16 * i + 4 * g + r && p0 + n < a.N ? 1.f : 0.f;
      }
    } else if (turn > 0 && !LOCAL) {
      state_add<NT>(st, a.part_state + ((turn - 1) * all + head) * cells, p0, a.P, a.N, 1.f);
    } else if (turn == 0 && ba.dmemory != nullptr) {
      state_add<NT>(st, ba.dmemory + head * cells, p0, a.P, a.N, 1.f);
    }
    B8 tf[kDFrags][3], gp[S][3], kr[2][4][NI];
    auto row_keys = [&](const uint16_t* from, int s) {
#pragma unroll
      for (int t = 0; t < 4; ++t) row_parts_t<KT, NI>(from, L::kpart, 16 * t, 32 * s, kr[s & 1][t]);
    };
    auto keep_state = [&](int c) {  // (before the first chunk: behind the last value row, where nothing is stored)
      if constexpr (LOCAL) return;
#pragma unroll
      for (int s = 0; s < S; ++s)
        state_out<VEC>(st, 2 * s, ba.gstates + ((static_cast<int64_t>(b) * a.C + (c < first ? first : c)) * a.H + h) * cells,
                       c < first ? a.P : p0, a.P, a.N);
    };
#pragma unroll
    for (int s = 0; s < S; ++s) split2<3>(st[2 * s], st[2 * s + 1], gp[s]);
    if (chunks > first) {
      stored_triangle<3>(reinterpret_cast<const uint16_t*>(work + (chunks - 1) * delta_chunk_bytes(3)), tf, lane);
      keep_state(chunks - 1);
    }
    __syncthreads();
    __syncthreads();
    if (chunks > first) row_keys(kt + ((chunks - 1) & 1) * NI * L::kpart, 0);
    for (int c = chunks - 1; c >= first; --c) {
      const uint16_t* kc = kt + (c & 1) * NI * L::kpart;
      const float* scc = sc + (c & 1) * L::SCAL;
      const int next = c > first ? c - 1 : first;
      f32x4 z[4], z0[4];
      float4 e[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        z[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        z0[t] = zf[64 * t];
        e[t] = *reinterpret_cast<const float4*>(scc + 64 + 16 * t + 4 * g);
      }
      hold_order();
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (s + 1 < S) row_keys(kc, s + 1);
        mma_many<3, true>(kr[s & 1], gp[s], z);
        hold_order();
      }
      f32x4 du[4];
      {
        B8 zp[2][3];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          z[t] = f32x4{fmaf(z[t][0], e[t].x, z0[t][0]), fmaf(z[t][1], e[t].y, z0[t][1]), fmaf(z[t][2], e[t].z, z0[t][2]),
                       fmaf(z[t][3], e[t].w, z0[t][3])};
          du[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) split2<3>(z[2 * s], z[2 * s + 1], zp[s]);
        mma_triangle<3, false, true>(tf, zp, du);
      }
      if constexpr (!LOCAL) {
#pragma unroll
        for (int t = 0; t < 4; ++t) uf[64 * t] = du[t];
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
      // G0 = e^{c_63} G + (D dH)^T Q - (D b du)^T K, two tiles of keys at a time.
      const float keep = scc[63];
      const uint16_t* tn = reinterpret_cast<const uint16_t*>(work + next * delta_chunk_bytes(3));
      B8 ep[2][3];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        f32x4 em[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 d = *reinterpret_cast<const float4*>(scc + 32 * s + 16 * i + 4 * g),
                       bb = *reinterpret_cast<const float4*>(scc + 128 + 32 * s + 16 * i + 4 * g);
          const f32x4 v = du[2 * s + i];
          em[i] = f32x4{-v[0] * (d.x * bb.x), -v[1] * (d.y * bb.y), -v[2] * (d.z * bb.z), -v[3] * (d.w * bb.w)};
        }
        split2<3>(em[0], em[1], ep[s]);
      }
#pragma unroll
      for (int j = 0; j < S; ++j) {
        if (j + 1 < S) pair_keys(j + 1);
        f32x4 y[2] = {st[2 * j] * keep + cf[64 * (2 * j)], st[2 * j + 1] * keep + cf[64 * (2 * j + 1)]};
#pragma unroll
        for (int s = 0; s < 2; ++s) mma_many<3, true>(kf[j & 1][s], ep[s], y);
        st[2 * j] = y[0];
        st[2 * j + 1] = y[1];
        constexpr int per = (kDFrags + S - 1) / S;
#pragma unroll
        for (int f = j * per; f < (j + 1) * per; ++f)
          if (f < kDFrags) stored_parts<3>(tn, f, tf[f], lane);
        if (j > 0) split2<3>(st[2 * j - 2], st[2 * j - 1], gp[j - 1]);
        hold_order();
      }
      split2<3>(st[NT - 2], st[NT - 1], gp[S - 1]);
      keep_state(c - 1);
      row_keys(kt + (next & 1) * NI * L::kpart, 0);  // (there since the chunk's first barrier)
      __syncthreads();
    }
    if (map) state_store<NT>(st, a.part_map + (turn * all + head) * a.N * a.N, p0, a.N, a.N);
    else if (LOCAL) state_store<NT>(st, a.part_state + (turn * all + head) * cells, p0, a.P, a.N);
    else if (part == 0) state_store<NT>(st, ba.dm + head * cells, p0, a.P, a.N);
  } else {
    const int tid = static_cast<int>(threadIdx.x) - kThreads;
    const raw* kp = static_cast<const raw*>(a.keys) + b * a.kb + static_cast<int64_t>(gi) * a.N;
    const raw* qp = static_cast<const raw*>(a.queries) + b * a.qb + static_cast<int64_t>(gi) * a.N;
    const raw* vp = static_cast<const raw*>(ba.dhidden) + b * a.T * row + static_cast<int64_t>(h) * a.P + (map ? 0 : col0);
    TileLoad<E, KT, BF16, VEC, kDTokens, NK, kThreads> kl;
    TileLoad<E, QT, BF16, VEC, kDTokens, NK, kThreads> ql;
    TileLoad<E, VT, E, VEC, kDTokens, kDCols, kThreads> vl;
    kl.init(a.kt, a.N, tid);
    ql.init(a.qt, a.N, tid);
    vl.init(row, prows - col0 < kDCols ? prows - col0 : kDCols, tid);
    float sreg = 0.f, warm = 0.f;
    B8 pf[kDFrags][3];
    auto fetch = [&](int want) {  // (before the first chunk it is loaded again)
      const int c = want > first ? want : first;
      const int64_t t0 = static_cast<int64_t>(c) * kDTokens;
      sreg = reinterpret_cast<const float*>(work + c * delta_chunk_bytes(3) + 6 * kDFrags * kDFragElems * 2)[tid < 192 ? tid : 0];
      kl.load(kp + t0 * a.kt, len - t0, tid);
      ql.load(qp + t0 * a.qt, len - t0, tid);
      vl.load(vp + t0 * row, map ? 0 : len - t0, tid);  // (a map's rows have no values)
    };
    auto place = [&](int c) {
      store_parts<KT, NI, E>(kl, kt + (c & 1) * NI * L::kpart, L::kpart, kDTokens, tid);
      store_parts<QT, NI, E>(ql, qt, L::qpart, kDTokens, tid);
      vl.store(vt, tid);
      if (tid < 192) sc[(c & 1) * L::SCAL + tid] = sreg;
    };
    auto weights = [&](int want) {
      stored_triangle<3>(reinterpret_cast<const uint16_t*>(work + (want > first ? want : first) * delta_chunk_bytes(3)) + 3 * kDFrags * kDFragElems, pf, lane);
    };
    // One word of every line of a later chunk's matrices, so that they lie in the L2 when they are called for.
    auto warm_up = [&](int want) {
      asm volatile("" ::"v"(warm));
      constexpr int lines = static_cast<int>(delta_chunk_bytes(3) / 128);
      for (int i = tid; i < lines; i += kThreads) warm = *reinterpret_cast<const float*>(work + (want > first ? want : first) * delta_chunk_bytes(3) + 128 * i);
    };
    f32x4 cc[NT];
    // What hangs on no state: (W * Q K^T)^T dH for the state waves, (D dH)^T Q into cc.
    auto ahead = [&](int c) {
      B8 hp[2][NI];
      f32x4 dh[4], z[4];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const Frag8<E> f = col_frag<VT, E>(vt, 32 * s, 16 * w);
        input_parts<E, NI>(__builtin_bit_cast(U8<E>, f), hp[s]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          dh[2 * s][r] = ET<E>::to_f(f.e[r]);
          dh[2 * s + 1][r] = ET<E>::to_f(f.e[4 + r]);
        }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) z[t] = f32x4{0.f, 0.f, 0.f, 0.f};
      mma_triangle<3, false, true>(pf, hp, z);
#pragma unroll
      for (int t = 0; t < 4; ++t) zf[64 * t] = z[t];
#pragma unroll
      for (int i = 0; i < NT; ++i) cc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        B8 dp[3], qf[NT][NI];
        scaled_pair(dh[2 * s], dh[2 * s + 1], sc + (c & 1) * L::SCAL + 32 * s, g, dp);
#pragma unroll
        for (int i = 0; i < NT; ++i) col_parts<QT, NI>(qt, L::qpart, 32 * s, 16 * i, qf[i]);
        mma_many<3, true>(qf, dp, cc);
      }
    };
    if (chunks > first) {
      fetch(chunks - 1);
      weights(chunks - 1);
      place(chunks - 1);
      fetch(chunks - 2);
    }
    __syncthreads();
    if (chunks > first) ahead(chunks - 1);
    __syncthreads();
    for (int c = chunks - 1; c >= first; --c) {
      const int64_t t0 = static_cast<int64_t>(c) * kDTokens;
#pragma unroll
      for (int i = 0; i < NT; ++i) cf[64 * i] = cc[i];
      weights(c - 1);  // (loads are dealt to both halves of a chunk)
      if (c > first) place(c - 1);
      warm_up(c - 3);
      __syncthreads();
      if constexpr (!LOCAL) {
        const __amdgpu_buffer_rsrc_t to = make_rsrc(ba.du + (b * a.T + t0) * row + static_cast<int64_t>(h) * a.P, 0x7ffffff0u);
        f32x4 du[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) du[t] = uf[64 * t];
        rows_out<VEC>(du, to, static_cast<int>(row) * 4, len - t0, p0, a.P);
      }
      if (c > first) ahead(c - 1);
      fetch(c - 2);
      __syncthreads();
    }
  }
}

// LDS of the gradients: two state tiles of 32 value rows and the fragments of m while products over values run, then keys,
// queries and the two matrices between tokens.
template <class E, int NK>
struct GradLds {
  using ST = SelTile<BF16, NK, true>;
  using KT = SelTile<BF16, NK, false>;  // keys and queries: read by rows, by columns and in 8 bytes
  static constexpr int NI = DParts<E>::IN, XS = 68;
  static constexpr int spart = 32 * ST::STRIDE, kpart = kDTokens * KT::STRIDE;
  static constexpr size_t gs = 3 * spart * 2, mf = gs + 3 * spart * 2, stage = mf + 4 * 3 * kDFragElems * 2, end1 = 2 * stage;
  static constexpr size_t k = 0, q = k + NI * kpart * 2, x = q + NI * kpart * 2, y = x + 64 * XS * 4, end2 = y + 64 * XS * 4;
  static constexpr size_t cum = end1 > end2 ? end1 : end2, dc = cum + 64 * 8, b = dc + 12 * 64 * 8, red = b + 64 * 4,
                          bytes = red + 16 * 8;
};

// Sum over the 16 lanes of a row, in every lane of it (rotations by 8, 4, 2, 1), and over the four rows (rows' exchanges): no
// trip through LDS.
template <int CTRL>
__device__ __forceinline__ float rotated(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ double rotated(double x) {
  return dpp_f64<CTRL, 0xf>(x);
}
template <class T>
__device__ __forceinline__ T row_sum(T x) {
  x += rotated<0x128>(x);
  x += rotated<0x124>(x);
  x += rotated<0x122>(x);
  return x + rotated<0x121>(x);
}
__device__ __forceinline__ float quad_sum(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ double quad_sum(double x) {
  auto both = [](auto lo, auto hi) {
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi[0]) << 32 | lo[0]) +
           __builtin_bit_cast(double, static_cast<uint64_t>(hi[1]) << 32 | lo[1]);
  };
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t l = static_cast<uint32_t>(u), h = static_cast<uint32_t>(u >> 32);
  x = both(__builtin_amdgcn_permlane16_swap(l, l, false, false), __builtin_amdgcn_permlane16_swap(h, h, false, false));
  const uint64_t v = __builtin_bit_cast(uint64_t, x);
  const uint32_t m = static_cast<uint32_t>(v), k = static_cast<uint32_t>(v >> 32);
  return both(__builtin_amdgcn_permlane32_swap(m, m, false, false), __builtin_amdgcn_permlane32_swap(k, k, false, false));
}

// x, from here on: addresses made from it are made anew instead of being held (and spilled) since before a loop.
__device__ __forceinline__ int anew(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Values p + 0..3 and p + 16..19 of a row at byte offset `off`, as they lie in memory; zeros where not `ok` or from P on.
template <class E, bool VEC>
__device__ __forceinline__ U8<E> load_slots(__amdgpu_buffer_rsrc_t r, int off, int p, int P, bool ok) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  constexpr int ES = static_cast<int>(sizeof(typename ET<E>::raw));
  if constexpr (VEC) {
    const int a = ok && p < P ? off + p * ES : kBufOOB, b = ok && p + 16 < P ? off + (p + 16) * ES : kBufOOB;
    if constexpr (ES == 2) {
      const u32x2 lo = __builtin_amdgcn_raw_buffer_load_b64(r, a, 0, 0), hi = __builtin_amdgcn_raw_buffer_load_b64(r, b, 0, 0);
      return __builtin_bit_cast(U8<E>, make_uint4(lo[0], lo[1], hi[0], hi[1]));
    } else {
      struct { u32x4 lo, hi; } v = {__builtin_amdgcn_raw_buffer_load_b128(r, a, 0, 0), __builtin_amdgcn_raw_buffer_load_b128(r, b, 0, 0)};
      return __builtin_bit_cast(U8<E>, v);
    }
  } else {
    U8<E> v;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = p + (e < 4 ? e : 12 + e);
      v.e[e] = buf_load1<E>(r, ok && c < P ? off + c * ES : kBufOOB);
    }
    return v;
  }
}

// One workgroup a chunk of a share of a group's heads.  Two waves a tile of 16 tokens, each with half of the keys: gradients
// of keys and queries (transposed: a lane has four keys of one token) are summed over the heads in registers.
// Tiles of the states lie in two stages: while one is worked on the next is split into its parts and the one behind it loaded.
// 461-521 us for 8 x 2048 bf16 tokens x 16 heads of 128 x 128 (656 MB): one workgroup of two waves a SIMD fits the registers (256
// each; a third wave spills), so loads, splits and products, 18% of a SIMD's time, take turns at the barriers.  A wave a token
// tile with all keys took 720; halves that do their products in different order, or keys called for behind the last state
// tile, gave nothing (543 and 471-554).
template <class E, int NK, bool VEC>
__global__ __launch_bounds__(kGradThreads, kGradWaves) void delta_grad_kernel(DeltaBwdArgs ba) {
  using raw = typename ET<E>::raw;
  using L = GradLds<E, NK>;
  using ST = typename L::ST;
  using KT = typename L::KT;
  constexpr int NI = L::NI, NO = DParts<E>::OUT, S = NK / 32, NT = NK / 32, ES = static_cast<int>(sizeof(raw));
  const DeltaArgs& a = ba.f;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  uint16_t* kt = reinterpret_cast<uint16_t*>(lds + L::k);
  uint16_t* qt = reinterpret_cast<uint16_t*>(lds + L::q);
  float* xm = reinterpret_cast<float*>(lds + L::x);
  float* ym = reinterpret_cast<float*>(lds + L::y);
  double* cum_s = reinterpret_cast<double*>(lds + L::cum);
  double* dc_s = reinterpret_cast<double*>(lds + L::dc);  // [12][64]: own and row sums of both halves, column sums of every wave
  float* b_s = reinterpret_cast<float*>(lds + L::b);
  double* red = reinterpret_cast<double*>(lds + L::red);
  const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid >> 6), w = wave & 3, half = wave >> 2;
  const int g = lane >> 4, n = lane & 15, key0 = half * (NK / 2);
  const uint32_t at = xcd_order(blockIdx.x, gridDim.x);
  const int share = static_cast<int>(at % ba.shares), gi = static_cast<int>(at / ba.shares % a.G);
  const int c = static_cast<int>(at / ba.shares / a.G % a.C), b = static_cast<int>(at / ba.shares / a.G / a.C);
  const int64_t len = delta_length(a, b), t0 = static_cast<int64_t>(c) * kDTokens;
  const int rows = static_cast<int>(max_i64(0, min_i64(kDTokens, len - t0)));
  const int all = static_cast<int>(min_i64(kDTokens, a.T - t0));  // rows of the outputs
  const int hpg = a.H / a.G, h0 = gi * hpg + share * ba.per, h1 = min(h0 + ba.per, (gi + 1) * hpg);
  const int64_t row = static_cast<int64_t>(a.H) * a.P;
  const int tok = 16 * w + n;
  const bool in = tok < rows;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};

  f32x4 dk[NT], dq[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) dk[i] = dq[i] = zero;

  for (int h = h0; h < h1 && rows > 0; ++h) {
    const int lane = anew(lane_id()), tid = wave * 64 + lane, g = lane >> 4, n = lane & 15, tok = 16 * w + n;
    const bool in = tok < rows;
    // Scalars, lane = token, in every wave.
    float bt = 0.f, gt = 0.f;
    if (lane < rows) {
      const int64_t i = b * a.sb + (t0 + lane) * a.st + h, j = b * a.db + (t0 + lane) * a.dt + h;
      bt = a.s_f32 ? static_cast<const float*>(a.strengths)[i] : ET<E>::to_f(static_cast<const raw*>(a.strengths)[i]);
      if (a.decays != nullptr)
        gt = a.d_f32 ? static_cast<const float*>(a.decays)[j] : ET<E>::to_f(static_cast<const raw*>(a.decays)[j]);
    }
    // Products over the values, 32 at a time; a tile's loads are under way while the one before is worked on.
    const int64_t cells = static_cast<int64_t>(a.P) * a.N, slab = ((static_cast<int64_t>(b) * a.C + c) * a.H + h) * cells;
    const int64_t first = (b * a.T + t0) * row + static_cast<int64_t>(h) * a.P;
    const __amdgpu_buffer_rsrc_t mr = make_rsrc(a.miss + first, 0x7ffffff0u), ur = make_rsrc(ba.du + first, 0x7ffffff0u),
                                 hr = make_rsrc(static_cast<const raw*>(ba.dhidden) + first, 0x7ffffff0u),
                                 dr = make_rsrc(static_cast<raw*>(ba.dv) + first, 0x7ffffff0u);
    const int off = tok * static_cast<int>(row);
    TileLoad<F32, ST, BF16, VEC, 32, NK, kGradThreads> sl, gl;
    sl.init(a.N, a.N, tid);
    gl.init(a.N, a.N, tid);
    U8<F32> mv, uv;
    U8<E> hv;
    float dots = 0.f, mu = 0.f;
    const int tiles = (a.P + 31) / 32;
    auto fetch = [&](int want) {  // (behind the last tile it is loaded again)
      const int p0 = 32 * (want < tiles ? want : tiles - 1);
      sl.load(a.states + slab + static_cast<int64_t>(p0) * a.N, a.P - p0, tid);
      gl.load(ba.gstates + slab + static_cast<int64_t>(p0) * a.N, a.P - p0, tid);
      mv = load_slots<F32, VEC>(mr, off * 4, p0 + 4 * g, a.P, in);
      uv = load_slots<F32, VEC>(ur, off * 4, p0 + 4 * g, a.P, in);
      hv = load_slots<E, VEC>(hr, off * ES, p0 + 4 * g, a.P, in);
    };
    auto place = [&](int tile) {
      char* to = lds + (tile & 1) * L::stage;
      store_parts<ST, 3, F32>(sl, reinterpret_cast<uint16_t*>(to), L::spart, 32, tid);
      store_parts<ST, 3, F32>(gl, reinterpret_cast<uint16_t*>(to + L::gs), L::spart, 32, tid);
      if (half == 0) {  // this wave's rows of m for the others
        B8 mo[3];
        split8<3>(mv.e, mo);
        uint16_t* mf = reinterpret_cast<uint16_t*>(to + L::mf) + w * 3 * kDFragElems + 8 * lane;
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<uint4*>(mf + p * kDFragElems) = __builtin_bit_cast(uint4, mo[p]);
      }
      if (tile < tiles && (sl.UNITS >= kGradThreads || tid < sl.UNITS)) {
#pragma unroll
        for (int i = 0; i < sl.PER; ++i) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            dots = fmaf(__uint_as_float(sl.r[i][e >> 2][e & 3]), __uint_as_float(gl.r[i][e >> 2][e & 3]), dots);
        }
      }
    };
    fetch(0);
    double l = static_cast<double>(gt) * 1.4426950408889634;
    l = l < -200.0 ? -200.0 : l;
    const double cum = wave_prefix(l), total = lane_value(cum, 63);
    const double mycum = __shfl(cum, tok);
    const float myb = __shfl(bt, tok), myd = exp2_d(mycum), mye = exp2_d(total - mycum);
    const float eb = mye * myb, db = -myd * myb;
    __syncthreads();  // (the last head's readers are done)
    if (wave == 0) {
      cum_s[lane] = cum;
      b_s[lane] = bt;
    }

    f32x4 yq[NT], yk[NT], yg[NT], wz[4];
#pragma unroll
    for (int i = 0; i < NT; ++i) yq[i] = yk[i] = yg[i] = zero;
#pragma unroll
    for (int i = 0; i < 4; ++i) wz[i] = zero;
    place(0);
    for (int tile = 0; tile < tiles; ++tile) {
      const int p0 = 32 * tile;
      B8 up[3], hp[NI];
      split8<3>(uv.e, up);
      input_parts<E, NI>(hv, hp);
      if (half == 1) {  // dV, and the strengths' sums
        float dv[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          dv[e] = myb * uv.e[e];
          // (A float32 product, so that every form rounds it alike: one value's conversion to float16 would take the product in.)
          if constexpr (!VEC) asm volatile("" : "+v"(dv[e]));
          mu = fmaf(uv.e[e], mv.e[e], mu);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int p = p0 + 4 * g + 16 * u;
          if (VEC) {
            buf_store4<E>(dr, in && p < a.P ? (off + p) * ES : kBufOOB, f32x4{dv[4 * u], dv[4 * u + 1], dv[4 * u + 2], dv[4 * u + 3]});
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) buf_store1<E>(dr, in && p + r < a.P ? (off + p + r) * ES : kBufOOB, dv[4 * u + r]);
          }
        }
      }
      fetch(tile + 1);
      __syncthreads();
      const char* from = lds + (tile & 1) * L::stage;
      const uint16_t* stile = reinterpret_cast<const uint16_t*>(from);
      const uint16_t* gtile = reinterpret_cast<const uint16_t*>(from + L::gs);
      const uint16_t* mfrag = reinterpret_cast<const uint16_t*>(from + L::mf);
      {
        B8 mp[3];
#pragma unroll
        for (int p = 0; p < 3; ++p)
          mp[p] = __builtin_bit_cast(B8, *reinterpret_cast<const uint4*>(mfrag + (w * 3 + p) * kDFragElems + 8 * lane));
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          B8 sf[3], gf[3];
          col_parts<ST, 3>(stile, L::spart, 0, key0 + 16 * i, sf);
          col_parts<ST, 3>(gtile, L::spart, 0, key0 + 16 * i, gf);
#pragma unroll
          for (int o = 2; o >= 0; --o) {  // (three sums in turn: a product waits for none of the two before it)
#pragma unroll
            for (int k = 0; k <= o; ++k) {
              yk[i] = mfma8(sf[k], up[o - k], yk[i]);
              yg[i] = mfma8(gf[k], mp[o - k], yg[i]);
              if (o - k < NI) yq[i] = mfma8(sf[k], hp[o - k], yq[i]);
            }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j <= w) {
          B8 f[3];
#pragma unroll
          for (int p = 0; p < 3; ++p)
            f[p] = __builtin_bit_cast(B8, *reinterpret_cast<const uint4*>(mfrag + (j * 3 + p) * kDFragElems + 8 * lane));
          // Rows i = 16 w + 4 g + r, column j = 16 j + n: half 0 du m^T, half 1 dH m^T.
          if (half == 0) wz[j] = mma_parts<3>(up, f, wz[j]);
          else wz[j] = mma_parts<3>(hp, f, wz[j]);
        }
      }
      place(tile + 1);
    }
    __syncthreads();  // (the tiles make room)
    {
      TileLoad<E, KT, BF16, VEC, kDTokens, NK, kGradThreads> kl, ql;
      kl.init(a.kt, a.N, tid);
      ql.init(a.qt, a.N, tid);
      kl.load(static_cast<const raw*>(a.keys) + b * a.kb + t0 * a.kt + static_cast<int64_t>(gi) * a.N, rows, tid);
      ql.load(static_cast<const raw*>(a.queries) + b * a.qb + t0 * a.qt + static_cast<int64_t>(gi) * a.N, rows, tid);
      store_parts<KT, NI, E>(kl, kt, L::kpart, kDTokens, tid);
      store_parts<KT, NI, E>(ql, qt, L::kpart, kDTokens, tid);
    }
    __syncthreads();
    // q.(dH S), k.(du S), k.(m G): a lane's four keys of every tile.
    float al = 0.f, be = 0.f, ep = 0.f;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      f32x4 kv = zero, qv = zero;
#pragma unroll
      for (int p = NI - 1; p >= 0; --p) {
        const uint2 ku = *reinterpret_cast<const uint2*>(kt + p * L::kpart + KT::at(tok, key0 + 16 * i + 4 * g));
        const uint2 qu = *reinterpret_cast<const uint2*>(qt + p * L::kpart + KT::at(tok, key0 + 16 * i + 4 * g));
        kv += f32x4{__uint_as_float(ku.x << 16), __uint_as_float(ku.x & 0xffff0000u), __uint_as_float(ku.y << 16),
                    __uint_as_float(ku.y & 0xffff0000u)};
        qv += f32x4{__uint_as_float(qu.x << 16), __uint_as_float(qu.x & 0xffff0000u), __uint_as_float(qu.y << 16),
                    __uint_as_float(qu.y & 0xffff0000u)};
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        al = fmaf(qv[r], yq[i][r], al);
        be = fmaf(kv[r], yk[i][r], be);
        ep = fmaf(kv[r], yg[i][r], ep);
      }
      dq[i] += yq[i] * myd;
      dk[i] += yg[i] * eb + yk[i] * db;
    }
    // <G, S>, and the sum of k.(E b m G), over the workgroup.
    const double eps = static_cast<double>(ep) * static_cast<double>(eb);
    {
      double e = eps + static_cast<double>(dots) * static_cast<double>(exp2_d(total));
      e = quad_sum(row_sum(e));
      if (lane == 0) red[wave] = e;
    }
    const double own = quad_sum(static_cast<double>(al) * static_cast<double>(myd) + static_cast<double>(be) * static_cast<double>(db) - eps);
    mu = quad_sum(mu);
    if (g == 0) {
      dc_s[half * 64 + tok] = own;
      if (half == 1 && tok < all) {
        const int64_t i = (b * a.T + t0 + tok) * a.H + h;
        const float v = in ? mu : 0.f;
        if (a.s_f32) static_cast<float*>(ba.ds)[i] = v;
        else static_cast<raw*>(ba.ds)[i] = ET<E>::from_f(v);
      }
    }

    // The matrices between tokens, half 0 X and half 1 Y, and their shares of T's row and column sums.
    f32x4 dot[4];
    const int lane2 = anew(lane), g2 = lane2 >> 4, n2 = lane2 & 15;
    {
      const uint16_t* left = half == 0 ? kt : qt;
#pragma unroll
      for (int j = 0; j < 4; ++j) dot[j] = zero;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        B8 li[NI], kj[4][NI];
        row_parts_t<KT, NI>(left, L::kpart, 16 * w, 32 * s, li);
#pragma unroll
        for (int j = 0; j < 4; ++j) row_parts_t<KT, NI>(kt, L::kpart, 16 * j, 32 * s, kj[j]);
        mma_many<3, false>(kj, li, dot);  // (tiles above the diagonal are not used)
      }
    }
    double rsum[4] = {0.0, 0.0, 0.0, 0.0}, ci[4];
    float bi[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      ci[r] = cum_s[16 * w + 4 * g2 + r];
      bi[r] = half == 0 ? -b_s[16 * w + 4 * g2 + r] : 1.f;
    }
    float* mat = half == 0 ? xm : ym;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      double csum = 0.0;
      if (j <= w) {
        const int tj = 16 * j + n2;
        const double cj = cum_s[tj];
        const float bj = b_s[tj];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int ti = 16 * w + 4 * g2 + r;
          const bool below = tj < ti, seen = half == 0 ? below : tj <= ti;
          const float x = (seen ? exp2_f(static_cast<float>(ci[r] - cj)) * (bi[r] * bj) : 0.f) * wz[j][r];
          // (What lies above the diagonal goes to the row's padding.)
          mat[ti * L::XS + (tj <= ti ? tj : 64)] = x;
          if (half == 0) mat[tj <= ti ? tj * L::XS + ti : ti * L::XS + 64] = x;
          // (A token's weight of itself does not decay.  Row and column sums take the same rounded product, so that what
          // cancels between them does so whole.)
          const double tau = below ? static_cast<double>(x * dot[j][r]) : 0.0;
          rsum[r] += tau;
          csum += tau;
        }
      }
      csum = quad_sum(csum);
      if (g2 == 0) dc_s[(4 + wave) * 64 + 16 * j + n2] = csum;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      rsum[r] = row_sum(rsum[r]);
      if (n2 == 0) dc_s[(2 + half) * 64 + 16 * w + 4 * g2 + r] = rsum[r];
    }
    __syncthreads();
    if (wave == 0 && ba.dd != nullptr) {
      double d = 0.0;
#pragma unroll
      for (int i = 0; i < 12; ++i) d += i < 4 ? dc_s[64 * i + lane] : -dc_s[64 * i + lane];
      const double pre = wave_prefix(d), whole = lane_value(pre, 63);
      double dg = whole - pre + d;
#pragma unroll
      for (int i = 0; i < kGradThreads / 64; ++i) dg += red[i];
      if (lane < all) {
        const int64_t i = (b * a.T + t0 + lane) * a.H + h;
        const float v = lane < rows ? static_cast<float>(dg) : 0.f;
        if (a.d_f32) static_cast<float*>(ba.dd)[i] = v;
        else static_cast<raw*>(ba.dd)[i] = ET<E>::from_f(v);
      }
    }
    // dQ^T += K^T Y^T, dK^T += K^T (X + X^T) + Q^T Y.
    const int lane3 = anew(lane), g3 = lane3 >> 4, tok3 = 16 * w + (lane3 & 15);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      float yr[8], xr[8], yc[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int k = 32 * s + (e < 4 ? 4 * g3 + e : 12 + 4 * g3 + e);
        // (Y is not written above the diagonal.)
        const float up = ym[tok3 * L::XS + k], down = ym[k * L::XS + tok3];
        yr[e] = k <= tok3 ? up : 0.f;
        yc[e] = k >= tok3 ? down : 0.f;
        xr[e] = xm[tok3 * L::XS + k];
      }
      B8 yp[NO], xp[NO], cp[NO];
      split8<NO>(yr, yp);
      split8<NO>(xr, xp);
      split8<NO>(yc, cp);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        B8 kf[NI], qf[NI];
        col_parts<KT, NI>(kt, L::kpart, 32 * s, key0 + 16 * i, kf);
        col_parts<KT, NI>(qt, L::kpart, 32 * s, key0 + 16 * i, qf);
        dq[i] = mma_parts<NO>(kf, yp, dq[i]);
        dk[i] = mma_parts<NO>(kf, xp, dk[i]);
        dk[i] = mma_parts<NO>(qf, cp, dk[i]);
      }
    }
  }
  // Rows behind the length.
  if (rows < all) {
    for (int h = h0; h < h1; ++h) {
      for (int i = tid; i < (all - rows) * a.P; i += kGradThreads) {
        const int r = rows + i / a.P;
        static_cast<raw*>(ba.dv)[(b * a.T + t0 + r) * row + static_cast<int64_t>(h) * a.P + i % a.P] = 0;
      }
      if (rows == 0 && tid < all) {
        const int64_t i = (b * a.T + t0 + tid) * a.H + h;
        if (a.s_f32) static_cast<float*>(ba.ds)[i] = 0.f;
        else static_cast<raw*>(ba.ds)[i] = 0;
        if (ba.dd != nullptr) {
          if (a.d_f32) static_cast<float*>(ba.dd)[i] = 0.f;
          else static_cast<raw*>(ba.dd)[i] = 0;
        }
      }
    }
  }
  if (tok < all) {
    if (!in) {  // (a state that is no number makes NaN of the zeros that stand for these rows)
#pragma unroll
      for (int i = 0; i < NT; ++i) dk[i] = dq[i] = zero;
    }
    const int64_t to = ((b * a.T + t0 + tok) * a.G + gi) * a.N;
    const int64_t plane = static_cast<int64_t>(a.B) * a.T * a.G * a.N;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int k = key0 + 16 * i + 4 * g;
      if (k >= a.N) continue;
      if (ba.part != nullptr) {
        float* pk = ba.part + share * plane + to + k;
        float* pq = pk + ba.shares * plane;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (k + r < a.N) {
            pk[r] = dk[i][r];
            pq[r] = dq[i][r];
          }
        }
      } else {
        raw* pk = static_cast<raw*>(ba.dk) + to + k;
        raw* pq = static_cast<raw*>(ba.dq) + to + k;
        if (ba.whole) {
          store4_raw<E>(pk, dk[i]);
          store4_raw<E>(pq, dq[i]);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (k + r < a.N) {
              pk[r] = ET<E>::from_f(dk[i][r]);
              pq[r] = ET<E>::from_f(dq[i][r]);
            }
          }
        }
      }
    }
  }
}

// The shares' gradients of keys and queries, added up.
template <class E>
__global__ __launch_bounds__(kThreads) void delta_share_sum_kernel(const float* part, void* dk, void* dq, int64_t plane, int shares) {
  for (int64_t i = blockIdx.x * int64_t{kThreads} + threadIdx.x; i < 2 * plane; i += int64_t{gridDim.x} * kThreads) {
    const int64_t which = i >= plane ? 1 : 0, at = i - which * plane;
    const float* p = part + which * shares * plane + at;
    float s = 0.f;
    for (int j = 0; j < shares; ++j) s += p[j * plane];
    (which ? static_cast<typename ET<E>::raw*>(dq) : static_cast<typename ET<E>::raw*>(dk))[at] = ET<E>::from_f(s);
  }
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }

// Enough workgroups for two on each of 256 CUs, where the heads of the groups allow it.
int share_count(int64_t B, int64_t C, int64_t H, int64_t G) {
  const int64_t hpg = H / G, wgs = B * C * G;
  int64_t shares = wgs > 0 ? (512 + wgs - 1) / wgs : 1;
  if (shares > hpg) shares = hpg;
  const int64_t per = (hpg + shares - 1) / shares;
  return static_cast<int>((hpg + per - 1) / per);
}

struct Work {
  int64_t chunks, states, du, part, part_state, part_map, part_chunks, bytes;
  int parts;
};
Work work_of(int64_t B, int64_t T, int64_t H, int64_t P, int64_t G, int64_t N) {
  const int64_t C = (T + kDTokens - 1) / kDTokens, shares = share_count(B, C, H, G);
  Work w{};
  w.chunks = 0;
  w.states = up16(B * H * C * delta_chunk_bytes(3));
  w.du = w.states + up16(B * C * H * P * N * 4);
  w.part = w.du + up16(B * T * H * P * 4);
  w.part_state = w.part + up16(shares > 1 ? 2 * shares * B * T * G * N * 4 : 0);
  // (Of any type: what takes no parts needs less.)
  w.parts = delta_time_parts(B * H, P, N, C, GRM_HIP_BF16, true, &w.part_chunks);
  w.part_map = w.part_state + up16((w.parts - 1) * B * H * P * N * 4);
  w.bytes = w.part_map + (w.parts - 1) * B * H * N * N * 4;
  return w;
}

}  // namespace
}  // namespace grmhip

using namespace grmhip;

extern "C" int64_t grm_hip_delta_scan_bwd_workspace(int64_t batch, int64_t seq_len, int64_t heads, int64_t value_dim,
                                                    int64_t groups, int64_t key_dim) {
  if (batch <= 0 || seq_len <= 0 || heads <= 0 || value_dim <= 0 || groups <= 0 || key_dim <= 0 || heads % groups != 0) return 0;
  return work_of(batch, seq_len, heads, value_dim, groups, key_dim).bytes;
}

extern "C" int grm_hip_delta_scan_bwd(const grm_hip_delta_args* u, const float* states, const float* miss,
                                      const void* grad_hidden, const float* grad_memory_out, void* grad_keys,
                                      void* grad_values, void* grad_queries, void* grad_strengths, void* grad_log_decays,
                                      float* grad_memory, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "delta_scan backward";
  if (int rc = delta_check(u, what, false)) return rc;
  if (u->batch == 0) return GRM_HIP_OK;
  if (grad_memory == nullptr || !aligned(grad_memory) || !aligned(grad_memory_out) ||
      (u->seq_len > 0 && (states == nullptr || miss == nullptr || grad_hidden == nullptr || grad_keys == nullptr ||
                          grad_values == nullptr || grad_queries == nullptr || grad_strengths == nullptr || !aligned(states) ||
                          workspace == nullptr || !aligned(workspace)))) {
    set_error("%s: states, miss, grad_hidden, the gradients and a workspace are required, states 16-byte aligned", what);
    return GRM_HIP_EINVAL;
  }
  const Work wk = work_of(u->batch, u->seq_len, u->heads, u->value_dim, u->groups, u->key_dim);
  if (u->seq_len > 0 && workspace_bytes < wk.bytes) {
    set_error("%s: workspace too small", what);
    return GRM_HIP_EINVAL;
  }
  const hipStream_t hs = static_cast<hipStream_t>(stream);
  DeltaBwdArgs a{};
  a.f = delta_args(u);
  a.f.states = const_cast<float*>(states);
  a.f.miss = const_cast<float*>(miss);
  a.f.work = static_cast<char*>(workspace);
  a.f.memory = nullptr;
  a.dhidden = grad_hidden; a.dmemory = grad_memory_out;
  a.dk = grad_keys; a.dv = grad_values; a.dq = grad_queries; a.ds = grad_strengths; a.dd = grad_log_decays; a.dm = grad_memory;
  a.whole = (u->key_dim & 3) == 0 && aligned(grad_keys) && aligned(grad_queries);
  int64_t part_chunks = 0;
  if (u->seq_len > 0) {
    a.gstates = reinterpret_cast<float*>(a.f.work + wk.states);
    a.du = reinterpret_cast<float*>(a.f.work + wk.du);
    a.shares = share_count(u->batch, a.f.C, u->heads, u->groups);
    a.per = static_cast<int>((u->heads / u->groups + a.shares - 1) / a.shares);
    a.part = a.shares > 1 ? reinterpret_cast<float*>(a.f.work + wk.part) : nullptr;
    a.f.parts = delta_time_parts(u->batch * u->heads, u->value_dim, u->key_dim, a.f.C, u->dtype, true, &part_chunks);
    a.f.part_chunks = static_cast<int>(part_chunks);
    a.f.mirror = 1;
    a.f.part_state = reinterpret_cast<float*>(a.f.work + wk.part_state);
    a.f.part_map = reinterpret_cast<float*>(a.f.work + wk.part_map);
    if (int rc = launch_delta_prep(a.f, u->dtype, true, hs, what)) return rc;
  }
  auto set_lds = [&](const void* kernel, size_t bytes) {
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e == hipSuccess) return GRM_HIP_OK;
    set_error("%s: %s", what, hipGetErrorString(e));
    return static_cast<int>(e);
  };
  int rc = GRM_HIP_OK;
  delta_with_form(u->dtype, a.f.N, a.f.vec != 0 && aligned(grad_hidden) && aligned(grad_values), [&](auto e, auto nk, auto vec) {
    using E = decltype(e);
    constexpr int NK = decltype(nk)::value;
    constexpr bool VEC = decltype(vec)::value;
    {
      auto go = [&](auto kernel, int64_t tiles, int threads, size_t lds) {
        if (rc != GRM_HIP_OK || (rc = set_lds(reinterpret_cast<const void*>(kernel), lds)) != GRM_HIP_OK) return;
        kernel<<<dim3(static_cast<uint32_t>(a.f.B) * a.f.H * static_cast<uint32_t>(tiles)), dim3(threads), lds, hs>>>(a);
        rc = check_launch(what);
      };
      if constexpr (MirrorLds<E, NK>::fits) {
        constexpr size_t lds = MirrorLds<E, NK>::bytes;
        if (a.f.parts > 1) {
          go(delta_mirror_kernel<E, NK, VEC, true>, (a.f.PT + a.f.NT) * (a.f.parts - 1), 2 * kThreads, lds);
          if (rc == GRM_HIP_OK) rc = launch_delta_join(a.f, hs, what);
        }
        go(delta_mirror_kernel<E, NK, VEC, false>, a.f.PT * a.f.parts, 2 * kThreads, lds);
      } else {
        go(delta_reverse_kernel<E, NK, VEC>, a.f.PT, kThreads, ReverseLds<E, NK>::bytes);
      }
      if (rc != GRM_HIP_OK || a.f.C == 0) return;
    }
    auto kernel = delta_grad_kernel<E, NK, VEC>;
    constexpr size_t lds = GradLds<E, NK>::bytes;
    if ((rc = set_lds(reinterpret_cast<const void*>(kernel), lds)) != GRM_HIP_OK) return;
    kernel<<<dim3(static_cast<uint32_t>(a.f.B) * a.f.C * a.f.G * a.shares), dim3(kGradThreads), lds, hs>>>(a);
    if ((rc = check_launch(what)) != GRM_HIP_OK || a.part == nullptr) return;
    const int64_t plane = static_cast<int64_t>(a.f.B) * a.f.T * a.f.G * a.f.N, blocks = (2 * plane + kThreads - 1) / kThreads;
    delta_share_sum_kernel<E><<<dim3(static_cast<uint32_t>(blocks < 4096 ? blocks : 4096)), dim3(kThreads), 0, hs>>>(
        a.part, a.dk, a.dq, plane, a.shares);
    rc = check_launch(what);
  });
  return rc;
}
