// Gradients of the gated delta rule.  With the states S before every chunk and m from the forward (delta.h), and G the gradient
// of the state behind a chunk:
//   z  = (W * Q K^T)^T dH + E K G^T,  du = (I + b A)^-T z       (du: of what a token writes, u = b m)
//   G0 = e^{c_63} G + (D dH)^T Q - (D b du)^T K,  dV = b du,  db = sum_p du m
//   Y  = W b_j (dH m^T)  (j <= i),  X = -W b_i b_j (du m^T)  (j < i)
//   dQ = D dH S + Y K,  dK = -D b du S + E b m G + Y^T Q + (X + X^T) K
// and for the log decays, dc_i = row sums less column sums of T = X * K K^T + Y * Q K^T, + q.(D dH S) - k.(D b du S) - e_i
// with e = k.(E b m G); dg_t = sum_{i >= t} dc_i + sum e + e^{c_63} <G, S>.
// The walk over the chunks from the last to the first leaves du and G (delta_reverse_kernel); all else is done for all chunks
// side by side (delta_grad_kernel).  No atomics: sums are taken in a fixed order.
#include "delta.h"

namespace grmhip {
namespace {

constexpr int kThreads = 256;

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

// The walk's mirror: 16 value columns of the gradient's state a wave, chunks from the last to the first.
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

// LDS of the gradients: two state tiles of 32 value rows and the fragments of m while products over values run, then keys,
// queries and the two matrices between tokens.
template <class E, int NK>
struct GradLds {
  using ST = SelTile<BF16, NK, true>;
  static constexpr int NI = DParts<E>::IN, XS = 68;
  static constexpr int spart = 32 * ST::STRIDE, kpart = kDTokens * ST::STRIDE;
  static constexpr size_t s = 0, gs = s + 3 * spart * 2, mf = gs + 3 * spart * 2, end1 = mf + 4 * 3 * kDFragElems * 2;
  static constexpr size_t k = 0, q = k + NI * kpart * 2, x = q + NI * kpart * 2, y = x + 64 * XS * 4, end2 = y + 64 * XS * 4;
  static constexpr size_t cum = end1 > end2 ? end1 : end2, dc = cum + 64 * 8, b = dc + 64 * 8, red = b + 64 * 4,
                          bytes = red + 16 * 8;
};

// Sum over the 16 lanes of a row, in every lane of it; and over the four rows.
__device__ __forceinline__ double row_sum(double x) {
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) x += __shfl_xor(x, o);
  return x;
}
template <class T>
__device__ __forceinline__ T quad_sum(T x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// One workgroup a chunk of a share of a group's heads; wave w holds token tile w, its gradients of keys and queries (transposed: a
// lane has four keys of one token) summed over the heads in registers.
template <class E, int NK, bool VEC>
__global__ __launch_bounds__(kThreads) void delta_grad_kernel(DeltaBwdArgs ba) {
  using raw = typename ET<E>::raw;
  using L = GradLds<E, NK>;
  using ST = typename L::ST;
  constexpr int NI = L::NI, NO = DParts<E>::OUT, S = NK / 32, NT = NK / 16;
  const DeltaArgs& a = ba.f;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  uint16_t* stile = reinterpret_cast<uint16_t*>(lds + L::s);
  uint16_t* gtile = reinterpret_cast<uint16_t*>(lds + L::gs);
  uint16_t* mfrag = reinterpret_cast<uint16_t*>(lds + L::mf);
  uint16_t* kt = reinterpret_cast<uint16_t*>(lds + L::k);
  uint16_t* qt = reinterpret_cast<uint16_t*>(lds + L::q);
  float* xm = reinterpret_cast<float*>(lds + L::x);
  float* ym = reinterpret_cast<float*>(lds + L::y);
  double* cum_s = reinterpret_cast<double*>(lds + L::cum);
  double* dc_s = reinterpret_cast<double*>(lds + L::dc);
  float* b_s = reinterpret_cast<float*>(lds + L::b);
  double* red = reinterpret_cast<double*>(lds + L::red);
  const int tid = threadIdx.x, lane = lane_id(), w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, n = lane & 15;
  const uint32_t at = xcd_order(blockIdx.x, gridDim.x);
  const int share = static_cast<int>(at % ba.shares), gi = static_cast<int>(at / ba.shares % a.G);
  const int c = static_cast<int>(at / ba.shares / a.G % a.C), b = static_cast<int>(at / ba.shares / a.G / a.C);
  const int64_t len = delta_length(a, b), t0 = static_cast<int64_t>(c) * kDTokens;
  const int rows = static_cast<int>(max_i64(0, min_i64(kDTokens, len - t0)));
  const int all = static_cast<int>(min_i64(kDTokens, a.T - t0));  // rows of the outputs
  const int hpg = a.H / a.G, h0 = gi * hpg + share * ba.per, h1 = min(h0 + ba.per, (gi + 1) * hpg);
  const int64_t row = static_cast<int64_t>(a.H) * a.P;
  const int tok = 16 * w + n;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};

  f32x4 dk[NT], dq[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) dk[i] = dq[i] = zero;

  for (int h = h0; h < h1 && rows > 0; ++h) {
    // Scalars, lane = token, in every wave.
    float bt = 0.f, gt = 0.f;
    if (lane < rows) {
      const int64_t i = b * a.sb + (t0 + lane) * a.st + h, j = b * a.db + (t0 + lane) * a.dt + h;
      bt = a.s_f32 ? static_cast<const float*>(a.strengths)[i] : ET<E>::to_f(static_cast<const raw*>(a.strengths)[i]);
      if (a.decays != nullptr)
        gt = a.d_f32 ? static_cast<const float*>(a.decays)[j] : ET<E>::to_f(static_cast<const raw*>(a.decays)[j]);
    }
    double l = static_cast<double>(gt) * 1.4426950408889634;
    l = l < -200.0 ? -200.0 : l;
    const double cum = wave_prefix(l), total = lane_value(cum, 63);
    __syncthreads();  // (the last head's readers are done)
    if (w == 0) {
      cum_s[lane] = cum;
      b_s[lane] = bt;
      dc_s[lane] = 0.0;
    }
    const double mycum = __shfl(cum, tok);
    const float myb = __shfl(bt, tok), myd = exp2_d(mycum), mye = exp2_d(total - mycum);

    // Products over the values, 32 at a time.
    f32x4 yq[NT], yk[NT], yg[NT], wt[4], zt[4];
#pragma unroll
    for (int i = 0; i < NT; ++i) yq[i] = yk[i] = yg[i] = zero;
#pragma unroll
    for (int i = 0; i < 4; ++i) wt[i] = zt[i] = zero;
    const int64_t cells = static_cast<int64_t>(a.P) * a.N, slab = ((static_cast<int64_t>(b) * a.C + c) * a.H + h) * cells;
    const int64_t my = (b * a.T + t0 + tok) * row + static_cast<int64_t>(h) * a.P;
    const bool in = tok < rows;
    TileLoad<F32, ST, BF16, VEC, 32, NK, kThreads> sl, gl;
    sl.init(a.N, a.N, tid);
    gl.init(a.N, a.N, tid);
    float dots = 0.f, dbs = 0.f;
    for (int p0 = 0; p0 < a.P; p0 += 32) {
      sl.load(a.states + slab + static_cast<int64_t>(p0) * a.N, a.P - p0, tid);
      gl.load(ba.gstates + slab + static_cast<int64_t>(p0) * a.N, a.P - p0, tid);
      // This wave's rows: slots 0-3 are values 4 g + e, 4-7 are 16 + 4 g + e.
      float mv[8], uv[8];
      U8<E> hv;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int p = p0 + (e < 4 ? 4 * g + e : 12 + 4 * g + e);
        const bool ok = in && p < a.P;
        mv[e] = ok ? a.miss[my + p] : 0.f;
        uv[e] = ok ? ba.du[my + p] : 0.f;
        hv.e[e] = ok ? static_cast<const raw*>(ba.dhidden)[my + p] : raw(0);
      }
      B8 mp[3], up[3], hp[NI];
      split8<3>(mv, mp);
      split8<3>(uv, up);
      input_parts<E, NI>(hv, hp);
      __syncthreads();
      store_parts<ST, 3, F32>(sl, stile, L::spart, 32, tid);
      store_parts<ST, 3, F32>(gl, gtile, L::spart, 32, tid);
#pragma unroll
      for (int i = 0; i < sl.PER; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          dots = fmaf(__uint_as_float(sl.r[i][e >> 2][e & 3]), __uint_as_float(gl.r[i][e >> 2][e & 3]), dots);
      }
#pragma unroll
      for (int p = 0; p < 3; ++p)
        *reinterpret_cast<uint4*>(mfrag + (w * 3 + p) * kDFragElems + 8 * lane) = __builtin_bit_cast(uint4, mp[p]);
      // dV and the strengths' sums.
      raw* dv = static_cast<raw*>(ba.dv) + my + p0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int p = e < 4 ? 4 * g + e : 12 + 4 * g + e;
        dbs = fmaf(uv[e], mv[e], dbs);
        if (in && p0 + p < a.P) dv[p] = ET<E>::from_f(myb * uv[e]);
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        B8 sf[3], gf[3];
        col_parts<ST, 3>(stile, L::spart, 0, 16 * i, sf);
        col_parts<ST, 3>(gtile, L::spart, 0, 16 * i, gf);
        yq[i] = mma_parts<3>(sf, hp, yq[i]);
        yk[i] = mma_parts<3>(sf, up, yk[i]);
        yg[i] = mma_parts<3>(gf, mp, yg[i]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j <= w) {
          B8 f[3];
#pragma unroll
          for (int p = 0; p < 3; ++p)
            f[p] = __builtin_bit_cast(B8, *reinterpret_cast<const uint4*>(mfrag + (j * 3 + p) * kDFragElems + 8 * lane));
          wt[j] = mma_parts<3>(up, f, wt[j]);  // rows i = 16 w + 4 g + r, column j = 16 j + n
          zt[j] = mma_parts<3>(hp, f, zt[j]);
        }
      }
    }
    // <G, S> over the workgroup.
    double dot = static_cast<double>(dots);
    dot = quad_sum(row_sum(dot));
    if (lane == 0) red[w] = dot;
    __syncthreads();  // (the tiles make room)
    {
      TileLoad<E, ST, BF16, VEC, kDTokens, NK, kThreads> kl;
      kl.init(a.kt, a.N, tid);
      kl.load(static_cast<const raw*>(a.keys) + b * a.kb + t0 * a.kt + static_cast<int64_t>(gi) * a.N, rows, tid);
      store_parts<ST, NI, E>(kl, kt, L::kpart, kDTokens, tid);
      kl.init(a.qt, a.N, tid);
      kl.load(static_cast<const raw*>(a.queries) + b * a.qb + t0 * a.qt + static_cast<int64_t>(gi) * a.N, rows, tid);
      store_parts<ST, NI, E>(kl, qt, L::kpart, kDTokens, tid);
    }
    __syncthreads();
    // q.(D dH S), k.(D b du S), k.(E b m G): a lane's four keys of every tile, then over the four rows of lanes.
    float al = 0.f, be = 0.f, ep = 0.f;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      f32x4 kv = zero, qv = zero;
#pragma unroll
      for (int p = NI - 1; p >= 0; --p) {
        const uint2 ku = *reinterpret_cast<const uint2*>(kt + p * L::kpart + ST::at(tok, 16 * i + 4 * g));
        const uint2 qu = *reinterpret_cast<const uint2*>(qt + p * L::kpart + ST::at(tok, 16 * i + 4 * g));
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
      dk[i] += yg[i] * (mye * myb) - yk[i] * (myd * myb);
    }
    const double eps = quad_sum(static_cast<double>(ep) * static_cast<double>(mye * myb));
    const double own = quad_sum(static_cast<double>(al) * static_cast<double>(myd) -
                                static_cast<double>(be) * static_cast<double>(myd * myb)) - eps;
    dbs = quad_sum(dbs);
    const double esum = row_sum(eps);  // of this wave's 16 tokens
    if (lane == 0) red[4 + w] = esum;

    // The matrices between tokens, and what they give the decays.
    double rsum[4] = {0.0, 0.0, 0.0, 0.0}, csum[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j <= w) {
        f32x4 kk = zero, qk = zero;
#pragma unroll
        for (int s = 0; s < S; ++s) {
          B8 ki[NI], qi[NI], kj[NI];
          row_parts_t<ST, NI>(kt, L::kpart, 16 * w, 32 * s, ki);
          row_parts_t<ST, NI>(qt, L::kpart, 16 * w, 32 * s, qi);
          row_parts_t<ST, NI>(kt, L::kpart, 16 * j, 32 * s, kj);
          kk = mma_parts<3>(ki, kj, kk);
          qk = mma_parts<3>(qi, kj, qk);
        }
        const int tj = 16 * j + n;
        const double cj = cum_s[tj];
        const float bj = b_s[tj];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int ti = 16 * w + 4 * g + r;
          const float decay = tj <= ti ? exp2_d(cum_s[ti] - cj) : 0.f;
          const float y = decay * bj * zt[j][r];
          const float x = tj < ti ? -decay * b_s[ti] * bj * wt[j][r] : 0.f;
          ym[ti * L::XS + tj] = y;
          if (tj <= ti) xm[ti * L::XS + tj] = xm[tj * L::XS + ti] = x;
          if (tj < ti) {  // (a token's weight of itself does not decay)
            const double tau = static_cast<double>(x) * static_cast<double>(kk[r]) + static_cast<double>(y) * static_cast<double>(qk[r]);
            rsum[r] += tau;
            csum[j] += tau;
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) rsum[r] = row_sum(rsum[r]);
    // One wave at a time adds its column sums: a fixed order.
    for (int v = 0; v < 4; ++v) {
      if (v == w) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const double cs = quad_sum(csum[j]);
          if (j <= w && g == 0) dc_s[16 * j + n] -= cs;
        }
      }
      __syncthreads();
    }
    // (A wave's own rows from here on.)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n == 0) dc_s[16 * w + 4 * g + r] += rsum[r];
    __syncthreads();
    if (g == 0) dc_s[tok] += own;
    __syncthreads();
    if (w == 0) {
      // dg_t = sum_{i >= t} dc_i + sum e + e^{c_63} <G, S>.
      const double d = dc_s[lane], pre = wave_prefix(d), whole = lane_value(pre, 63);
      const double dg = whole - pre + d + (red[4] + red[5] + red[6] + red[7]) +
                        static_cast<double>(exp2_d(total)) * (red[0] + red[1] + red[2] + red[3]);
      if (ba.dd != nullptr && lane < all) {
        const int64_t i = (b * a.T + t0 + lane) * a.H + h;
        const float v = lane < rows ? static_cast<float>(dg) : 0.f;
        if (a.d_f32) static_cast<float*>(ba.dd)[i] = v;
        else static_cast<raw*>(ba.dd)[i] = ET<E>::from_f(v);
      }
    }
    if (g == 0 && tok < all) {
      const int64_t i = (b * a.T + t0 + tok) * a.H + h;
      const float v = in ? dbs : 0.f;
      if (a.s_f32) static_cast<float*>(ba.ds)[i] = v;
      else static_cast<raw*>(ba.ds)[i] = ET<E>::from_f(v);
    }
    // dQ^T += K^T Y^T, dK^T += K^T (X + X^T) + Q^T Y.
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      float yr[8], xr[8], yc[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int k = 32 * s + (e < 4 ? 4 * g + e : 12 + 4 * g + e);
        // (16 x 16 tiles above the diagonal of Y are not written.)
        yr[e] = (k >> 4) <= w ? ym[tok * L::XS + k] : 0.f;
        yc[e] = (k >> 4) >= w ? ym[k * L::XS + tok] : 0.f;
        xr[e] = xm[tok * L::XS + k];
      }
      B8 yp[NO], xp[NO], cp[NO];
      split8<NO>(yr, yp);
      split8<NO>(xr, xp);
      split8<NO>(yc, cp);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        B8 kf[NI], qf[NI];
        col_parts<ST, NI>(kt, L::kpart, 32 * s, 16 * i, kf);
        col_parts<ST, NI>(qt, L::kpart, 32 * s, 16 * i, qf);
        dq[i] = mma_parts<NO>(kf, yp, dq[i]);
        dk[i] = mma_parts<NO>(kf, xp, dk[i]);
        dk[i] = mma_parts<NO>(qf, cp, dk[i]);
      }
    }
  }
  // Rows behind the length.
  if (rows < all) {
    for (int h = h0; h < h1; ++h) {
      for (int i = tid; i < (all - rows) * a.P; i += kThreads) {
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
    const int64_t to = ((b * a.T + t0 + tok) * a.G + gi) * a.N;
    const int64_t plane = static_cast<int64_t>(a.B) * a.T * a.G * a.N;
    const bool whole = (a.N & 3) == 0;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int k = 16 * i + 4 * g;
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
        if (whole) {
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
  int64_t chunks, states, du, part, bytes;
};
Work work_of(int64_t B, int64_t T, int64_t H, int64_t P, int64_t G, int64_t N) {
  const int64_t C = (T + kDTokens - 1) / kDTokens, shares = share_count(B, C, H, G);
  Work w{};
  w.chunks = 0;
  w.states = up16(B * H * C * delta_chunk_bytes(3));
  w.du = w.states + up16(B * C * H * P * N * 4);
  w.part = w.du + up16(B * T * H * P * 4);
  w.bytes = w.part + (shares > 1 ? 2 * shares * B * T * G * N * 4 : 0);
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
  if (u->seq_len > 0) {
    a.gstates = reinterpret_cast<float*>(a.f.work + wk.states);
    a.du = reinterpret_cast<float*>(a.f.work + wk.du);
    a.shares = share_count(u->batch, a.f.C, u->heads, u->groups);
    a.per = static_cast<int>((u->heads / u->groups + a.shares - 1) / a.shares);
    a.part = a.shares > 1 ? reinterpret_cast<float*>(a.f.work + wk.part) : nullptr;
    if (int rc = launch_delta_prep(a.f, u->dtype, true, hs, what)) return rc;
  }
  auto set_lds = [&](const void* kernel, size_t bytes) {
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e == hipSuccess) return GRM_HIP_OK;
    set_error("%s: %s", what, hipGetErrorString(e));
    return static_cast<int>(e);
  };
  int rc = GRM_HIP_OK;
  delta_with_form(u->dtype, a.f.N, a.f.vec != 0 && aligned(grad_hidden), [&](auto e, auto nk, auto vec) {
    using E = decltype(e);
    constexpr int NK = decltype(nk)::value;
    constexpr bool VEC = decltype(vec)::value;
    {
      auto kernel = delta_reverse_kernel<E, NK, VEC>;
      constexpr size_t lds = ReverseLds<E, NK>::bytes;
      if ((rc = set_lds(reinterpret_cast<const void*>(kernel), lds)) != GRM_HIP_OK) return;
      kernel<<<dim3(static_cast<uint32_t>(a.f.B) * a.f.H * a.f.PT), dim3(kThreads), lds, hs>>>(a);
      if ((rc = check_launch(what)) != GRM_HIP_OK || a.f.C == 0) return;
    }
    auto kernel = delta_grad_kernel<E, NK, VEC>;
    constexpr size_t lds = GradLds<E, NK>::bytes;
    if ((rc = set_lds(reinterpret_cast<const void*>(kernel), lds)) != GRM_HIP_OK) return;
    kernel<<<dim3(static_cast<uint32_t>(a.f.B) * a.f.C * a.f.G * a.shares), dim3(kThreads), lds, hs>>>(a);
    if ((rc = check_launch(what)) != GRM_HIP_OK || a.part == nullptr) return;
    const int64_t plane = static_cast<int64_t>(a.f.B) * a.f.T * a.f.G * a.f.N, blocks = (2 * plane + kThreads - 1) / kThreads;
    delta_share_sum_kernel<E><<<dim3(static_cast<uint32_t>(blocks < 4096 ? blocks : 4096)), dim3(kThreads), 0, hs>>>(
        a.part, a.dk, a.dq, plane, a.shares);
    rc = check_launch(what);
  });
  return rc;
}
