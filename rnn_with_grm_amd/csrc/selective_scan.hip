// Selective state scan (forward) and its single-token form, gfx950.
//
//   d_t = softplus(steps_t + bias),  M_t = exp(d_t A) M_{t-1} + d_t v_t k_t^T,  h_t = M_t q_t + D v_t
//
// per head, state M of [P value rows, N key columns], keys and queries shared by the heads of a
// group.  Over a chunk of L tokens from state M, with c_i the summed log decays:
//   h_i = e^{c_i} M q_i + sum_{j<=i} e^{c_i - c_j} d_j (q_i . k_j) v_j + D v_i
//   M'  = e^{c_L} M + sum_j e^{c_L - c_j} d_j v_j k_j^T
//
// One workgroup walks one (sequence, head, 64 value rows) chunk by chunk, so the inputs are read
// and the outputs written once, and no state but the last one reaches memory (under autograd: one
// per 128 tokens).  Eight waves in two roles with one barrier a chunk.  In the step of chunk c
//   waves 0-3  bring chunk c + 2 from memory into the third of three LDS stages, and form the weights
//              between the tokens of chunk c + 1, e^{c_i - c_j} d_j (q_i . k_j), into one of two LDS tiles;
//   waves 4-7  hold the state in float32 accumulators, 16 value rows each, which lie as the queries' product
//              wants its operand; they write the chunk's outputs and move the state.
// Where heads are too few to fill 256 CUs, sequences are cut in time: a first launch sums each part's own
// writes, and each part of the second starts from the combination of the parts before it.
#include <stdint.h>

#include "selective.h"

namespace grmhip {
namespace {

constexpr int kWalkThreads = 512;
constexpr int kPassThreads = 512;
constexpr int kStepThreads = 256;
constexpr int kMaxParts = 32;

// Weights between a chunk's tokens in LDS: the 16 x 16 tiles on and below the diagonal, each as its lanes hold it, four
// columns a lane, which is how the product reads it again.  bfloat16 inputs: as two bfloat16 parts, as is the state where a
// query reads it: 2^-16 of a term is lost, far below the rounding of the output that it is summed into.  (8 x 2048 tokens x
// 32 heads take 101 us so; with one part, whose 2^-8 of every term is seen in the outputs, they took 90.)
template <class M>
struct WeightTile {
  static constexpr int NIT = SelShape<M>::L / 16, TILES = NIT * (NIT + 1) / 2;
  static constexpr int PARTS = SelShape<M>::kHalf ? 2 : 1, PART = TILES * 256;
  using raw = typename ET<M>::raw;
  __device__ __forceinline__ static int at(int it, int jt, int lane) { return (it * (it + 1) / 2 + jt) * 256 + 4 * lane; }
  __device__ __forceinline__ static void put(raw* m, int it, int jt, int lane, f32x4 v) {
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      store4_raw<M>(m + p * PART + at(it, jt, lane), v);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = part_rest<M>(v[r], ET<M>::from_f(v[r]));
    }
  }
  // Row tile `it`, columns 32 s to 32 s + 31: zeros where they lie in a tile above the diagonal.
  __device__ __forceinline__ static Frag8<M> frag(const raw* m, int part, int it, int s, int lane) {
    const raw* p = m + part * PART + at(it, 2 * s, lane);
    if (2 * s + 1 <= it) return lds_frag_4x2<M>(p, p + 256);
    Frag8<M> f = {};
#pragma unroll
    for (int e = 0; e < 4; ++e) f.e[e] = p[e];
    return f;
  }
};

template <class M, int NP>
struct WalkLds {
  using S = SelShape<M>;
  using KT = SelTile<M, NP, true>;         // keys: columns
  using QT = SelTile<M, NP, false>;        // queries: rows in 8-byte pieces
  using XT = SelTile<M, kSelRows, true>;   // values: columns
  using W4 = WeightTile<M>;                // weights between tokens
  static constexpr int Q0 = S::L * KT::STRIDE, X0 = Q0 + S::L * QT::STRIDE;
  static constexpr int STAGES = 3, STAGE = X0 + S::L * XT::STRIDE;  // a chunk's tiles
  static constexpr int MIX = W4::PARTS * W4::PART;  // a chunk's weights
  static constexpr int SCAL = 5 * S::L + 8;  // hi, lo, d, tail weight, decay; total; whether a value is infinite or NaN, by wave
  static constexpr size_t bytes =
      (STAGES * STAGE + 2 * MIX) * sizeof(typename ET<M>::raw) + STAGES * SCAL * sizeof(float);
  static_assert(bytes <= 160 * 1024, "one CU's LDS");
};

struct WalkPlace {
  int b, h, g, pt, part;
};

__device__ __forceinline__ WalkPlace walk_place(const SelArgs& a, uint32_t v) {
  WalkPlace w;
  w.pt = static_cast<int>(v % a.PT);
  v /= a.PT;
  w.h = static_cast<int>(v % a.H);
  v /= a.H;
  w.part = static_cast<int>(v % a.parts);
  w.b = static_cast<int>(v / a.parts);
  w.g = w.h / (a.H / a.G);
  return w;
}

// A part's starting state: the given one and the sums of the parts before (REV: behind) it, decayed.
template <int NT, bool REV>
__device__ __forceinline__ void part_start(f32x4 (&acc)[NT], const SelArgs& a, const WalkPlace& w, int p0) {
  const int64_t head = static_cast<int64_t>(w.b) * a.H + w.h, one = static_cast<int64_t>(a.P) * a.N;
  const int64_t all = static_cast<int64_t>(a.B) * a.H;
  double log = 0.0;
  const int end = REV ? a.parts : -1;
  for (int q = REV ? w.part + 1 : w.part - 1; q != end; q += REV ? 1 : -1) {
    state_add<NT>(acc, a.part_state + (q * all + head) * one, p0, a.P, a.N, exp2_d(log));
    log += a.part_log[q * all + head];
  }
  if (a.memory != nullptr) state_add<NT>(acc, a.memory + head * one, p0, a.P, a.N, exp2_d(log));
}

template <class E, class M, int NP, bool VEC>
__global__ __launch_bounds__(kWalkThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void selective_walk_kernel(SelArgs a) {
  using S = SelShape<M>;
  using Lds = WalkLds<M, NP>;
  using raw = typename ET<M>::raw;
  using eraw = typename ET<E>::raw;
  using KT = typename Lds::KT;
  using QT = typename Lds::QT;
  using XT = typename Lds::XT;
  using W4 = typename Lds::W4;
  constexpr int L = S::L, NT = NP / 16, NK = NP / 32, NIT = L / 16, NS32 = L / 32;
  extern __shared__ __align__(16) unsigned char smem[];
  raw* stage = reinterpret_cast<raw*>(smem);
  raw* mix = stage + Lds::STAGES * Lds::STAGE;
  float* scal = reinterpret_cast<float*>(mix + 2 * Lds::MIX);

  const WalkPlace w = walk_place(a, xcd_order(blockIdx.x, gridDim.x));
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, g = lane >> 4, n16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int p0 = w.pt * kSelRows, pw = a.P - p0;
  const int64_t len = sel_length(a, w.b);
  const int64_t t_first = w.part * a.part_tokens, t_last = min_i64(t_first + a.part_tokens, a.T);
  const int live = static_cast<int>(max_i64(0, min_i64(len, t_last) - t_first));  // tokens of this walk
  const int chunks = (live + L - 1) / L;
  eraw* hid = static_cast<eraw*>(a.hidden) + ((w.b * a.T + t_first) * a.H + w.h) * a.P + p0;
  const int64_t hstride = static_cast<int64_t>(a.H) * a.P;

  if (wave < 4) {
    const float rate = a.rates[w.h], bias = a.bias == nullptr ? 0.f : a.bias[w.h];
    const eraw* kp = static_cast<const eraw*>(a.keys) + w.b * a.kb + t_first * a.kt + w.g * a.N;
    const eraw* qp = static_cast<const eraw*>(a.queries) + w.b * a.qb + t_first * a.qt + w.g * a.N;
    const eraw* xp = static_cast<const eraw*>(a.values) + w.b * a.vb + t_first * a.vt + w.h * a.P + p0;
    TileLoad<E, KT, M, VEC, L, NP, kWalkThreads / 2> kr;
    TileLoad<E, QT, M, VEC, L, NP, kWalkThreads / 2> qr;
    TileLoad<E, XT, M, VEC, L, kSelRows, kWalkThreads / 2> xr;
    kr.init(a.kt, a.N, tid);
    qr.init(a.qt, a.N, tid);
    xr.init(a.vt, pw < kSelRows ? pw : kSelRows, tid);
    uint32_t z = 0;  // the loaded chunk's steps
    constexpr int kStepWave = 3;
    int at = 0;      // tokens before the next chunk to load
    auto load = [&]() {
      kr.load(kp + at * a.kt, live - at, tid);
      qr.load(qp + at * a.qt, live - at, tid);
      xr.load(xp + at * a.vt, live - at, tid);
      if (wave == kStepWave) z = load_step<E>(a, w.b, t_first + at + lane, w.h, lane < L && at + lane < live);
      at += L;
    };
    auto put = [&](int slot) {
      raw* s = stage + slot * Lds::STAGE;
      kr.store(s, tid);
      qr.store(s + Lds::Q0, tid);
      xr.store(s + Lds::X0, tid);
      const bool odd = __any(xr.odd());
      if (lane == 0) scal[slot * Lds::SCAL + 5 * L + 4 + wave] = odd ? 1.f : 0.f;
      if (wave == kStepWave) {
        const TokenScalars s = token_scalars<L>(a, step_value<E>(a, z) + bias, at - L + lane < live, rate);
        float* o = scal + slot * Lds::SCAL;
        if (lane < L) {
          const float hi = static_cast<float>(s.cum);
          o[lane] = hi;
          o[L + lane] = static_cast<float>(s.cum - hi);
          o[2 * L + lane] = s.d;
          o[3 * L + lane] = s.d * exp2_d(s.total - s.cum);
          o[4 * L + lane] = exp2_d(s.cum);
        }
        if (lane == 0) o[5 * L] = exp2_d(s.total);
      }
    };
    // 16-bit types: waves 0 to 2 form a 32 x 32 block of the weights each, its fragments read once for two tiles;
    // float32: waves 0 to 2 one tile each.  The last wave has the step sizes.
    auto weights = [&](int slot, int c) {
      if (wave == 3) return;
      const raw *ks = stage + slot * Lds::STAGE, *qs = ks + Lds::Q0;
      const float* sc = scal + slot * Lds::SCAL;
      raw* m = mix + (c & 1) * Lds::MIX;
      constexpr int NB = NIT / 2;  // tiles of a block each way
      const int it0 = NB * (wave == 1 ? 0 : 1), jt0 = NB * (wave == 2 ? 1 : 0);
      Frag8<M> kf[NB][NK], qf[NB][NK];
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) {
#pragma unroll
        for (int u = 0; u < NB; ++u) {
          kf[u][kk] = row_frag<KT, M>(ks, (jt0 + u) * 16, kk * 32);
          qf[u][kk] = row_frag<QT, M>(qs, (it0 + u) * 16, kk * 32);
        }
      }
      hold_order();
#pragma unroll
      for (int u = 0; u < NB; ++u) {
#pragma unroll
        for (int v = 0; v < NB; ++v) {
          const int it = it0 + u, jt = jt0 + v;
          if (jt > it) continue;
          f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kk = 0; kk < NK; ++kk) d = mfma8(kf[v][kk], qf[u][kk], d);
          const int j0 = jt * 16 + 4 * g, i = it * 16 + n16;
          const f32x4 hj = *reinterpret_cast<const f32x4*>(sc + j0), lj = *reinterpret_cast<const f32x4*>(sc + L + j0),
                      dj = *reinterpret_cast<const f32x4*>(sc + 2 * L + j0);
          const float hi_i = sc[i], lo_i = sc[L + i];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            // Above the diagonal both factors are zeros: a select of their product would become a branch round
            // the exponential.
            const bool in = j0 + r <= i;
            const float x = (hi_i - hj[r]) + (lo_i - lj[r]);
            d[r] = (in ? d[r] * dj[r] : 0.f) * exp2_f(in ? x : -INFINITY);
          }
          W4::put(m, it, jt, lane, d);
        }
      }
    };
    if (chunks > 0) {
      load();
      put(0);
      if (chunks > 1) load();
    }
    __syncthreads();
    if (chunks > 0) weights(0, 0);
    if (chunks > 1) put(1);
    __syncthreads();
    int s1 = 1, s2 = 2;  // stages of chunks c + 1 and c + 2
    for (int c = 0; c < chunks; ++c) {
      if (c + 2 < chunks) load();
      if (c + 1 < chunks) weights(s1, c + 1);
      if (c + 2 < chunks) put(s2);
      __syncthreads();
      s1 = s2;
      s2 = s2 == 2 ? 0 : s2 + 1;
    }
  } else {
    const int rw = 16 * (wave & 3), sp = p0 + rw;  // this wave's first row
    const float skip = a.skip == nullptr ? 0.f : a.skip[w.h];
    f32x4 acc[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    part_start<NT, false>(acc, a, w, sp);
    const int col = rw + 4 * g;  // this lane's first value column, of four
    const bool hvec = VEC && (a.P & 3) == 0;
    __syncthreads();
    __syncthreads();
    int s0 = 0;  // stage of chunk c
    Frag8<M> qf[NK][NIT];
    auto ask_queries = [&](int slot) {
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) {
#pragma unroll
        for (int it = 0; it < NIT; ++it) qf[kk][it] = row_frag_t<QT, M>(stage + slot * Lds::STAGE + Lds::Q0, it * 16, kk * 32);
      }
    };
    if (chunks > 0) ask_queries(0);
    for (int c = 0; c < chunks; ++c) {
      const raw* ks = stage + s0 * Lds::STAGE;
      const raw* xs = ks + Lds::X0;
      const float* sc = scal + s0 * Lds::SCAL;
      const raw* m = mix + (c & 1) * Lds::MIX;
      if (a.states != nullptr && c * L % S::LB == 0) {
        const int64_t blk = (t_first + static_cast<int64_t>(c) * L) / S::LB;
        state_store<NT>(acc, a.states + ((w.b * a.nsave + blk) * a.H + w.h) * a.P * a.N, sp, a.P, a.N);
      }
      // Reads are issued a phase ahead of the products that want them: the weights and the first keys with
      // the state's product, the next chunk's queries with the last of the update.
      Frag8<M> xf[NS32], mf[NS32][NIT], kf[NT];
      f32x4 xv[NIT];
      float e[NIT];
#pragma unroll
      for (int it = 0; it < NIT; ++it) e[it] = sc[4 * L + it * 16 + n16];
      const f32x4 flags = *reinterpret_cast<const f32x4*>(sc + 5 * L + 4);
#pragma unroll
      for (int s = 0; s < NS32; ++s) {
        xf[s] = col_frag<XT, M>(xs, 32 * s, rw);
#pragma unroll
        for (int it = 2 * s; it < NIT; ++it) mf[s][it] = W4::frag(m, W4::PARTS - 1, it, s, lane);
      }
      hold_order();
      f32x4 y[NIT];
#pragma unroll
      for (int it = 0; it < NIT; ++it) y[it] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) {
        Frag8<M> sf[W4::PARTS];
        split_pair<M>(acc[2 * kk], acc[2 * kk + 1], sf);
#pragma unroll
        for (int p = W4::PARTS - 1; p >= 0; --p) {
#pragma unroll
          for (int it = 0; it < NIT; ++it) y[it] = mfma8(sf[p], qf[kk][it], y[it]);
        }
      }
      const bool odd = __any(flags[0] + flags[1] + flags[2] + flags[3] != 0.f);
      if (__builtin_expect(odd, 0)) {
        // A weight of zero does not keep an infinity or a NaN out of a product: all outputs one token i at a time, with
        // the values of the tokens behind it taken out.  (The lane's number anew: what is made of it here is not to be
        // kept in registers for the case.)
        int ln = lane_id();
        asm volatile("" : "+v"(ln));
#pragma unroll
        for (int it = 0; it < NIT; ++it) {
          f32x4 from;
#pragma unroll
          for (int r = 0; r < 4; ++r) from[r] = y[it][r] * e[it];
#pragma unroll 1
          for (int k = 0; k < 16; ++k) {
            f32x4 one = from;
#pragma unroll
            for (int s = 0; 2 * s <= it; ++s) {
              Frag8<M> x = xf[s];
#pragma unroll
              for (int u = 0; u < 8; ++u) {
                const int t = 32 * s + 4 * (ln >> 4) + (u < 4 ? u : 12 + u);
                x.e[u] = t <= it * 16 + k ? x.e[u] : static_cast<raw>(0);
              }
              one = mfma8(x, W4::frag(m, 0, it, s, ln), one);
              if constexpr (W4::PARTS == 2) {  // a weight's rest is of either sign or zero: not for an infinity
#pragma unroll
                for (int u = 0; u < 8; ++u) x.e[u] = isfinite(ET<M>::to_f(x.e[u])) ? x.e[u] : static_cast<raw>(0);
                one = mfma8(x, W4::frag(m, 1, it, s, ln), one);
              }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) y[it][r] = (ln & 15) == k ? one[r] : y[it][r];
          }
        }
      }
      key_frags<KT, M, NT>(kf, ks, 0);
#pragma unroll
      for (int it = 0; it < NIT; ++it) xv[it] = lds_row4<M>(xs + XT::at(it * 16 + n16, col));
      f32x4 w0 = *reinterpret_cast<const f32x4*>(sc + 3 * L + 4 * g), w1 = *reinterpret_cast<const f32x4*>(sc + 3 * L + 16 + 4 * g);
      const float decay = sc[5 * L];
      Frag8<M> mt[NS32][NIT];  // the weights' first part
      if constexpr (W4::PARTS == 2) {
#pragma unroll
        for (int s = 0; s < NS32; ++s) {
#pragma unroll
          for (int it = 2 * s; it < NIT; ++it) mt[s][it] = W4::frag(m, 0, it, s, lane);
        }
      }
      hold_order();
      if (__builtin_expect(!odd, 1)) {
#pragma unroll
        for (int it = 0; it < NIT; ++it) {
#pragma unroll
          for (int r = 0; r < 4; ++r) y[it][r] *= e[it];
        }
#pragma unroll
        for (int s = 0; s < NS32; ++s) {
#pragma unroll
          for (int it = 2 * s; it < NIT; ++it) y[it] = mfma8(xf[s], mf[s][it], y[it]);
        }
        if constexpr (W4::PARTS == 2) {
#pragma unroll
          for (int s = 0; s < NS32; ++s) {
#pragma unroll
            for (int it = 2 * s; it < NIT; ++it) y[it] = mfma8(xf[s], mt[s][it], y[it]);
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[nt][r] *= decay;
      }
      Frag8<M> part[S::PARTS];
      weigh_frag<M>(xf[0], w0, w1, part);
#pragma unroll
      for (int it = 0; it < NIT; ++it) {
        const int t = c * L + it * 16 + n16;
        f32x4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r)  // (without `skip` no product with zero: an infinite value would make a NaN of it)
          v[r] = t < live ? (a.skip != nullptr ? fmaf(skip, xv[it][r], y[it][r]) : y[it][r]) : 0.f;
        if (t_first + t < t_last) {
          eraw* o = hid + t * hstride + col;
          if (hvec) {
            if (col < pw) {
              if constexpr (sizeof(eraw) == 2) {
                typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
                store_as(reinterpret_cast<u32x2*>(o), u32x2{pack2<E>(v[0], v[1]), pack2<E>(v[2], v[3])}, a.stream != 0);
              } else {
                store_as(reinterpret_cast<f32x4*>(o), v, a.stream != 0);
              }
            }
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              if (col + r < pw) o[r] = ET<E>::from_f(v[r]);
            }
          }
        }
      }
#pragma unroll
      for (int s = 0; s < NS32; ++s) {
        Frag8<M> kn[NT];
        if (s + 1 < NS32) {
          key_frags<KT, M, NT>(kn, ks, 32 * (s + 1));
          w0 = *reinterpret_cast<const f32x4*>(sc + 3 * L + 32 * (s + 1) + 4 * g);
          w1 = *reinterpret_cast<const f32x4*>(sc + 3 * L + 32 * (s + 1) + 16 + 4 * g);
        }
        if (s + 1 == NS32 && c + 1 < chunks) ask_queries(s0 == 2 ? 0 : s0 + 1);
        hold_order();
        update_step<M, NT>(acc, kf, part);
        if (s + 1 < NS32) {
          weigh_frag<M>(xf[s + 1 < NS32 ? s + 1 : 0], w0, w1, part);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) kf[nt] = kn[nt];
        }
      }
      if (__builtin_expect(odd && a.N < NP, 0)) {  // an infinity times the zeros of the columns past the keys' width
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[nt][r] = nt * 16 + 4 * g + r < a.N ? acc[nt][r] : 0.f;
        }
      }
      __syncthreads();
      s0 = s0 == 2 ? 0 : s0 + 1;
    }
    if (w.part == a.parts - 1)
      state_store<NT>(acc, a.memory_out + (static_cast<int64_t>(w.b) * a.H + w.h) * a.P * a.N, sp, a.P, a.N);
  }
  // Tokens behind the length (the walk's last chunk has written its own).
  const int cols = pw < kSelRows ? pw : kSelRows;
  for (int64_t t = chunks * L + wave; t < t_last - t_first; t += kWalkThreads / 64) {
    if (lane < cols) hid[t * hstride + lane] = ET<E>::from_f(0.f);
  }
}

// The state's walk alone.  Forward: from zero over a part, leaving the part's sum and log decay.  REV
// (the backward's adjoint): `keys` are the queries and `values` the output's gradient,
//   G_{before} = e^{c_L} G + sum_i e^{c_i} dy_i q_i^T,
// from the gradient of the final state back to the first, G kept at the end of every backward chunk.
// Waves 0-3 bring the chunks, one in LDS and one on its way; waves 4-7 hold 16 rows of the state each.  (One
// role for all waves measured 120 us at 8 x 2048 tokens x 32 heads where this took 96: a state's stores then stand between a load and its use.)
template <class E, class M, int NP, bool VEC, bool REV, bool LOCAL>
__global__ __launch_bounds__(kPassThreads) __attribute__((amdgpu_waves_per_eu(2, 4))) void selective_pass_kernel(SelArgs a) {
  using S = SelShape<M>;
  using raw = typename ET<M>::raw;
  using eraw = typename ET<E>::raw;
  using KT = SelTile<M, NP, true>;
  using XT = SelTile<M, kSelRows, true>;
  constexpr int L = S::L, NT = NP / 16, X0 = L * KT::STRIDE, STAGE = X0 + L * XT::STRIDE, SCAL = L + 4;
  // The adjoint of bfloat16 inputs changes its sign from chunk to chunk, against the bf16 products' leaning to one side (see
  // selective_grad_kernel): it meets keys and values that are mostly of one sign in the step sizes' gradients.
  constexpr bool TURN = REV && S::kHalf;
  extern __shared__ __align__(16) unsigned char smem[];
  raw* stage = reinterpret_cast<raw*>(smem);
  float* scal = reinterpret_cast<float*>(stage + 2 * STAGE);

  const WalkPlace w = walk_place(a, xcd_order(blockIdx.x, gridDim.x));
  // Parts whose sums nothing asks for: the last one of a forward walk, the first of a reverse one.
  if (LOCAL && w.part == (REV ? 0 : a.parts - 1)) return;
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int p0 = w.pt * kSelRows, pw = a.P - p0;
  const int64_t t_first = w.part * a.part_tokens, t_last = min_i64(t_first + a.part_tokens, a.T);
  const int live = static_cast<int>(max_i64(0, min_i64(sel_length(a, w.b), t_last) - t_first));
  const int chunks = (live + L - 1) / L;
  const int64_t head = static_cast<int64_t>(w.b) * a.H + w.h, one = static_cast<int64_t>(a.P) * a.N;
  const int64_t slot = static_cast<int64_t>(w.part) * a.B * a.H + head;
  auto chunk_of = [&](int i) { return REV ? chunks - 1 - i : i; };
  if (wave < 4) {
    constexpr int kStepWave = 3;
    const float rate = a.rates[w.h], bias = a.bias == nullptr ? 0.f : a.bias[w.h];
    TileLoad<E, KT, M, VEC, L, NP, kPassThreads / 2> kr;
    TileLoad<E, XT, M, VEC, L, kSelRows, kPassThreads / 2> xr;
    kr.init(a.kt, a.N, tid);
    xr.init(a.vt, pw < kSelRows ? pw : kSelRows, tid);
    const eraw* kp = static_cast<const eraw*>(a.keys) + w.b * a.kb + t_first * a.kt + w.g * a.N;
    const eraw* xp = static_cast<const eraw*>(a.values) + w.b * a.vb + t_first * a.vt + w.h * a.P + p0;
    uint32_t z = 0;  // the chunk's steps
    double log = 0.0;
    auto load = [&](int i) {
      const int t = chunk_of(i) * L;
      kr.load(kp + t * a.kt, live - t, tid);
      xr.load(xp + t * a.vt, live - t, tid);
      if (wave == kStepWave) z = load_step<E>(a, w.b, t_first + t + lane, w.h, lane < L && t + lane < live);
    };
    auto put = [&](int i) {
      raw* s = stage + (i & 1) * STAGE;
      kr.store(s, tid);
      xr.store(s + X0, tid);
      if (wave == kStepWave) {
        const TokenScalars t = token_scalars<L>(a, step_value<E>(a, z) + bias, chunk_of(i) * L + lane < live, rate);
        float* o = scal + (i & 1) * SCAL;
        if (lane < L) o[lane] = REV ? (TURN && !(i & 1) ? -1.f : 1.f) * exp2_d(t.cum) : t.d * exp2_d(t.total - t.cum);
        if (lane == 0) o[L] = (TURN ? -1.f : 1.f) * exp2_d(t.total);
        log += t.total;
      }
    };
    if (chunks > 0) {
      load(0);
      put(0);
      if (chunks > 1) load(1);
    }
    __syncthreads();
    for (int i = 0; i < chunks; ++i) {
      if (i + 1 < chunks) put(i + 1);
      if (i + 2 < chunks) load(i + 2);
      __syncthreads();
    }
    if (LOCAL && wave == kStepWave && lane == 0 && w.pt == 0) a.part_log[slot] = log;
  } else {
    const int rw = 16 * (wave & 3), sp = p0 + rw, g = lane >> 4;
    f32x4 acc[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (!LOCAL) part_start<NT, REV>(acc, a, w, sp);
    __syncthreads();
    for (int i = 0; i < chunks; ++i) {
      const raw* ks = stage + (i & 1) * STAGE;
      const float* sc = scal + (i & 1) * SCAL;
      Frag8<M> xf[L / 32], kf[NT], part[S::PARTS];
#pragma unroll
      for (int s = 0; s < L / 32; ++s) xf[s] = col_frag<XT, M>(ks + X0, 32 * s, rw);
      key_frags<KT, M, NT>(kf, ks, 0);
      if (REV && !LOCAL) {
        const int64_t t = t_first + static_cast<int64_t>(chunk_of(i)) * L;
        if (i == 0 || (t + L) % S::LB == 0)
          state_store<NT>(acc, a.states + ((w.b * a.nsave + t / S::LB) * a.H + w.h) * a.P * a.N, sp, a.P, a.N,
                          TURN && (i & 1) ? -1.f : 1.f);
      }
      const float decay = sc[L];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[nt][r] *= decay;
      }
#pragma unroll
      for (int s = 0; s < L / 32; ++s) {
        weigh_frag<M>(xf[s], *reinterpret_cast<const f32x4*>(sc + 32 * s + 4 * g),
                      *reinterpret_cast<const f32x4*>(sc + 32 * s + 16 + 4 * g), part);
        update_step<M, NT>(acc, kf, part);
        if (s + 1 < L / 32) key_frags<KT, M, NT>(kf, ks, 32 * (s + 1));
      }
      __syncthreads();
    }
    const float sign = TURN && (chunks & 1) ? -1.f : 1.f;
    if (LOCAL) state_store<NT>(acc, a.part_state + slot * one, sp, a.P, a.N, sign);
    else if (w.part == 0) state_store<NT>(acc, a.memory_out + head * one, sp, a.P, a.N, sign);
  }
}

// One token: a row of the state lies on LPR lanes (4 columns each), a wave moves 64 / LPR rows at a
// time, each element read and written by one thread (so memory_out may be memory).
template <class E, int LPR>
__global__ __launch_bounds__(kStepThreads) void selective_step_kernel(SelArgs a) {
  using raw = typename ET<E>::raw;
  constexpr int RPW = 64 / LPR, U = 4;  // rows a wave moves at once, and in how many loads
  const int lane = lane_id(), wave = static_cast<int>(threadIdx.x) >> 6;
  const int head = static_cast<int>(blockIdx.x), b = head / a.H, h = head - b * a.H, gi = h / (a.H / a.G);
  const int col = lane % LPR * 4;
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
  const float d = step_size(a, raw_step<E>(a, b, 0, h));
  const float keep = __expf(d * a.rates[h]), skip = a.skip == nullptr ? 0.f : a.skip[h];
  const raw* xp = static_cast<const raw*>(a.values) + b * a.vb + static_cast<int64_t>(h) * a.P;
  const float* mp = a.memory + static_cast<int64_t>(head) * a.P * a.N;
  float* op = a.memory_out + static_cast<int64_t>(head) * a.P * a.N;
  raw* hp = static_cast<raw*>(a.hidden) + static_cast<int64_t>(head) * a.P;
  const int stride = static_cast<int>(gridDim.y) * 4 * RPW * U;
  for (int p0 = (static_cast<int>(blockIdx.y) * 4 + wave) * RPW * U; p0 < a.P; p0 += stride) {
    float4 m[U];
    float x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int p = p0 + u * RPW + lane / LPR;
      m[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      x[u] = p < a.P ? ET<E>::to_f(xp[p]) : 0.f;
      if (p < a.P && col < a.N) {
        const float* s = mp + static_cast<int64_t>(p) * a.N + col;
        if (whole) {
          m[u] = *reinterpret_cast<const float4*>(s);
        } else {
          m[u].x = s[0];
          if (col + 1 < a.N) m[u].y = s[1];
          if (col + 2 < a.N) m[u].z = s[2];
          if (col + 3 < a.N) m[u].w = s[3];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int p = p0 + u * RPW + lane / LPR;
      const float dx = d * x[u];
      m[u].x = fmaf(dx, k[0], keep * m[u].x);
      m[u].y = fmaf(dx, k[1], keep * m[u].y);
      m[u].z = fmaf(dx, k[2], keep * m[u].z);
      m[u].w = fmaf(dx, k[3], keep * m[u].w);
      float y = fmaf(m[u].x, q[0], fmaf(m[u].y, q[1], fmaf(m[u].z, q[2], m[u].w * q[3])));
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) y += __shfl_xor(y, o);
      if (p < a.P && col < a.N) {
        float* s = op + static_cast<int64_t>(p) * a.N + col;
        if (whole) {
          store_as(reinterpret_cast<f32x4*>(s), f32x4{m[u].x, m[u].y, m[u].z, m[u].w}, a.stream != 0);
        } else {
          s[0] = m[u].x;
          if (col + 1 < a.N) s[1] = m[u].y;
          if (col + 2 < a.N) s[2] = m[u].z;
          if (col + 3 < a.N) s[3] = m[u].w;
        }
      }
      if (p < a.P && lane % LPR == 0) hp[p] = ET<E>::from_f(a.skip != nullptr ? fmaf(skip, x[u], y) : y);
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

uint32_t walk_blocks(const SelArgs& a) { return static_cast<uint32_t>(a.B) * a.H * a.PT * a.parts; }

}  // namespace

int64_t sel_block(int dtype) { return dtype == GRM_HIP_BF16 ? SelShape<BF16>::LB : SelShape<F32>::LB; }

// Enough parts for a workgroup on each of 256 CUs, of at least four backward chunks each: a part costs a
// second reading of its keys and values (32768 bf16 tokens x 16 heads of one sequence: 165 us in 16 parts,
// 1400 us in one).
int sel_parts(int64_t seqs, int64_t T, int dtype, int64_t* part_tokens) {
  const int64_t block = sel_block(dtype), blocks = T > 0 ? sel_ceil(T, block) : 1;
  int64_t parts = 256 / (seqs > 0 ? seqs : 1);
  if (parts > blocks / 4) parts = blocks / 4;
  if (parts > kMaxParts) parts = kMaxParts;
  if (parts < 1) parts = 1;
  const int64_t per = sel_ceil(blocks, parts);
  *part_tokens = per * block;
  return static_cast<int>(sel_ceil(blocks, per));
}

int sel_check(const grm_hip_selective_args* u, const char* what, bool step) {
  auto bad = [&](const char* why) {
    set_error("%s: %s", what, why);
    return GRM_HIP_EINVAL;
  };
  if (u == nullptr) return bad("no arguments");
  if (u->batch < 0 || u->seq_len < 0 || u->heads < 1 || u->value_dim < 1 || u->groups < 1 || u->key_dim < 1)
    return bad("batch and seq_len must be >= 0, the other sizes >= 1");
  if (u->heads % u->groups != 0) return bad("heads must be a multiple of groups");
  if (u->dtype < 0 || u->dtype > 2 || (u->steps_dtype != u->dtype && u->steps_dtype != GRM_HIP_F32)) {
    set_error("%s: keys, values and queries must be float32, float16 or bfloat16, steps the same or float32", what);
    return GRM_HIP_EUNSUPPORTED;
  }
  if (u->key_dim > 128) {
    set_error("%s: key_dim must be <= 128, got %lld", what, static_cast<long long>(u->key_dim));
    return GRM_HIP_EUNSUPPORTED;
  }
  const int64_t most = int64_t{1} << 21;
  if (u->seq_len > (1 << 30)) {
    set_error("%s: seq_len must be at most 2^30", what);
    return GRM_HIP_EUNSUPPORTED;
  }
  // (One by one first: no product passes 63 bits.)
  if (u->heads > most || u->value_dim > most || u->groups > most || u->keys_token_stride < 0 ||
      u->keys_token_stride > most || u->values_token_stride < 0 || u->values_token_stride > most ||
      u->queries_token_stride < 0 || u->queries_token_stride > most || u->heads * u->value_dim > most ||
      u->groups * u->key_dim > most) {
    set_error("%s: token strides and row widths must be at most 2^21 elements", what);
    return GRM_HIP_EUNSUPPORTED;
  }
  // (A grid dimension has fewer than 2^32 threads.)
  const int64_t batch = min_i64(u->batch, int64_t{1} << 32);
  const int64_t wgs = u->heads * batch * (step ? 1 : sel_ceil(u->value_dim, kSelRows)), threads = step ? kStepThreads : kWalkThreads;
  if (wgs * threads > UINT32_MAX) {
    set_error("%s: batch * heads%s must be below %lld", what, step ? "" : " * ceil(value_dim / 64)",
              static_cast<long long>((int64_t{UINT32_MAX} + 1) / threads));
    return GRM_HIP_EUNSUPPORTED;
  }
  if (u->seq_len > 1 && (u->keys_token_stride < u->groups * u->key_dim || u->queries_token_stride < u->groups * u->key_dim ||
                         u->values_token_stride < u->heads * u->value_dim))
    return bad("token strides must not be below a row's width");
  if (u->batch > 0 && u->rates == nullptr) return bad("rates are required");
  if (u->batch > 0 && u->seq_len > 0 &&
      (u->keys == nullptr || u->values == nullptr || u->queries == nullptr || u->steps == nullptr))
    return bad("keys, values, queries and steps are required");
  if (!aligned(u->memory)) return bad("memory must be 16-byte aligned");
  return GRM_HIP_OK;
}

SelArgs sel_args(const grm_hip_selective_args* u) {
  SelArgs a{};
  a.keys = u->keys; a.values = u->values; a.queries = u->queries; a.steps = u->steps;
  a.rates = u->rates; a.skip = u->skip; a.bias = u->step_bias; a.lengths = u->lengths; a.memory = u->memory;
  a.kb = u->keys_batch_stride; a.kt = u->keys_token_stride;
  a.vb = u->values_batch_stride; a.vt = u->values_token_stride;
  a.qb = u->queries_batch_stride; a.qt = u->queries_token_stride;
  a.sb = u->steps_batch_stride; a.st = u->steps_token_stride;
  a.T = u->seq_len;
  a.B = static_cast<int>(u->batch); a.H = static_cast<int>(u->heads); a.P = static_cast<int>(u->value_dim);
  a.G = static_cast<int>(u->groups); a.N = static_cast<int>(u->key_dim);
  a.PT = static_cast<int>(sel_ceil(u->value_dim, kSelRows));
  a.parts = 1;
  a.steps_f32 = u->steps_dtype == GRM_HIP_F32;
  a.softplus = u->softplus;
  // Whole 16-byte loads where every row of 8-element units allows them: 8 x 2048 bf16 tokens x 32 heads take half the
  // time of element by element so (121 and 240 us, back to back).
  a.vec = u->value_dim % 8 == 0 && u->key_dim % 8 == 0 && aligned(u->keys) && aligned(u->values) &&
          aligned(u->queries) && (u->keys_batch_stride | u->keys_token_stride | u->values_batch_stride |
                                  u->values_token_stride | u->queries_batch_stride | u->queries_token_stride) % 8 == 0;
  return a;
}

int launch_state_pass(const SelArgs& a, int dtype, bool reverse, bool local, hipStream_t stream, const char* what) {
  int rc = GRM_HIP_OK;
  sel_with_form(dtype, a.N, a.vec != 0, [&](auto e, auto m, auto np, auto vec) {
    constexpr bool VEC = decltype(vec)::value;
    using E = decltype(e);
    using M = decltype(m);
    constexpr int NP = decltype(np)::value;
    using S = SelShape<M>;
    constexpr size_t lds = 2 * S::L * (SelTile<M, NP, true>::STRIDE + SelTile<M, kSelRows, true>::STRIDE) * sizeof(typename ET<M>::raw) + 2 * (S::L + 4) * sizeof(float);
    auto go = [&](auto kernel) {
      if ((rc = set_lds(reinterpret_cast<const void*>(kernel), lds, what)) != GRM_HIP_OK) return;
      kernel<<<dim3(walk_blocks(a)), dim3(kPassThreads), lds, stream>>>(a);
      rc = check_launch(what);
    };
    if (reverse && local) go(selective_pass_kernel<E, M, NP, VEC, true, true>);
    else if (reverse) go(selective_pass_kernel<E, M, NP, VEC, true, false>);
    else go(selective_pass_kernel<E, M, NP, VEC, false, true>);
  });
  return rc;
}

}  // namespace grmhip

using namespace grmhip;

extern "C" int64_t grm_hip_selective_scan_block(int dtype) { return dtype < 0 || dtype > 2 ? 0 : sel_block(dtype); }

extern "C" int64_t grm_hip_selective_scan_workspace(int64_t batch, int64_t seq_len, int64_t heads, int64_t value_dim,
                                                    int64_t key_dim, int dtype) {
  if (batch <= 0 || seq_len < 0 || heads <= 0 || value_dim <= 0 || key_dim <= 0 || dtype < 0 || dtype > 2) return 0;
  int64_t per = 0;
  const int64_t parts = sel_parts(batch * heads * sel_ceil(value_dim, kSelRows), seq_len, dtype, &per);
  return parts == 1 ? 0 : sel_ceil(parts * batch * heads * 8, 16) * 16 + parts * batch * heads * value_dim * key_dim * 4;
}

extern "C" int grm_hip_selective_scan_fwd(const grm_hip_selective_args* u, void* hidden, float* memory_out,
                                          float* states, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "selective_scan";
  if (int rc = sel_check(u, what)) return rc;
  if (u->batch == 0) return GRM_HIP_OK;
  const int64_t state_bytes = u->batch * u->heads * u->value_dim * u->key_dim * 4;
  if (memory_out == nullptr || (u->seq_len > 0 && hidden == nullptr) || !aligned(memory_out) || !aligned(states)) {
    set_error("%s: hidden and memory_out are required, memory_out and states 16-byte aligned", what);
    return GRM_HIP_EINVAL;
  }
  if (ranges_overlap(u->memory, state_bytes, memory_out, state_bytes)) {
    set_error("%s: memory_out may not overlap memory", what);
    return GRM_HIP_EINVAL;
  }
  SelArgs a = sel_args(u);
  a.hidden = hidden; a.memory_out = memory_out; a.states = states;
  a.stream = sel_streams(u->batch * u->seq_len * u->heads * u->value_dim * (u->dtype == GRM_HIP_F32 ? 4 : 2));
  a.vec = a.vec && aligned(hidden);
  a.nsave = sel_ceil(u->seq_len, sel_block(u->dtype));
  a.parts = sel_parts(static_cast<int64_t>(a.B) * a.H * a.PT, a.T, u->dtype, &a.part_tokens);
  if (a.parts > 1) {
    if (workspace == nullptr || !aligned(workspace) ||
        workspace_bytes < grm_hip_selective_scan_workspace(u->batch, u->seq_len, u->heads, u->value_dim, u->key_dim, u->dtype)) {
      set_error("%s: workspace missing, misaligned or too small", what);
      return GRM_HIP_EINVAL;
    }
    a.part_log = static_cast<double*>(workspace);
    a.part_state = reinterpret_cast<float*>(static_cast<char*>(workspace) + sel_ceil(int64_t{a.parts} * a.B * a.H * 8, 16) * 16);
    if (int rc = launch_state_pass(a, u->dtype, false, true, static_cast<hipStream_t>(stream), what)) return rc;
  }
  int rc = GRM_HIP_OK;
  sel_with_form(u->dtype, a.N, a.vec != 0, [&](auto e, auto m, auto np, auto vec) {
    using E = decltype(e);
    using M = decltype(m);
    constexpr int NP = decltype(np)::value;
    auto kernel = selective_walk_kernel<E, M, NP, decltype(vec)::value>;
    if ((rc = set_lds(reinterpret_cast<const void*>(kernel), WalkLds<M, NP>::bytes, what)) != GRM_HIP_OK) return;
    kernel<<<dim3(walk_blocks(a)), dim3(kWalkThreads), WalkLds<M, NP>::bytes, static_cast<hipStream_t>(stream)>>>(a);
    rc = check_launch(what);
  });
  return rc;
}

extern "C" int grm_hip_selective_step(const grm_hip_selective_args* u, void* hidden, float* memory_out, void* stream) {
  const char* what = "selective_step";
  if (int rc = sel_check(u, what, true)) return rc;
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
  SelArgs a = sel_args(u);
  a.hidden = hidden; a.memory_out = memory_out;
  a.stream = sel_streams(state_bytes);
  auto go = [&](auto e, auto lpr) {
    constexpr int LPR = decltype(lpr)::value, rows = 4 * (64 / LPR) * 4;  // of a workgroup at a time
    const int64_t tiles = sel_ceil(a.P, rows), most = 65535;  // a grid's second dimension; the kernel goes round
    selective_step_kernel<decltype(e), LPR>
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
