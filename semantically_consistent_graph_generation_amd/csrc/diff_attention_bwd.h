// Differential attention, backward kernels.  Included by the translation unit of each element type.
//
//   dV = A^T dO,  dP = dO V^T (the same for both maps),  dS_i = w_i P_i (dP - delta_i) with w_1 = 1, w_2 = -lambda,
//   delta_i = sum_j P_i dP,  dQ_i = scale dS_i K_i,  dK_i = scale dS_i^T Q_i,  dlambda = - sum delta_2
//
// Two kernels, each of which owns what it writes (no atomics): one over queries for delta and dQ, one over keys for dK and dV.
// delta comes from a sweep of its own, formed in 32 bits: dlambda is its sum, and dS a difference with it (dO . out would save the sweep, but out
// is rounded, and the gradient of a row with one key would not be zero).
// Bound: neither the vector nor the matrix unit alone.  32 heads of 4096 x 4096, d = 64, dv = 128, bf16, mean of a trace (the forward 726 us): dQ 990 us,
// vector instructions issue in 60 % of the cycles, the matrix unit is busy in 44; dK 730 us, 51 and 39 %; dV 553 us, 45 and 39 %.  4096 causal, 8 heads on 4:
// dQ 73 + 114 with 5 + 8 for its joins, dK 137, dV 101, join 12, forward 167.
#pragma once
#include "diff_attention_fwd.h"

namespace scgg {
namespace diffattn {

template <class T, int DP, int DVP>
struct DqShape {
  static constexpr int P = Type<T>::planes, ND = (DP + 31) / 32;
  typedef Tile<2 * DP, P> KTile;
  typedef Tile<DVP, P> VTile;
  static constexpr int MERGE = 2 * 2 * ND * 16 * 64 * 4;
  static constexpr int TILES = KTile::BYTES + VTile::BYTES;
  static constexpr int WORDS = TILES > MERGE ? TILES : MERGE;
  static constexpr int LDS = WORDS + WINDOW * 8;
  static constexpr int MIN_BLOCKS = P == 3 ? 1 : 2;
};

// delta [B,H,3,N]: delta_1, delta_2, and the largest |dP| of the query.
// PHASE 0: both sweeps.  With few queries the keys are split over `dq_splits` workgroups, and the sweeps are launches of their own: 1 writes
// the splits' deltas to `part` (delta_join adds them), 2 the splits' dQ in 32 bits (dq_join).
template <class T, int DP, int DVP, int KW, int PHASE>
__global__ __launch_bounds__(THREADS, (DqShape<T, DP, DVP>::MIN_BLOCKS)) void dq_kernel(Args a) {
  typedef DqShape<T, DP, DVP> S;
  typedef typename S::KTile KTile;
  typedef typename S::VTile VTile;
  constexpr int P = S::P, QW = 4 / KW, BQ = 32 * QW, ND = S::ND;
  extern __shared__ __align__(256) char lds[];
  char* kt = lds;
  char* vt = lds + KTile::BYTES;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 5, l31 = lane & 31;
  const int qw = wave / KW, kw = wave - qw * KW;
  const int q_tiles = (a.N + BQ - 1) / BQ, splits = PHASE == 0 ? 1 : a.dq_splits;
  const unsigned whole = die_major(blockIdx.x, gridDim.x), id = whole / splits;
  const int split = PHASE == 0 ? 0 : (int)(whole - id * splits);
  const int bh = id / q_tiles, qt = a.causal ? q_tiles - 1 - (int)(id - bh * q_tiles) : (int)(id - bh * q_tiles);
  const int b = bh / a.H, h = bh - b * a.H, hk = h / (a.H / a.Hkv);
  const int q = qt * BQ + 32 * qw + l31;
  const bool q_on = q < a.N;
  const long long off = (long long)a.M - a.N;
  const T* kp = static_cast<const T*>(a.k) + b * a.kb + 2ll * hk * a.kh;
  const T* vp = static_cast<const T*>(a.v) + b * a.vb + (long long)hk * a.vh;

  Frag<P> qf[2][DP / 16], gf[DVP / 16];
  float mc[2], il[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    load_rows<T, DP>(qf[i], static_cast<const T*>(a.q) + b * a.qb + (long long)q * a.qn + (2ll * h + i) * a.qh, q_on, a.d, g);
    float2 st = make_float2(INFINITY, 0.f);
    if (q_on) st = a.stats[((long long)bh * 2 + i) * a.N + q];
    mc[i] = st.x;
    il[i] = st.y;
  }
  const bool seeing = il[0] != 0.f || il[1] != 0.f;   // a query that sees no key gets and gives no gradient, whatever its dO holds
  load_rows<T, DVP>(gf, static_cast<const T*>(a.dout) + b * a.gb + (long long)q * a.gn + (long long)h * a.gh, q_on && seeing, a.dv_w, g);
  // Odd queries take - dO: the matrix instructions round dP with a bias of one sign (fp16: 1e-2 of a step), and dlambda, the sum of P dP over all
  // queries, would add it up (2e-5 of 30 over 1554 queries); so it has the other sign in every second one.
  const float side = (l31 & 1) ? -1.f : 1.f;
  const unsigned flip = (l31 & 1) ? 0x80008000u : 0u;
#pragma unroll
  for (int c = 0; c < DVP / 16; ++c)
#pragma unroll
    for (int i = 0; i < P; ++i) gf[c].p[i] ^= flip;

  KeyBits keys;
  keys.mask = a.mask ? a.mask + b * a.mb : nullptr;
  keys.words = reinterpret_cast<u64*>(lds + S::WORDS);
  keys.M = a.M;
  keys.end = (a.M + TILE - 1) / TILE;
  if (a.causal) {
    const long long q_last = (qt + 1) * BQ < a.N ? (qt + 1) * BQ - 1 : a.N - 1, last = q_last + off;
    const int e = last < 0 ? 0 : (int)(last / TILE) + 1;
    if (e < keys.end) keys.end = e;
  }
  const long long wave_last = (long long)qt * BQ + 32 * qw + 31 + off;
  int first = 0;
  if constexpr (PHASE != 0) {
    const int tiles = keys.end;
    first = (int)((long long)tiles * split / splits);
    keys.end = (int)((long long)tiles * (split + 1) / splits);
  }

  Stage<T, 2 * DP, 2> ks;
  Stage<T, DVP, 1> vs;
  ks.init(a.kn, a.kh, a.d, tid);
  vs.init(a.vn, 0, a.dv_w, tid);
  auto score = [&](int i, int hh) {
    Dot<T> s;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) s.add(KTile::rows(kt, 32 * hh, i * (DP / 16) + c, lane), qf[i][c]);
    return s.sum();
  };
  auto dprob = [&](int hh) {
    Dot<T> s;
#pragma unroll
    for (int c = 0; c < DVP / 16; ++c) s.add(VTile::rows(vt, 32 * hh, c, lane), gf[c]);
    return s.sum();
  };
  auto seen = [&](int t, u64 bits) { return a.causal ? bits & upto(q + off - (long long)t * TILE) : bits; };
  auto begin = [&](int& t, u64& bits) {
    keys.start(first, wave, lane);
    t = keys.next(first, bits, wave, lane);
    if (t < keys.end) {
      ks.load(kp + (long long)t * TILE * a.kn, bits, tid);
      vs.load(vp + (long long)t * TILE * a.vn, bits, tid);
    }
  };
  auto advance = [&](int t, u64& bits_next) {       // this tile into LDS, the next one's loads under way
    __syncthreads();
    ks.put(kt, tid);
    vs.put(vt, tid);
    __syncthreads();
    const int tn = keys.next(t + 1, bits_next, wave, lane);
    if (tn < keys.end) {
      ks.load(kp + (long long)tn * TILE * a.kn, bits_next, tid);
      vs.load(vp + (long long)tn * TILE * a.vn, bits_next, tid);
    }
    return tn;
  };

  float delta[2] = {0.f, 0.f}, top = 0.f;
  u64 bits, bits_next;
  int t;
  if constexpr (PHASE != 2) {
    begin(t, bits);
    while (t < keys.end) {
      const int tn = advance(t, bits_next);
      if (!a.causal || (long long)t * TILE <= wave_last) {
        const u64 see = seen(t, bits);
        const bool part = __any(see != ~0ull);
#pragma unroll
        for (int half = 0; half < 2 / KW; ++half) {
          const int hh = KW == 1 ? half : kw;
          const f32x16 dp = dprob(hh);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            f32x16 s = score(i, hh);
            if (part) hide(s, see, hh, g);
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) sum = fmaf(__builtin_amdgcn_exp2f(fmaf(s[r], a.c, -mc[i])), dp[r], sum);
            delta[i] = fmaf(sum, side * il[i], delta[i]);                  // dlambda is held to 32 bits: 1 / sum as a factor, not in the exponent
          }
          if (__is_same(T, _Float16)) {
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(dp[r]));
          }
        }
      }
      t = tn;
      bits = bits_next;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) delta[i] += __shfl_xor(delta[i], 32);
    top = fmaxf(top, __shfl_xor(top, 32));
    if constexpr (KW == 2) {
      float* box = reinterpret_cast<float*>(lds);
      __syncthreads();
      if (g == 0) { box[(wave * 3) * 32 + l31] = delta[0]; box[(wave * 3 + 1) * 32 + l31] = delta[1]; box[(wave * 3 + 2) * 32 + l31] = top; }
      __syncthreads();
      const int w0 = wave & ~1;
      delta[0] = box[(w0 * 3) * 32 + l31] + box[(w0 * 3 + 3) * 32 + l31];
      delta[1] = box[(w0 * 3 + 1) * 32 + l31] + box[(w0 * 3 + 4) * 32 + l31];
      top = fmaxf(box[(w0 * 3 + 2) * 32 + l31], box[(w0 * 3 + 5) * 32 + l31]);
    }
    if (il[0] == 0.f && il[1] == 0.f) delta[0] = delta[1] = top = 0.f;
    if (q_on && kw == 0 && g == 0) {
      float* dst = (PHASE == 1 ? a.part + (long long)split * a.B * a.H * 3 * a.N : a.delta) + (long long)bh * 3 * a.N + q;
      dst[0] = delta[0];
      dst[a.N] = delta[1];
      dst[2ll * a.N] = top;
    }
    if constexpr (PHASE == 1) return;
  } else if (q_on) {
    const float* src = a.delta + (long long)bh * 3 * a.N + q;
    delta[0] = src[0];
    delta[1] = src[a.N];
    top = src[2ll * a.N];
  }
  const float lam = a.lambda[h];
  float up = 1.f;                                   // |dS| <= 2 max(1, |lambda|) max |dP|
  if (__is_same(T, _Float16)) up = pow2_below(16384.f, 2.f * fmaxf(1.f, fabsf(lam)) * top);
  const Prob<T> prob[2] = {Prob<T>(mc[0], il[0], 1.f), Prob<T>(mc[1], il[1], 1.f)};
  const float wd[2] = {-up * delta[0], up * lam * delta[1]}, w[2] = {side * up, -side * up * lam};

  f32x16 o[2][ND];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < ND; ++j) o[i][j] = zero16();
  __syncthreads();
  begin(t, bits);
  while (t < keys.end) {
    const int tn = advance(t, bits_next);
    if (!a.causal || (long long)t * TILE <= wave_last) {
      const u64 see = seen(t, bits);
      const bool part = __any(see != ~0ull);
#pragma unroll
      for (int half = 0; half < 2 / KW; ++half) {
        const int hh = KW == 1 ? half : kw;
        const f32x16 dp = dprob(hh);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          f32x16 s = score(i, hh);
          if (part) hide(s, see, hh, g);
          float ds[16];
#pragma unroll
          for (int r = 0; r < 16; ++r) ds[r] = prob[i](s[r], a.c) * fmaf(dp[r], w[i], wd[i]);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const Frag<P> df = pack8<T>(ds + 8 * u), rest = TWO_TERMS<T> ? rest8<T>(ds + 8 * u, df) : df;
#pragma unroll
            for (int j = 0; j < ND; ++j) {
              const Frag<P> kc = KTile::cols(kt, 32 * hh + 16 * u, i * DP + 32 * j, lane, (i + 1) * DP);
              if (TWO_TERMS<T>) accumulate<T>(o[i][j], kc, rest);
              accumulate<T>(o[i][j], kc, df);
            }
          }
        }
      }
    }
    t = tn;
    bits = bits_next;
  }
  if constexpr (KW == 2) {
    float* box = reinterpret_cast<float*>(lds) + (size_t)qw * 2 * ND * 16 * 64;
    __syncthreads();
    if (kw == 1) {
#pragma unroll
      for (int i = 0; i < 2 * ND; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) box[(i * 16 + r) * 64 + lane] = o[i / ND][i % ND][r];
    }
    __syncthreads();
    if (kw == 1) return;
#pragma unroll
    for (int i = 0; i < 2 * ND; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[i / ND][i % ND][r] += box[(i * 16 + r) * 64 + lane];
  }
  if (!q_on) return;
  const float f = a.scale / up;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const long long row = ((long long)b * a.N + q) * 2 * a.H + 2 * h + i;
    T* dst = static_cast<T*>(a.dq) + row * a.d;
    float* part = PHASE == 2 ? a.part + ((long long)split * a.B * a.N * 2 * a.H + row) * a.d : nullptr;
#pragma unroll
    for (int j = 0; j < ND; ++j)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int col = 32 * j + 2 * r + 4 * g;
        if (col >= a.d) continue;
        f32x4 v = {o[i][j][r] * f, o[i][j][r + 1] * f, o[i][j][r + 2] * f, o[i][j][r + 3] * f};
        if (prob[0].never() && prob[1].never()) v = f32x4{0.f, 0.f, 0.f, 0.f};
        if constexpr (PHASE == 2) *reinterpret_cast<f32x4*>(part + col) = v;
        else store4<T>(dst + col, v[0], v[1], v[2], v[3]);
      }
  }
}

// the splits' deltas, in order
static __global__ __launch_bounds__(256) void delta_join(Args a, long long rows) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows) return;
  const long long bh = i / a.N, at = bh * 3 * a.N + (i - bh * a.N), step = rows * 3;
  float d1 = 0.f, d2 = 0.f, top = 0.f;
  for (int s = 0; s < a.dq_splits; ++s) {
    const float* p = a.part + s * step + at;
    d1 += p[0];
    d2 += p[a.N];
    top = fmaxf(top, p[2ll * a.N]);
  }
  a.delta[at] = d1;
  a.delta[at + a.N] = d2;
  a.delta[at + 2ll * a.N] = top;
}

// the splits' dQ of four neighbouring columns, in order
template <class T>
__global__ __launch_bounds__(256) void dq_join(Args a, long long quads) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= quads) return;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.dq_splits; ++s) v += *reinterpret_cast<const f32x4*>(a.part + (s * quads + i) * 4);
  store4<T>(static_cast<T*>(a.dq) + i * 4, v[0], v[1], v[2], v[3]);
}

template <class T, int DP, int DVP>
struct DkvShape {
  static constexpr int P = Type<T>::planes, ND = (DP + 31) / 32, NV = DVP / 32;
  // d > 32: the sums and operands of both gradients are more than half the registers of a SIMD, and one wave alone waits for each of its
  // products; dK and dV then have a kernel each (the maps are formed twice), and their tiles are 32 queries, which halves what is under way
  static constexpr bool APART = DP > 32;
  static constexpr int MIN_BLOCKS = P == 1 ? 2 : 1, TQ = APART ? 32 : 64;
  typedef Tile<2 * DP, P, TQ> QTile;
  typedef Tile<DVP, P, TQ> GTile;
  static constexpr int ROWS = QTile::BYTES + GTile::BYTES;          // offset of the rows' statistics [6][TQ]
  static constexpr int KEYS = ROWS + 6 * TQ * 4;                    // offset of v, where it is kept in LDS
  typedef Tile<DVP, P, 128> VTile;
  // dK at d > 32 in 16 bits: with v in registers too a few of them would go to memory, and every such access waits for the next tile's loads
  static constexpr bool V_LDS = APART && P == 1;
  static constexpr int lds(int what) { return KEYS + (V_LDS && what == 1 ? VTile::BYTES : 0); }
};
constexpr int BK = 128;                                             // keys of a workgroup: 32 per wave

// Over keys: a wave keeps 32 of them (k1, k2 and v as operands, dK1, dK2 and dV as sums) and the queries of all heads that share the key
// head stream by.  With few keys the queries are split over `splits` workgroups, whose sums go to `part` [splits][B M Hkv][2 d + dv]
// in 32 bits and are added in order by dkv_join.  WHAT: 1 dK, 2 dV, 3 both.
template <class T, int DP, int DVP, int WHAT>
__global__ __launch_bounds__(THREADS, (DkvShape<T, DP, DVP>::MIN_BLOCKS)) void dkv_kernel(Args a) {
  constexpr bool DK = WHAT & 1, DV = WHAT & 2;
  typedef DkvShape<T, DP, DVP> S;
  typedef typename S::QTile QTile;
  typedef typename S::GTile GTile;
  constexpr int P = S::P, TQ = S::TQ, ND = S::ND, NV = S::NV;
  extern __shared__ __align__(256) char lds[];
  char* qt = lds;
  char* gt = lds + QTile::BYTES;
  float* rowst = reinterpret_cast<float*>(lds + S::ROWS);          // of the tile's queries: m and il of both maps (Prob), - w_i delta_i
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 5, l31 = lane & 31;
  const int k_tiles = (a.M + BK - 1) / BK, group = a.H / a.Hkv, heads = a.B * a.Hkv;
  int bk, kt, split;
  if (a.causal) {                                                   // long ones first, over all dies
    split = blockIdx.x % a.splits;
    const int rest = blockIdx.x / a.splits;
    kt = rest / heads;
    bk = rest - kt * heads;
  } else {
    const unsigned id = die_major(blockIdx.x, gridDim.x);
    split = id % a.splits;
    const int rest = id / a.splits;
    bk = rest / k_tiles;
    kt = rest - bk * k_tiles;
  }
  const int b = bk / a.Hkv, hk = bk - b * a.Hkv;
  const int key = kt * BK + 32 * wave + l31;
  const bool k_in = key < a.M, k_on = k_in && (a.mask == nullptr || a.mask[b * a.mb + key] != 0);
  const long long off = (long long)a.M - a.N;                      // causal: key j is seen by the queries >= j - off
  constexpr bool V_LDS = S::V_LDS && WHAT == 1;
  char* vt = lds + S::KEYS;
  Frag<P> kf[2][DP / 16], vf[V_LDS ? 1 : DVP / 16];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    load_rows<T, DP>(kf[i], static_cast<const T*>(a.k) + b * a.kb + (long long)key * a.kn + (2ll * hk + i) * a.kh, k_on, a.d, g);
  const T* v_row = static_cast<const T*>(a.v) + b * a.vb + (long long)key * a.vn + (long long)hk * a.vh;
  if constexpr (V_LDS) {                                           // a wave reads its own rows only
#pragma unroll
    for (int c = 0; c < DVP / 16; ++c) {
      Raw<T> r;
      const int col = 16 * c + 8 * g;
      if (k_on && col < a.dv_w) r.load(v_row + col);
      else r.clear();
      S::VTile::put(vt, 32 * wave + l31, 2 * c + g, r.frag());
    }
  } else if constexpr (DK) {
    load_rows<T, DVP>(vf, v_row, k_on, a.dv_w, g);
  }

  f32x16 dk[2][ND], dv[NV];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < ND; ++j) dk[i][j] = zero16();
#pragma unroll
  for (int j = 0; j < NV; ++j) dv[j] = zero16();

  float up_a = 1.f, up_s = 1.f;                                    // fp16: one scale for all heads that are summed here
  if constexpr (__is_same(T, _Float16)) {
    float lam = 1.f, top = 0.f;
    for (int i = 0; i < group; ++i) lam = fmaxf(lam, fabsf(a.lambda[hk * group + i]));
    for (int i = 0; i < group; ++i) {
      const float* d = a.delta + ((long long)(b * a.H + hk * group + i) * 3 + 2) * a.N;
      for (int n = tid; n < a.N; n += THREADS) top = fmaxf(top, d[n]);
    }
    for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
    if (lane == 0) rowst[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(rowst[0], rowst[1]), fmaxf(rowst[2], rowst[3]));
    up_a = pow2_below(16384.f, lam);
    up_s = pow2_below(16384.f, 2.f * lam * top);
  }

  const int n_tiles = (a.N + TQ - 1) / TQ;
  int t_first = 0;
  if (a.causal) {
    const long long q_first = (long long)kt * BK - off;
    if (q_first > 0) t_first = q_first / TQ < n_tiles ? (int)(q_first / TQ) : n_tiles;
  }
  // the first of the workgroup's keys that the mask leaves; a workgroup that has none has nothing to sum
  int* firsts = reinterpret_cast<int*>(rowst + 4);
  const u64 on_keys = __ballot(k_on);
  if (lane == 0) firsts[wave] = on_keys != 0 ? kt * BK + 32 * wave + __builtin_ctzll(on_keys) : a.M;
  __syncthreads();
  const int first_key = min(min(firsts[0], firsts[1]), min(firsts[2], firsts[3]));
  const bool any = first_key < a.M;
  Stage<T, 2 * DP, 2, TQ> qs;
  Stage<T, DVP, 1, TQ> gs;
  qs.init(a.qn, a.qh, a.d, tid);
  gs.init(a.gn, 0, a.dv_w, tid);
  float2 rs;
  float rlam;
  auto load = [&](int hg, int t) {
    const int h = hk * group + hg;
    const long long left = (long long)a.N - (long long)t * TQ;
    u64 bits = left >= TQ ? ~0ull : (1ull << left) - 1;
    const long long from = a.causal ? first_key - off - (long long)t * TQ : 0;   // queries before it see none of the keys (and may see none at all):
    if (from > 0) bits &= from < 64 ? ~0ull << from : 0ull;                      // whatever they and their dO hold, they are zeros here
    const long long bh = (long long)b * a.H + h;
    const int n = t * TQ + lane % TQ;                                  // waves 0, 1: statistics of map 0, 1; wave 2: both deltas
    rlam = a.lambda[h];
    rs = wave < 2 ? make_float2(INFINITY, 0.f) : make_float2(0.f, 0.f);
    if (n < a.N && lane % TQ >= from) {
      if (wave < 2) rs = a.stats[(bh * 2 + wave) * a.N + n];
      else if (wave == 2) rs = make_float2(a.delta[bh * 3 * a.N + n], a.delta[(bh * 3 + 1) * a.N + n]);
    }
    qs.load(static_cast<const T*>(a.q) + b * a.qb + 2ll * h * a.qh + (long long)t * TQ * a.qn, bits, tid);
    gs.load(static_cast<const T*>(a.dout) + b * a.gb + (long long)h * a.gh + (long long)t * TQ * a.gn, bits, tid);
  };
  const long long per_head = n_tiles - t_first, steps = per_head * group;
  long long step = steps * split / a.splits;
  const long long last_step = any ? steps * (split + 1) / a.splits : step;
  int hg = per_head > 0 ? (int)(step / per_head) : 0, t = t_first + (int)(step - hg * per_head);
  if (step < last_step) load(hg, t);
  for (; step < last_step; ++step) {
    __syncthreads();
    qs.put(qt, tid);
    gs.put(gt, tid);
    const float lam = rlam, w1 = up_s, w2 = -lam * up_s;
    if (wave < 2) {
      const Prob<T> pr(rs.x, rs.y, 1.f);
      rowst[2 * wave * TQ + lane % TQ] = pr.m;
      if (!Prob<T>::folded) rowst[(2 * wave + 1) * TQ + lane % TQ] = pr.f;
    } else if (wave == 2) {
      rowst[4 * TQ + lane % TQ] = -w1 * rs.x;
      rowst[5 * TQ + lane % TQ] = -w2 * rs.y;
    }
    __syncthreads();
    int t_next = t + 1, hg_next = hg;
    if (t_next == n_tiles) { t_next = t_first; ++hg_next; }
    if (step + 1 < last_step) load(hg_next, t_next);
#pragma unroll
    for (int hh = 0; hh < TQ / 32; ++hh) {
      const long long last_q = (long long)t * TQ + 32 * hh + 31;
      if (a.causal && last_q + off < (long long)kt * BK + 32 * wave) continue;   // no query of these sees a key of the wave
      auto score = [&](int i) {
        Dot<T> s;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) s.add(QTile::rows(qt, 32 * hh, i * (DP / 16) + c, lane), kf[i][c]);
        return s.sum();
      };
      f32x16 dp;
      if (DK) {
        Dot<T> dot;
#pragma unroll
        for (int c = 0; c < DVP / 16; ++c) dot.add(GTile::rows(gt, 32 * hh, c, lane), V_LDS ? S::VTile::rows(vt, 32 * wave, c, lane) : vf[V_LDS ? 0 : c]);
        dp = dot.sum();
      }
      const bool cut = a.causal && (long long)t * TQ + 32 * hh + off < (long long)kt * BK + 32 * wave + 31;   // some query does not see some key
      const long long from = cut ? key - off - (long long)t * TQ - 32 * hh : 0;                          // the first that sees the lane's
      const int first = from < 0 ? 0 : from > 32 ? 32 : (int)from;
      Frag<P> fa[2], fs[2][2], rest_a[2], rest_s[2][2];
      float p[16];                                                  // P1, then A
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f32x16 s = score(i);
        if (cut) {
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = 8 * (r >> 2) + 4 * g + (r & 3) >= first ? s[r] : -INFINITY;
        }
        float ds[16];
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int row = 32 * hh + 8 * r4 + 4 * g;
          const f32x4 m = *reinterpret_cast<const f32x4*>(rowst + 2 * i * TQ + row), e = *reinterpret_cast<const f32x4*>(rowst + (4 + i) * TQ + row);
          f32x4 il = {1.f, 1.f, 1.f, 1.f};
          if (!Prob<T>::folded) il = *reinterpret_cast<const f32x4*>(rowst + (2 * i + 1) * TQ + row);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int r = 4 * r4 + x;
            float q = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -m[x]));
            if (!Prob<T>::folded) q *= il[x];
            if (DK) ds[r] = q * fmaf(dp[r], i == 0 ? w1 : w2, e[x]);
            p[r] = i == 0 ? q : fmaf(-lam, q, p[r]) * up_a;
          }
        }
        if (DK) {
          fs[i][0] = pack8<T>(ds);
          fs[i][1] = pack8<T>(ds + 8);
          if (TWO_TERMS<T>) { rest_s[i][0] = rest8<T>(ds, fs[i][0]); rest_s[i][1] = rest8<T>(ds + 8, fs[i][1]); }
        }
      }
      if (DV) {
        fa[0] = pack8<T>(p);
        fa[1] = pack8<T>(p + 8);
        if (TWO_TERMS<T>) { rest_a[0] = rest8<T>(p, fa[0]); rest_a[1] = rest8<T>(p + 8, fa[1]); }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int row0 = 32 * hh + 16 * u;
        if (DV) {
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            const Frag<P> gc = GTile::cols(gt, row0, 32 * j, lane, DVP);
            if (TWO_TERMS<T>) accumulate<T>(dv[j], gc, rest_a[u]);
            accumulate<T>(dv[j], gc, fa[u]);
          }
        }
        if (DK) {
#pragma unroll
          for (int j = 0; j < ND; ++j) {
            const Frag<P> q1 = QTile::cols(qt, row0, 32 * j, lane, DP), q2 = QTile::cols(qt, row0, DP + 32 * j, lane, 2 * DP);
            if (TWO_TERMS<T>) {
              accumulate<T>(dk[0][j], q1, rest_s[0][u]);
              accumulate<T>(dk[1][j], q2, rest_s[1][u]);
            }
            accumulate<T>(dk[0][j], q1, fs[0][u]);
            accumulate<T>(dk[1][j], q2, fs[1][u]);
          }
        }
      }
    }
    t = t_next;
    hg = hg_next;
  }
  if (!k_in) return;
  const float fv = k_on ? 1.f / up_a : 0.f, fk = k_on ? a.scale / up_s : 0.f;
  auto out = [&](float x, float f) { return k_on ? x * f : 0.f; };   // a hidden key's sums may hold anything
  const long long row = ((long long)b * a.M + key) * a.Hkv + hk;
  float* part = a.splits > 1 ? a.part + ((long long)split * a.B * a.M * a.Hkv + row) * (2 * a.d + a.dv_w) : nullptr;
  auto put = [&](T* dst, float* to, const f32x16& v, int r, float f) {
    if (part != nullptr) *reinterpret_cast<f32x4*>(to) = f32x4{out(v[r], f), out(v[r + 1], f), out(v[r + 2], f), out(v[r + 3], f)};
    else store4<T>(dst, out(v[r], f), out(v[r + 1], f), out(v[r + 2], f), out(v[r + 3], f));
  };
  if (DV) {
    T* dst = static_cast<T*>(a.dv) + row * a.dv_w;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int col = 32 * j + 2 * r + 4 * g;
        if (col < a.dv_w) put(dst + col, part + 2 * a.d + col, dv[j], r, fv);
      }
  }
  if (DK) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      T* dst = static_cast<T*>(a.dk) + (row * 2 + i) * a.d;
#pragma unroll
      for (int j = 0; j < ND; ++j)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const int col = 32 * j + 2 * r + 4 * g;
          if (col < a.d) put(dst + col, part + i * a.d + col, dk[i][j], r, fk);
        }
    }
  }
}

// the splits' sums of four neighbouring columns, in order
template <class T>
__global__ __launch_bounds__(256) void dkv_join(Args a, long long quads) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= quads) return;
  const int width = 2 * a.d + a.dv_w;
  const long long row = i / (width / 4);
  const int col = (int)(i - row * (width / 4)) * 4;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.splits; ++s) v += *reinterpret_cast<const f32x4*>(a.part + s * quads * 4 + i * 4);
  T* dst = col < 2 * a.d ? static_cast<T*>(a.dk) + row * 2 * a.d + col : static_cast<T*>(a.dv) + row * a.dv_w + (col - 2 * a.d);
  store4<T>(dst, v[0], v[1], v[2], v[3]);
}

template <class T, int DP, int DVP, int KW, int PHASE>
int launch_dq(const Args& a, hipStream_t st) {
  typedef DqShape<T, DP, DVP> S;
  const long long blocks = (long long)a.B * a.H * ((a.N + 128 / KW - 1) / (128 / KW)) * (PHASE == 0 ? 1 : a.dq_splits);
  if (blocks > MAX_BLOCKS) return -3;
  static LdsAttrOnce once;
  if (set_max_dynamic_lds(once, reinterpret_cast<const void*>(&dq_kernel<T, DP, DVP, KW, PHASE>), S::LDS)) return -2;
  if (blocks > 0) hipLaunchKernelGGL((dq_kernel<T, DP, DVP, KW, PHASE>), dim3((unsigned)blocks), dim3(THREADS), S::LDS, st, a);
  return 0;
}

template <class T, int DP, int DVP>
int launch_dq_split(const Args& a, hipStream_t st) {
  const long long rows = (long long)a.B * a.H * a.N, quads = rows * 2 * a.d / 4;
  if (rows == 0) return 0;
  if ((quads + 255) / 256 > MAX_BLOCKS) return -3;
  if (const int rc = launch_dq<T, DP, DVP, 2, 1>(a, st)) return rc;
  hipLaunchKernelGGL(delta_join, dim3((unsigned)((rows + 255) / 256)), dim3(256), 0, st, a, rows);
  if (const int rc = launch_dq<T, DP, DVP, 2, 2>(a, st)) return rc;
  hipLaunchKernelGGL((dq_join<T>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, st, a, quads);
  return 0;
}

template <class T, int DP, int DVP, int WHAT>
int launch_dkv(const Args& a, hipStream_t st) {
  typedef DkvShape<T, DP, DVP> S;
  const long long blocks = (long long)a.B * a.Hkv * ((a.M + BK - 1) / BK) * a.splits;
  if (blocks > MAX_BLOCKS) return -3;
  static LdsAttrOnce once;
  if (set_max_dynamic_lds(once, reinterpret_cast<const void*>(&dkv_kernel<T, DP, DVP, WHAT>), S::lds(WHAT))) return -2;
  if (blocks > 0) hipLaunchKernelGGL((dkv_kernel<T, DP, DVP, WHAT>), dim3((unsigned)blocks), dim3(THREADS), S::lds(WHAT), st, a);
  return 0;
}

template <class T, int DP, int DVP>
int launch_bwd(const Args& a, hipStream_t st) {
  // In 32 bits above d = 32 a wave with all of a tile's keys keeps many registers in memory: two share them at every size (2048 workgroups of 128
  // queries, training pass: d = 64, dv = 128 21.0 -> 15.3 ms, d = 48, dv = 96 13.0 -> 11.1; d = 32 would lose, 5.6 -> 6.2).  At d = 64, dv = 128 they
  // still keep 39 there.
  constexpr bool SHARED = Type<T>::planes == 3 && DP > 32;
  int rc;
  if (a.dq_splits > 1) rc = launch_dq_split<T, DP, DVP>(a, st);
  else if (SHARED || few_queries(a)) rc = launch_dq<T, DP, DVP, 2, 0>(a, st);
  else rc = launch_dq<T, DP, DVP, SHARED ? 2 : 1, 0>(a, st);
  if (rc) return rc;
  if constexpr (DkvShape<T, DP, DVP>::APART) {
    if (const int rc1 = launch_dkv<T, DP, DVP, 1>(a, st)) return rc1;
    if (const int rc2 = launch_dkv<T, DP, DVP, 2>(a, st)) return rc2;
  } else {
    if (const int rc3 = launch_dkv<T, DP, DVP, 3>(a, st)) return rc3;
  }
  const long long quads = (long long)a.B * a.M * a.Hkv * (2 * a.d + a.dv_w) / 4;
  if (a.splits > 1 && quads > 0) {
    if ((quads + 255) / 256 > MAX_BLOCKS) return -3;
    hipLaunchKernelGGL((dkv_join<T>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, st, a, quads);
  }
  return 0;
}

template <class T>
int run_backward(const Args& a, hipStream_t st) {
#define SCGG_X(DP, DVP) if (a.d <= DP && a.dv_w <= DVP) return launch_bwd<T, DP, DVP>(a, st);
  SCGG_DIFF_WIDTHS(SCGG_X)
#undef SCGG_X
  return -1;
}

}  // namespace diffattn
}  // namespace scgg
