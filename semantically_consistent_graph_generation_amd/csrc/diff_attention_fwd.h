// Differential attention, forward kernels.  Included by the translation unit of each element type.
#pragma once
#include "diff_attention.h"

namespace scgg {
namespace diffattn {

// fp16 holds values below 2^-14 with fewer bits: A and dS are multiplied by a power of two that brings their bound near 2^14
__device__ __forceinline__ float pow2_below(float limit, float bound) {   // the largest 2^e with bound 2^e <= limit; 1 if there is none
  if (!(bound > 0.f) || !(bound < INFINITY)) return 1.f;
  int e;
  frexpf(limit / bound, &e);                                              // limit / bound = m 2^e, m in [0.5, 1)
  return ldexpf(1.f, e - 1 < -100 ? -100 : e - 1 > 100 ? 100 : e - 1);
}

// Running softmax statistics of one map over 16 more scores of a lane: m = c times the largest score, rounded, l = sum of
// 2^(c s - m).  m is kept as it was rounded: a maximum that does not change then leaves the sum as it is, bit for bit.
__device__ __forceinline__ float row_max(const f32x16& s) {
  float t = fmaxf(fmaxf(s[0], s[1]), s[2]);
#pragma unroll
  for (int r = 3; r < 15; r += 2) t = fmaxf(fmaxf(t, s[r]), s[r + 1]);
  return fmaxf(t, s[15]);
}

__device__ __forceinline__ void add_stats(const f32x16& s, float c, float& m, float& l) {
  const float t = fmaxf(row_max(s) * c, m), base = t == -INFINITY ? 0.f : t;
  float a = 0.f, b = 0.f;           // on their own first: the long sum is rounded once for 16 terms
#pragma unroll
  for (int r = 0; r < 16; r += 2) {
    a += __builtin_amdgcn_exp2f(fmaf(s[r], c, -base));
    b += __builtin_amdgcn_exp2f(fmaf(s[r + 1], c, -base));
  }
  l = fmaf(l, __builtin_amdgcn_exp2f(m - base), a + b);
  m = t;
}

__device__ __forceinline__ void merge_stats(float& m, float& l, float m2, float l2) {
  const float t = fmaxf(m, m2), base = t == -INFINITY ? 0.f : t;
  l = l * __builtin_amdgcn_exp2f(m - base) + l2 * __builtin_amdgcn_exp2f(m2 - base);
  m = t;
}

// Two sweeps over the keys.  The first finds the maximum and the sum of both maps; the second forms A = P1 - lambda P2 in 32 bits, rounds
// it (16 bits: in two terms), and needs one product with v.  With dv = 2 d this is as many products as one sweep with an accumulator per map
// (2 d + 2 d + dv against 2 d + 2 dv per pair of tokens) and half the accumulators, and A, not P1 and P2, is rounded: where the maps
// cancel, rounding them apart would leave an error of the size of what was cancelled.
// A workgroup has 4 waves: 4 / KW groups of 32 queries, and KW waves that share a tile's keys.
// Bound: neither unit alone.  32 heads of 4096 x 4096, d = 64, dv = 128, bf16, 622 us: vector instructions issue in 59 % of the cycles, the matrix unit is
// busy in 40 %, no LDS bank conflicts (counters); a SIMD has two waves, which meet at two barriers a tile.  2 x 8192 queries and keys, ragged, 8 heads,
// bf16: 1.27 ms, 424 TFLOP/s of 4 d + 2 dv per pair (a large library matrix product: 1118), the second term's products not counted.
template <class T, int DP, int DVP>
struct FwdShape {
  static constexpr int P = Type<T>::planes;
  typedef Tile<2 * DP, P> KTile;
  typedef Tile<DVP, P> VTile;
  static constexpr int MERGE = 2 * DVP * 128;                 // two waves' 32 x DVP sums
  static constexpr int TILES = KTile::BYTES + VTile::BYTES;
  static constexpr int WORDS = TILES > MERGE ? TILES : MERGE; // offset of the mask words
  static constexpr int LDS = WORDS + WINDOW * 8;
  static constexpr int MIN_BLOCKS = P == 3 && DP > 32 ? 1 : 2;
};

template <class T, int DP, int DVP, int KW>
__global__ __launch_bounds__(THREADS, (FwdShape<T, DP, DVP>::MIN_BLOCKS)) void fwd_kernel(Args a) {
  typedef FwdShape<T, DP, DVP> S;
  typedef typename S::KTile KTile;
  typedef typename S::VTile VTile;
  constexpr int P = S::P, QW = 4 / KW, BQ = 32 * QW, NV = DVP / 32;
  extern __shared__ __align__(256) char lds[];
  char* kt = lds;
  char* vt = lds + KTile::BYTES;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 5, l31 = lane & 31;
  const int qw = wave / KW, kw = wave - qw * KW;
  const int q_tiles = (a.N + BQ - 1) / BQ;
  const unsigned id = die_major(blockIdx.x, gridDim.x);
  const int bh = id / q_tiles, qt = a.causal ? q_tiles - 1 - (int)(id - bh * q_tiles) : (int)(id - bh * q_tiles);   // causal: long ones first
  const int b = bh / a.H, h = bh - b * a.H, hk = h / (a.H / a.Hkv);
  const int q = qt * BQ + 32 * qw + l31;
  bool q_on = q < a.N;                                         // the lane's query is to be written
  const long long off = (long long)a.M - a.N;                  // causal: query q sees the keys <= q + off
  const T* kp = static_cast<const T*>(a.k) + b * a.kb + 2ll * hk * a.kh;
  const T* vp = static_cast<const T*>(a.v) + b * a.vb + (long long)hk * a.vh;

  Frag<P> qf[2][DP / 16];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    load_rows<T, DP>(qf[i], static_cast<const T*>(a.q) + b * a.qb + (long long)q * a.qn + (2ll * h + i) * a.qh, q_on, a.d, g);

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
  const long long wave_last = (long long)qt * BQ + 32 * qw + 31 + off;   // causal: last key that any query of the wave may see

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
  auto seen = [&](int t, u64 bits) { return a.causal ? bits & upto(q + off - (long long)t * TILE) : bits; };

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  u64 bits, bits_next;
  keys.start(0, wave, lane);
  int t = keys.next(0, bits, wave, lane);
  if (t < keys.end) ks.load(kp + (long long)t * TILE * a.kn, bits, tid);
  while (t < keys.end) {
    __syncthreads();
    ks.put(kt, tid);
    __syncthreads();
    const int tn = keys.next(t + 1, bits_next, wave, lane);
    if (tn < keys.end) ks.load(kp + (long long)tn * TILE * a.kn, bits_next, tid);
    if (!a.causal || (long long)t * TILE <= wave_last) {
      const u64 see = seen(t, bits);
      const bool part = __any(see != ~0ull);
      f32x16 s[2 / KW][2];
#pragma unroll
      for (int half = 0; half < 2 / KW; ++half)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          s[half][i] = score(i, KW == 1 ? half : kw);
          if (part) hide(s[half][i], see, KW == 1 ? half : kw, g);
        }
      // m need not be the largest score, only near enough that the sums stay in range: a tile whose sums are below 2^80 is added as it is
      bool rescale = __any(m[0] == -INFINITY || m[1] == -INFINITY);
      if (!rescale) {
        float sum[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float x = 0.f, y = 0.f;
#pragma unroll
          for (int half = 0; half < 2 / KW; ++half)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
              x += __builtin_amdgcn_exp2f(fmaf(s[half][i][r], a.c, -m[i]));
              y += __builtin_amdgcn_exp2f(fmaf(s[half][i][r + 1], a.c, -m[i]));
            }
          sum[i] = x + y;
        }
        rescale = __any(!(fmaxf(sum[0], sum[1]) <= 0x1p80f));
        if (!rescale) {
          l[0] += sum[0];
          l[1] += sum[1];
        }
      }
      if (rescale) {
#pragma unroll
        for (int half = 0; half < 2 / KW; ++half)
#pragma unroll
          for (int i = 0; i < 2; ++i) add_stats(s[half][i], a.c, m[i], l[i]);
      }
    }
    t = tn;
    bits = bits_next;
  }
  float mc[2], il[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) merge_stats(m[i], l[i], __shfl_xor(m[i], 32), __shfl_xor(l[i], 32));
  if constexpr (KW == 2) {
    float* box = reinterpret_cast<float*>(lds);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (g == 0) { box[(wave * 4 + 2 * i) * 32 + l31] = m[i]; box[(wave * 4 + 2 * i + 1) * 32 + l31] = l[i]; }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int w0 = wave & ~1;
      float m0 = box[(w0 * 4 + 2 * i) * 32 + l31], l0 = box[(w0 * 4 + 2 * i + 1) * 32 + l31];
      merge_stats(m0, l0, box[((w0 + 1) * 4 + 2 * i) * 32 + l31], box[((w0 + 1) * 4 + 2 * i + 1) * 32 + l31]);
      m[i] = m0;
      l[i] = l0;
    }
  }
  // a base far below the maximum (the sum is then that large) moves up to it: the backward multiplies 2^(c s - m) by dP before it takes 1 / sum, and
  // |dP| of 2^48 and more would overflow with the 2^80 that the sweep allows
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (l[i] > 0x1p32f) {
      int e;
      l[i] = frexpf(l[i], &e);
      const float t = m[i] + (float)e;
      l[i] *= __builtin_amdgcn_exp2f((m[i] - t) + (float)e);   // what the rounding of t left
      m[i] = t;
    }
#pragma unroll
  for (int i = 0; i < 2; ++i) {   // a query that sees nothing: every 2^(c s - mc) is 0
    mc[i] = l[i] == 0.f ? INFINITY : m[i];
    il[i] = l[i] == 0.f ? 0.f : 1.f / l[i];
    if (a.stats != nullptr && q_on && kw == 0 && g == 0)
      a.stats[((long long)(b * a.H + h) * 2 + i) * a.N + q] = make_float2(mc[i], il[i]);
  }
  if (q_on && il[0] == 0.f && il[1] == 0.f) {                  // sees nothing: zeros, whatever the tiles hold for others
    if (kw == 0 && g == 0)
      for (int col = 0; col < a.dv_w; col += 4) store4<T>(static_cast<T*>(a.out) + (((long long)b * a.N + q) * a.H + h) * a.dv_w + col, 0.f, 0.f, 0.f, 0.f);
    q_on = false;
  }
  const float lam = a.lambda[h];
  float up = 1.f;
  if constexpr (sizeof(T) == 2 && Type<T>::planes == 1) {
    if (__is_same(T, _Float16)) up = pow2_below(16384.f, fmaxf(1.f, fabsf(lam)));
  }
  const Prob<T> p1(mc[0], il[0], up), p2(mc[1], il[1], up);

  f32x16 o[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) o[i] = zero16();
  __syncthreads();
  keys.start(0, wave, lane);
  t = keys.next(0, bits, wave, lane);
  if (t < keys.end) {
    ks.load(kp + (long long)t * TILE * a.kn, bits, tid);
    vs.load(vp + (long long)t * TILE * a.vn, bits, tid);
  }
  while (t < keys.end) {
    __syncthreads();
    ks.put(kt, tid);
    vs.put(vt, tid);
    __syncthreads();
    const int tn = keys.next(t + 1, bits_next, wave, lane);
    if (tn < keys.end) {
      ks.load(kp + (long long)tn * TILE * a.kn, bits_next, tid);
      vs.load(vp + (long long)tn * TILE * a.vn, bits_next, tid);
    }
    if (!a.causal || (long long)t * TILE <= wave_last) {
      const u64 see = seen(t, bits);
      const bool part = __any(see != ~0ull);
#pragma unroll
      for (int half = 0; half < 2 / KW; ++half) {
        const int hh = KW == 1 ? half : kw;
        f32x16 s1 = score(0, hh), s2 = score(1, hh);
        if (part) { hide(s1, see, hh, g); hide(s2, see, hh, g); }
        float p[16];
#pragma unroll
        for (int r = 0; r < 16; ++r)
          p[r] = fmaf(-lam, p2(s2[r], a.c), p1(s1[r], a.c));
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const Frag<P> pf = pack8<T>(p + 8 * u), rest = TWO_TERMS<T> ? rest8<T>(p + 8 * u, pf) : pf;
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            const Frag<P> vf = VTile::cols(vt, 32 * hh + 16 * u, 32 * i, lane, DVP);
            if (TWO_TERMS<T>) accumulate<T>(o[i], vf, rest);
            accumulate<T>(o[i], vf, pf);
          }
        }
      }
    }
    t = tn;
    bits = bits_next;
  }
  if constexpr (KW == 2) {         // the two waves' sums, one after the other
    float* box = reinterpret_cast<float*>(lds) + (size_t)qw * NV * 16 * 64;
    __syncthreads();
    if (kw == 1) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) box[(i * 16 + r) * 64 + lane] = o[i][r];
    }
    __syncthreads();
    if (kw == 1) return;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[i][r] += box[(i * 16 + r) * 64 + lane];
  }
  if (!q_on) return;
  const float down = 1.f / up;
  T* op = static_cast<T*>(a.out) + (((long long)b * a.N + q) * a.H + h) * a.dv_w;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int col = 32 * i + 2 * r + 4 * g;
      if (col < a.dv_w) store4<T>(op + col, o[i][r] * down, o[i][r + 1] * down, o[i][r + 2] * down, o[i][r + 3] * down);
    }
}

// A few rows against many keys: one pass over k and v, the keys split over workgroups.  The rows of a key head's group (queries x
// heads that share it) are the columns of 32-wide blocks.  A wave takes one map and one half of a tile's keys and keeps its own
// maximum, sum and P v, which split_join merges.  P is at most 1 here and not yet A, so it is taken in two terms (h + l): the
// pass waits for memory, the products are free.  fp16 takes 2^14 P: where one key leads, all others together may matter and each be below its steps.  Bound: HBM.  16 sequences x 16
// heads on 4, one query each, against 32768 keys, d = 64, dv = 128, bf16: 205 - 209 us for 1.07 GB, 5.1 - 5.2 TB/s (a large copy: 4.9); ragged 169 us for
// 0.74 GB, 4.4 TB/s.
template <class T, int DP, int DVP>
__global__ __launch_bounds__(THREADS, (FwdShape<T, DP, DVP>::MIN_BLOCKS)) void split_kernel(Args a) {
  typedef FwdShape<T, DP, DVP> S;
  typedef typename S::KTile KTile;
  typedef typename S::VTile VTile;
  constexpr int P = S::P, NV = DVP / 32;
  extern __shared__ __align__(256) char lds[];
  char* kt = lds;
  char* vt = lds + KTile::BYTES;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 5, l31 = lane & 31;
  const int hh = wave & 1, map = wave >> 1;
  const int group = a.H / a.Hkv, rows = a.N * group, blocks = (rows + 31) / 32;
  const int at = blockIdx.x / a.splits, bk = at / blocks, b = bk / a.Hkv, hk = bk - b * a.Hkv, row = (at - bk * blocks) * 32 + l31;
  const int split = (int)((blockIdx.x + at) % a.splits);        // turned by the head: the dies (ids modulo 8) share the ends of short sequences
  const int n = row / group, h = hk * group + (row - n * group);
  const bool on = row < rows;
  const long long off = (long long)a.M - a.N;
  const T* kp = static_cast<const T*>(a.k) + b * a.kb + 2ll * hk * a.kh;
  const T* vp = static_cast<const T*>(a.v) + b * a.vb + (long long)hk * a.vh;
  Frag<P> qf[DP / 16];
  load_rows<T, DP>(qf, static_cast<const T*>(a.q) + b * a.qb + (long long)n * a.qn + (2ll * h + map) * a.qh, on, a.d, g);

  KeyBits keys;
  keys.mask = a.mask ? a.mask + b * a.mb : nullptr;
  keys.words = reinterpret_cast<u64*>(lds + S::WORDS);
  keys.M = a.M;
  constexpr float UP = __is_same(T, _Float16) ? 16384.f : 1.f;
  const int tiles = (a.M + TILE - 1) / TILE, first = split * a.split_tiles;
  keys.end = first + a.split_tiles < tiles ? first + a.split_tiles : tiles;

  Stage<T, 2 * DP, 2> ks;
  Stage<T, DVP, 1> vs;
  ks.init(a.kn, a.kh, a.d, tid);
  vs.init(a.vn, 0, a.dv_w, tid);
  f32x16 o[NV];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) o[j] = zero16();
  u64 bits, bits_next;
  keys.start(first, wave, lane);
  int t = keys.next(first, bits, wave, lane);
  if (t < keys.end) {
    ks.load(kp + (long long)t * TILE * a.kn, bits, tid);
    vs.load(vp + (long long)t * TILE * a.vn, bits, tid);
  }
  while (t < keys.end) {
    __syncthreads();
    ks.put(kt, tid);
    vs.put(vt, tid);
    __syncthreads();
    const int tn = keys.next(t + 1, bits_next, wave, lane);
    if (tn < keys.end) {
      ks.load(kp + (long long)tn * TILE * a.kn, bits_next, tid);
      vs.load(vp + (long long)tn * TILE * a.vn, bits_next, tid);
    }
    const u64 see = a.causal ? bits & upto(n + off - (long long)t * TILE) : bits;
    Dot<T> dot;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) dot.add(KTile::rows(kt, 32 * hh, map * (DP / 16) + c, lane), qf[c]);
    f32x16 s = dot.sum();
    if (__any(see != ~0ull)) hide(s, see, hh, g);
    float top = row_max(s) * a.c;
    top = fmaxf(fmaxf(top, __shfl_xor(top, 32)), m);            // one maximum for both halves of the wave: they share a column of o
    const float tc = top == -INFINITY ? 0.f : top, keep = __builtin_amdgcn_exp2f(m - tc);
    m = top;
    float p[16], sum = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      p[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -tc));
      sum += p[r];
      p[r] *= UP;
    }
    l = fmaf(l, keep, sum);
    if (__any(keep != 1.f)) {                                    // most tiles leave every maximum as it is
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[j][r] *= keep;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const Frag<P> pf = pack8<T>(p + 8 * u), rest = TWO_TERMS<T> ? rest8<T>(p + 8 * u, pf) : pf;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const Frag<P> vf = VTile::cols(vt, 32 * hh + 16 * u, 32 * j, lane, DVP);
        if (TWO_TERMS<T>) accumulate<T>(o[j], vf, rest);
        accumulate<T>(o[j], vf, pf);
      }
    }
    t = tn;
    bits = bits_next;
  }
  // part: [bk][row][2 splits + half][2 dv + 4]: o1, o2, m1, l1, m2, l2
  l += __shfl_xor(l, 32);
  if (!on) return;
  const int slots = 2 * a.splits, ld = 2 * a.dv_w + 4;
  float* out = a.part + (((long long)bk * rows + row) * slots + 2 * split + hh) * ld;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int col = 32 * j + 2 * r + 4 * g;
      if (col < a.dv_w) *reinterpret_cast<f32x4*>(out + map * a.dv_w + col) = f32x4{o[j][r], o[j][r + 1], o[j][r + 2], o[j][r + 3]} * (1.f / UP);
    }
  if (g == 0) { out[2 * a.dv_w + 2 * map] = m; out[2 * a.dv_w + 2 * map + 1] = l; }
}

// One workgroup per (sequence, query, head): the parts of a row.  A wave holds every part's weight (one lane a part, 64 at a time); the four
// waves each take every fourth part, and their sums are added in order.
template <class T>
__global__ __launch_bounds__(THREADS) void split_join(Args a) {
  __shared__ float w1[64], w2[64];
  __shared__ f32x4 sum[4][32];
  const int id = blockIdx.x, h = id % a.H, bn = id / a.H, n = bn % a.N, b = bn / a.N, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int group = a.H / a.Hkv, hk = h / group, rows = a.N * group, row = n * group + (h - hk * group);
  const int slots = 2 * a.splits, ld = 2 * a.dv_w + 4;
  const float* in = a.part + ((long long)(b * a.Hkv + hk) * rows + row) * slots * ld;
  float w[2], mc[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float m = -INFINITY, l = 0.f;
    for (int s = lane; s < slots; s += 64) merge_stats(m, l, in[s * ld + 2 * a.dv_w + 2 * i], in[s * ld + 2 * a.dv_w + 2 * i + 1]);
    for (int x = 1; x < 64; x <<= 1) merge_stats(m, l, __shfl_xor(m, x), __shfl_xor(l, x));
    mc[i] = l == 0.f ? INFINITY : m;
    w[i] = l == 0.f ? 0.f : 1.f / l;
    if (a.stats != nullptr && threadIdx.x == 0) a.stats[((long long)(b * a.H + h) * 2 + i) * a.N + n] = make_float2(mc[i], w[i]);
  }
  const bool none = w[0] == 0.f && w[1] == 0.f;                    // sees nothing: zeros, whatever the parts hold
  w[1] *= -a.lambda[h];
  const int c = 4 * (lane & 31), side = lane >> 5;                 // lanes 0..31: P1 v, 32..63: P2 v; four columns each
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < slots; s0 += 64) {
    __syncthreads();
    if (threadIdx.x < 64 && s0 + lane < slots) {
      const float* p = in + (long long)(s0 + lane) * ld + 2 * a.dv_w;
      w1[lane] = w[0] * __builtin_amdgcn_exp2f(p[0] - mc[0]);
      w2[lane] = w[1] * __builtin_amdgcn_exp2f(p[2] - mc[1]);
    }
    __syncthreads();
    const int end = slots - s0 < 64 ? slots - s0 : 64;
    if (c < a.dv_w) {
#pragma unroll 4
      for (int s = wave; s < end; s += 4) v += (side ? w2[s] : w1[s]) * *reinterpret_cast<const f32x4*>(in + (long long)(s0 + s) * ld + side * a.dv_w + c);
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] += __shfl_xor(v[r], 32);
  if (side == 0) sum[wave][lane] = v;
  __syncthreads();
  if (threadIdx.x >= 32 || c >= a.dv_w) return;
  v = (sum[0][lane] + sum[1][lane]) + (sum[2][lane] + sum[3][lane]);
  if (none) v = f32x4{0.f, 0.f, 0.f, 0.f};
  store4<T>(static_cast<T*>(a.out) + (((long long)b * a.N + n) * a.H + h) * a.dv_w + c, v[0], v[1], v[2], v[3]);
}

template <class T, int DP, int DVP, int KW>
int launch_fwd(const Args& a, hipStream_t st) {
  typedef FwdShape<T, DP, DVP> S;
  const long long blocks = (long long)a.B * a.H * ((a.N + 128 / KW - 1) / (128 / KW));
  if (blocks > MAX_BLOCKS) return -3;
  static LdsAttrOnce once;
  if (set_max_dynamic_lds(once, reinterpret_cast<const void*>(&fwd_kernel<T, DP, DVP, KW>), S::LDS)) return -2;
  hipLaunchKernelGGL((fwd_kernel<T, DP, DVP, KW>), dim3((unsigned)blocks), dim3(THREADS), S::LDS, st, a);
  return 0;
}

template <class T, int DP, int DVP>
int launch_split(const Args& a, hipStream_t st) {
  typedef FwdShape<T, DP, DVP> S;
  const long long blocks = (long long)a.B * a.Hkv * (((long long)a.N * (a.H / a.Hkv) + 31) / 32) * a.splits;
  if (blocks > MAX_BLOCKS || (long long)a.B * a.N * a.H > MAX_BLOCKS) return -3;
  static LdsAttrOnce once;
  if (set_max_dynamic_lds(once, reinterpret_cast<const void*>(&split_kernel<T, DP, DVP>), S::LDS)) return -2;
  hipLaunchKernelGGL((split_kernel<T, DP, DVP>), dim3((unsigned)blocks), dim3(THREADS), S::LDS, st, a);
  hipLaunchKernelGGL((split_join<T>), dim3((unsigned)(a.B * a.N * a.H)), dim3(THREADS), 0, st, a);
  return 0;
}

// Few workgroups (of 128 queries): half as many queries in each, the keys of a tile shared by two waves, so that a workgroup's chain of tiles is
// shorter.  It is more work in all, so fuller grids lose; a causal grid's longest chain is its time, and it gains up to two workgroups per CU.  us, one
// wave / two, bf16, 2048 tokens, d = 64, dv = 128: 288 workgroups 154 / 156, 384 155 / 156, 480 160 / 187, 576 239 / 238, 768 248 / 281 (256 of 4096
// tokens 212 / 191; d = 32, dv = 64: 384 117 / 96, 480 118 / 129); causal 384 156 / 111, 480 156 / 140, 576 157 / 166, 768 181 / 193.  The bounds are those
// of the 16-bit types; in fp32 a causal grid gains beyond them too (1024 workgroups 1134 / 991, d = 32 492 / 406, d = 48 844 / 796; 2048 of d = 48 lose,
// 1559 / 1591).  Up to 64 queries half of the waves would have none: two waves at every number of sequences (bf16, 2048 of 20 tokens, 3 heads of 32 / 64
// 66 / 55, 512 of 64 tokens, 6 heads 36 / 32, fp32 87 / 64; 700 of 70 tokens, 2 heads 30 / 39, fp32 73 / 78).
inline bool few_queries(const Args& a) {
  return a.N <= 64 || (long long)a.B * a.H * (((long long)a.N + 127) / 128) <= (a.causal ? 512 : 384);
}

template <class T>
int run_forward(const Args& a, hipStream_t st) {
  const bool few = few_queries(a);
#define SCGG_X(DP, DVP) \
  if (a.d <= DP && a.dv_w <= DVP) return few ? launch_fwd<T, DP, DVP, 2>(a, st) : launch_fwd<T, DP, DVP, 1>(a, st);
  SCGG_DIFF_WIDTHS(SCGG_X)
#undef SCGG_X
  return -1;
}

template <class T>
int run_split(const Args& a, hipStream_t st) {
#define SCGG_X(DP, DVP) if (a.d <= DP && a.dv_w <= DVP) return launch_split<T, DP, DVP>(a, st);
  SCGG_DIFF_WIDTHS(SCGG_X)
#undef SCGG_X
  return -1;
}

}  // namespace diffattn
}  // namespace scgg
