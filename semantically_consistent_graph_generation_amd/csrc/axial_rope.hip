// Rotary positions with several axes on the heads of q and k, and the RMS norm of every head in the same pass (gfx950).
//
// Pair i of a head belongs to the axis whose section holds i; with n_a pairs on axis a its j-th pair turns by
// t = p_a theta^(-j / n_a).  Pairs behind the last section are left as they are.  A pair is (x_2i, x_2i+1) when interleaved,
// else (x_i, x_{i + D/2}):  (x, y) -> (x cos t - y sin t, x sin t + y cos t); the backward turns by -t.
// With weights, n = h w with h = x / sqrt(mean x^2 + eps) is rotated instead of x, and backward
//   u = R^T g,  dw = sum over tokens and heads of u h,  dx = (u w - h mean(u w h)) / sqrt(mean x^2 + eps).
//
// Bound: HBM (x in, y out; backward g, x in, dx out).  A workgroup takes a tile of tokens.  Its threads first form the cosines
// and sines of the tile, each once for all heads of q and k: positions reach 1e6 and beyond, so the angle is a product in two
// 64-bit terms, reduced to an eighth of a turn there, and only then rounded to 32.  Then the heads stream through, 16 B per load: a
// head belongs to a power of two of lanes that hold whole pairs, so the rotation needs no exchange and the norm one butterfly.
// In the backward of a norm a workgroup belongs to q or to k, so that a lane has one side's weights and sums (281 -> 258 us for 4 x 16384 tokens of
// 20 bf16 heads of 128; 252 now, the forward 162, together 1.68 GB at 4.0 TB/s); elsewhere it takes both, and the cosines are formed once (21
// against 25 us for 27648 tokens of 16 heads of 64).  Statistics and products are 32-bit, each output is rounded once.  The weight gradients are summed per lane (a lane keeps
// its channels), per workgroup through LDS, and over the workgroups by a second kernel in a fixed order: no atomics, equal
// calls give equal bits.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/scgg.h"
#include "kernels.h"

namespace scgg {
namespace {

constexpr int ROPE_MAX_PAIRS = 128;      // head width up to 256
constexpr int ROPE_TILE = 64;            // tokens per workgroup tile at most
constexpr int ROPE_GROUPS = 1 << 23;     // workgroups at most (a launch counts its threads in 32 bits); each takes every gridDim.x-th tile
constexpr int ROPE_TRAIN_GROUPS = 2048;  // workgroups of a backward with weights, q's and k's: rows of the partial sums

struct RopeSide {
  const void* x;               // q or k as the forward takes it (backward with weights: again; without: unused)
  const void* g;               // backward: gradient of the output
  void* y;                     // forward: output; backward: gradient of q or k.  [B,N,heads,D] contiguous
  const void* w;               // norm weight [D] or null
  long long xb, xn, xh, gb, gn, gh;
  int heads, tile;             // tokens per tile
  unsigned blocks;             // workgroups
};
struct RopeArgs {
  RopeSide side[2];            // q, k; where they have workgroups of their own, q's come first
  const void* pos;
  long long pb, pn, pa;
  float* partial;              // [gridDim.x][D]
  int N, D, pairs, pos_type, w_f32, interleaved, lanes;
  int flat;                    // every batch stride is N token strides: the token's number is its place
  unsigned tokens;
  float eps;
  double turn[ROPE_MAX_PAIRS]; // theta^(-j / n_a) / (2 pi), and what its rounding left
  double turn_low[ROPE_MAX_PAIRS];
  uint8_t axis[ROPE_MAX_PAIRS];
};

template <class T, int V>
struct Vec { typedef T type __attribute__((ext_vector_type(V))); };
template <class T>
struct Vec<T, 1> { struct type { T v; __device__ T& operator[](int) { return v; } __device__ T operator[](int) const { return v; } }; };

__device__ __forceinline__ void rope_place(const RopeArgs& a, unsigned tok, long long& b, long long& n) {
  const unsigned bb = a.flat ? 0u : tok / (unsigned)a.N;
  b = bb;
  n = tok - bb * (unsigned)a.N;
}

__device__ __forceinline__ double rope_position(const RopeArgs& a, unsigned tok, int ax) {
  long long b, n;
  rope_place(a, tok, b, n);
  const long long at = b * a.pb + n * a.pn + ax * a.pa;
  if (a.pos_type == SCGG_POS_F32) return (double)static_cast<const float*>(a.pos)[at];
  if (a.pos_type == SCGG_POS_F64) return static_cast<const double*>(a.pos)[at];
  if (a.pos_type == SCGG_POS_I32) return (double)static_cast<const int32_t*>(a.pos)[at];
  return (double)static_cast<const int64_t*>(a.pos)[at];
}

// cos and sin of p (turn + low) turns.  The product is formed to twice 64 bits and its whole turns come off first, so every position that 64 bits
// hold keeps its angle (10^12 tokens out, a product rounded to 64 bits is off by 1e-4; past 2^50 it has no fraction).  Then the nearest quarter
// turn comes off (adding 1.5 2^52 rounds to a whole number and leaves it in the low word), so the one rounding to 32 happens to an angle of at most
// pi / 4: 2^-25.  There the series of sin and cos need five terms each: the first term left out is below x^11 / 11! = 2e-9.  The quarter is a
// swap and two signs.
__device__ __forceinline__ float2 rope_cos_sin(double p, double turn, double low) {
  double turns = fma(p, low, fma(p, turn, -rint(p * turn)));   // the inner sum is exact to 2^-54 of itself
  turns -= rint(turns);
  const double big = 6755399441055744.0, t = fma(4.0, turns, big), q = t - big;
  const int k = __double2loint(t);
  const float x = (float)(6.283185307179586 * fma(-0.25, q, turns)), y = x * x;
  const float s = fmaf(x * y, fmaf(y, fmaf(y, fmaf(y, 2.755731922e-6f, -1.984126984e-4f), 8.333333333e-3f), -1.666666667e-1f), x);
  const float c = fmaf(y, fmaf(y, fmaf(y, fmaf(y, fmaf(y, -2.755731922e-7f, 2.480158730e-5f), -1.388888889e-3f), 4.166666667e-2f), -0.5f), 1.f);
  const float cs = (k & 1) ? s : c, sn = (k & 1) ? c : s;
  return make_float2(((k + 1) & 2) ? -cs : cs, (k & 2) ? -sn : sn);
}

template <class T>
__device__ __forceinline__ float rope_weight(const void* w, bool f32, int i) {
  return f32 ? static_cast<const float*>(w)[i] : (float)static_cast<const T*>(w)[i];
}

// NORM: heads are normalised first.  BWD: gradient pass.  V: elements per load, CH: pair chunks of V per lane.
template <class T, int V, int CH, bool NORM, bool BWD>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
  typedef typename Vec<T, V>::type vec;
  extern __shared__ __align__(16) char rope_lds[];
  float2* cs = reinterpret_cast<float2*>(rope_lds);                       // [tile][D/2]
  const int tid = threadIdx.x, L = a.lanes, half = a.D >> 1;
  const int chunks = half / V, group = tid / L, groups = 256 / L, lane = tid - group * L;
  constexpr bool APART = NORM && BWD;                                      // q and k in workgroups of their own
  constexpr int SIDES = APART ? 1 : 2;
  const bool is_k = APART && blockIdx.x >= a.side[0].blocks;
  const RopeSide& mine = is_k ? a.side[1] : a.side[0];
  const unsigned block = blockIdx.x - (is_k ? a.side[0].blocks : 0u);
  int c0[CH], c1[CH];                                                     // element offsets of the lane's pairs: (c0 + i, c1 + i) or neighbours
  bool on[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int ch = lane + c * L;
    on[c] = ch < chunks;
    c0[c] = a.interleaved ? 2 * V * ch : V * ch;
    c1[c] = a.interleaved ? c0[c] + V : c0[c] + half;
  }
  float w[SIDES][CH][2 * V], dw[CH][2 * V];
  if (NORM) {
#pragma unroll
    for (int s = 0; s < SIDES; ++s) {
      const RopeSide& q = APART ? mine : a.side[s];
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const bool have = on[c] && q.heads > 0;
          w[s][c][i] = have ? rope_weight<T>(q.w, a.w_f32, c0[c] + i) : 0.f;
          w[s][c][V + i] = have ? rope_weight<T>(q.w, a.w_f32, c1[c] + i) : 0.f;
          if (BWD) dw[c][i] = dw[c][V + i] = 0.f;
        }
    }
  }
  const float inv_d = 1.0f / (float)a.D;
  const int q_heads = a.side[0].heads, heads = APART ? mine.heads : q_heads + a.side[1].heads;
  const int dk = groups / heads, dh = groups - dk * heads, k_first = group / heads, h_first = group - k_first * heads;
  const unsigned tiles = (a.tokens + mine.tile - 1) / mine.tile;
  for (unsigned t = block; t < tiles; t += mine.blocks) {
    const unsigned tok0 = t * mine.tile;
    const int count = (int)min(a.tokens - tok0, (unsigned)mine.tile);
    if (a.pairs > 0) {
      __syncthreads();                                                    // the previous tile's readers are done
      for (int i = tid; i < count * half; i += 256) {
        const int k = i / half, pair = i - k * half;
        float2 v = make_float2(1.f, 0.f);
        if (pair < a.pairs) {
          v = rope_cos_sin(rope_position(a, tok0 + k, a.axis[pair]), a.turn[pair], a.turn_low[pair]);
        }
        cs[i] = v;
      }
      __syncthreads();
    }
    int k = k_first, h = h_first;                                         // token of the tile, head
    while (k < count) {                                                   // uniform over the L lanes of a head
      const unsigned tok = tok0 + k;
      long long b, n;
      rope_place(a, tok, b, n);
      const bool s = APART ? is_k : h >= q_heads;
      const int hh = APART || !s ? h : h - q_heads;
      const RopeSide& q = a.side[0];
      const RopeSide& kk = a.side[1];
      const T* xp = (BWD && !NORM) ? nullptr
                                   : static_cast<const T*>(s ? kk.x : q.x) + b * (s ? kk.xb : q.xb) + n * (s ? kk.xn : q.xn) + hh * (s ? kk.xh : q.xh);
      const T* gp = BWD ? static_cast<const T*>(s ? kk.g : q.g) + b * (s ? kk.gb : q.gb) + n * (s ? kk.gn : q.gn) + hh * (s ? kk.gh : q.gh) : nullptr;
      T* yp = static_cast<T*>(s ? kk.y : q.y) + ((long long)tok * (s ? kk.heads : q.heads) + hh) * a.D;
      float x[CH][2 * V], g[CH][2 * V];
      float ss = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (on[c]) {
          if (!BWD || NORM) {
            const vec v0 = *reinterpret_cast<const vec*>(xp + c0[c]), v1 = *reinterpret_cast<const vec*>(xp + c1[c]);
#pragma unroll
            for (int i = 0; i < V; ++i) { x[c][i] = (float)v0[i]; x[c][V + i] = (float)v1[i]; }
          }
          if (BWD) {
            const vec v0 = *reinterpret_cast<const vec*>(gp + c0[c]), v1 = *reinterpret_cast<const vec*>(gp + c1[c]);
#pragma unroll
            for (int i = 0; i < V; ++i) { g[c][i] = (float)v0[i]; g[c][V + i] = (float)v1[i]; }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) x[c][i] = g[c][i] = 0.f;
        }
        if (NORM) {
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) ss = fmaf(x[c][i], x[c][i], ss);
        }
      }
      float r = 1.f;
      if (NORM) {
        for (int m = 1; m < L; m <<= 1) ss += __shfl_xor(ss, m);
        r = rsqrtf(ss * inv_d + a.eps);
      }
      float dot = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (!on[c]) continue;
        float2 t2[V];
        const int p0 = V * (lane + c * L);
        if (a.pairs > 0) {
#pragma unroll
          for (int i = 0; i < V; ++i) t2[i] = cs[k * half + p0 + i];
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) t2[i] = make_float2(1.f, 0.f);
        }
        float* z = BWD ? g[c] : x[c];
        if (NORM && !BWD) {
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) z[i] = z[i] * r * (!APART && s ? w[SIDES - 1][c][i] : w[0][c][i]);
        }
        if (a.interleaved) {
          // elements e = 0 .. 2V-1 of the lane are neighbours: pair i is (2i, 2i + 1)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float p = z[2 * i], q = z[2 * i + 1], sn = BWD ? -t2[i].y : t2[i].y;
            z[2 * i] = fmaf(p, t2[i].x, -(q * sn));
            z[2 * i + 1] = fmaf(p, sn, q * t2[i].x);
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float p = z[i], q = z[V + i], sn = BWD ? -t2[i].y : t2[i].y;
            z[i] = fmaf(p, t2[i].x, -(q * sn));
            z[V + i] = fmaf(p, sn, q * t2[i].x);
          }
        }
        if (NORM && BWD) {
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) {
            const float hx = x[c][i] * r;
            const float du = z[i] * hx;
            dw[c][i] += du;
            dot = fmaf(du, w[0][c][i], dot);
            x[c][i] = hx;
            z[i] *= w[0][c][i];
          }
        }
      }
      if (NORM && BWD) {
        for (int m = 1; m < L; m <<= 1) dot += __shfl_xor(dot, m);
        dot *= inv_d;
      }
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (!on[c]) continue;
        vec v0, v1;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float p = BWD ? g[c][i] : x[c][i], q = BWD ? g[c][V + i] : x[c][V + i];
          if (NORM && BWD) { p = r * fmaf(-x[c][i], dot, p); q = r * fmaf(-x[c][V + i], dot, q); }
          v0[i] = (T)p;
          v1[i] = (T)q;
        }
        *reinterpret_cast<vec*>(yp + c0[c]) = v0;
        *reinterpret_cast<vec*>(yp + c1[c]) = v1;
      }
      h += dh;
      k += dk;
      if (h >= heads) { h -= heads; ++k; }
    }
  }
  if (NORM && BWD) {
    // the workgroup's sums: [groups][D] of LDS, groups added in order
    float* red = reinterpret_cast<float*>(rope_lds);
    __syncthreads();
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if (on[c]) {
#pragma unroll
        for (int i = 0; i < V; ++i) { red[group * a.D + c0[c] + i] = dw[c][i]; red[group * a.D + c1[c] + i] = dw[c][V + i]; }
      }
    __syncthreads();
    for (int d = tid; d < a.D; d += 256) {
      double v = 0.0;
      for (int q = 0; q < groups; ++q) v += red[q * a.D + d];
      a.partial[(long long)blockIdx.x * a.D + d] = (float)v;
    }
  }
}

// gradient of a weight = sum of its workgroups' partials (rows [0, split) are q's, [split, rows) k's): 16 columns x 64 row lanes per
// workgroup, lanes added in order.  64 bits, as in the sum over a workgroup's groups: the terms cancel to about the root of their number, and some
// 150 additions of 32 bits in a row would add twice the terms' own rounding
template <class T>
__global__ __launch_bounds__(1024) void rope_dw_kernel(const float* __restrict__ partial, int split, int rows, int D, int w_f32, void* dw0, void* dw1) {
  __shared__ double red[64][17];
  const int d = blockIdx.x * 16 + (threadIdx.x & 15), rl = threadIdx.x >> 4;
  const int from = blockIdx.y == 0 ? 0 : split, to = blockIdx.y == 0 ? split : rows;
  double v = 0.0;
  if (d < D) {
#pragma unroll 4
    for (int r = from + rl; r < to; r += 64) v += partial[(long long)r * D + d];
  }
  red[rl][threadIdx.x & 15] = v;
  __syncthreads();
  void* o = blockIdx.y == 0 ? dw0 : dw1;
  if (rl != 0 || d >= D || o == nullptr) return;
  for (int q = 1; q < 64; ++q) v += red[q][threadIdx.x & 15];
  if (w_f32) static_cast<float*>(o)[d] = (float)v;
  else static_cast<T*>(o)[d] = (T)(float)v;
}

template <class T, int V, int CH, bool NORM>
void rope_launch2(const RopeArgs& a, bool bwd, unsigned blocks, size_t lds, hipStream_t st) {
  if (bwd) hipLaunchKernelGGL((rope_kernel<T, V, CH, NORM, true>), dim3(blocks), dim3(256), lds, st, a);
  else hipLaunchKernelGGL((rope_kernel<T, V, CH, NORM, false>), dim3(blocks), dim3(256), lds, st, a);
}
template <class T, int V, int CH>
void rope_launch1(const RopeArgs& a, bool norm, bool bwd, unsigned blocks, size_t lds, hipStream_t st) {
  if (norm) rope_launch2<T, V, CH, true>(a, bwd, blocks, lds, st);
  else rope_launch2<T, V, CH, false>(a, bwd, blocks, lds, st);
}
template <class T>
void rope_launch(const RopeArgs& a, int vec, bool norm, bool bwd, unsigned blocks, size_t lds, hipStream_t st) {
  constexpr int W = 16 / sizeof(T);
  if (vec == W) rope_launch1<T, W, 1>(a, norm, bwd, blocks, lds, st);
  else if (vec == 2) rope_launch1<T, 2, 1>(a, norm, bwd, blocks, lds, st);
  else rope_launch1<T, 1, 2>(a, norm, bwd, blocks, lds, st);
}

int rope_lanes(int chunks) {
  int L = 1;
  while (L < chunks && L < 64) L <<= 1;
  return L;
}

// The plan of a call: elements per load, lanes per head, and for q and k tokens per tile and workgroups.
struct RopePlan { int vec, lanes, tile[2]; long long blocks[2]; size_t lds; };
void rope_plan(const scgg_rope_args* p, bool bwd, bool norm, RopePlan* out) {
  const int size = p->dtype == SCGG_F32 ? 4 : 2, half = p->D / 2, wide = 16 / size;
  auto fits = [&](int v) {   // every row of every head starts at a multiple of the load's width
    if (half % v != 0) return false;
    const long long by = (long long)v * size;
    for (int s = 0; s < 2; ++s) {
      if (p->heads[s] == 0) continue;
      uintptr_t all = reinterpret_cast<uintptr_t>(p->y[s]);
      if (!bwd || norm) all |= reinterpret_cast<uintptr_t>(p->x[s]) | (uintptr_t)((p->x_stride_b[s] | p->x_stride_n[s] | p->x_stride_h[s]) * size);
      if (bwd) all |= reinterpret_cast<uintptr_t>(p->g[s]) | (uintptr_t)((p->g_stride_b[s] | p->g_stride_n[s] | p->g_stride_h[s]) * size);
      if (all % by != 0) return false;
    }
    return true;
  };
  out->vec = fits(wide) ? wide : fits(2) ? 2 : 1;
  out->lanes = rope_lanes(half / out->vec);
  const long long tokens = (long long)p->B * p->N;
  out->lds = 0;
  const long long all = (long long)p->heads[0] + p->heads[1];
  const bool apart = bwd && norm;
  for (int s = 0; s < 2; ++s) {
    // long inputs: a tile has about twelve heads for each group of lanes, and its cosines fill 16 KiB at most; shorter ones: smaller
    // tiles, so that there are some 1500 workgroups (q's and k's by their heads), down to one token each
    const long long own = apart ? p->heads[s] : s == 0 ? all : 0;
    out->tile[s] = 1;
    out->blocks[s] = 0;
    if (own == 0 || tokens == 0) continue;
    const long long many = tokens * all / own / 1536, turn = 12 * 256 / out->lanes / own + 1, room = 2048 / half;
    long long tile = many < turn ? many : turn;
    if (tile > room) tile = room;
    if (tile > ROPE_TILE) tile = ROPE_TILE;
    if (tile < 1) tile = 1;
    const long long groups = 256 / out->lanes;
    auto idle = [&](long long t) { return (double)((t * own + groups - 1) / groups * groups) / (double)(t * own); };
    for (long long t = tile, least = tile / 2 + 1; t >= least; --t)         // of the sizes down to half: the one whose last round is fullest
      if (idle(t) < idle(tile) - 1e-9) tile = t;
    const long long tiles = (tokens + tile - 1) / tile, cap = apart ? ROPE_TRAIN_GROUPS * own / all : ROPE_GROUPS;
    out->tile[s] = (int)tile;
    out->blocks[s] = tiles < cap ? tiles : cap < 1 ? 1 : cap;
    const size_t lds = p->n_sections > 0 ? (size_t)tile * half * sizeof(float2) : 0;
    if (lds > out->lds) out->lds = lds;
  }
  if (bwd && norm) {
    const size_t red = (size_t)(256 / out->lanes) * p->D * sizeof(float);
    if (red > out->lds) out->lds = red;
  }
}

int rope_check(const scgg_rope_args* p, const char* what) {
  if (!p) return fail("%s: null argument", what);
  if (p->dtype != SCGG_F32 && p->dtype != SCGG_BF16 && p->dtype != SCGG_F16) return fail("%s: unknown dtype %d", what, p->dtype);
  if (p->B < 0 || p->N < 0 || p->heads[0] < 0 || p->heads[1] < 0 || p->D < 2) return fail("%s: bad shape", what);
  if (p->D % 2 != 0 || p->D > 2 * ROPE_MAX_PAIRS) return fail("%s: head width %d: even and at most %d is supported", what, p->D, 2 * ROPE_MAX_PAIRS);
  if (p->heads[0] > 65535 || p->heads[1] > 65535) return fail("%s: too many heads", what);
  if (p->n_sections < 0 || p->n_sections > SCGG_ROPE_MAX_AXES) return fail("%s: %d axes: at most %d are supported", what, p->n_sections, SCGG_ROPE_MAX_AXES);
  long long pairs = 0;
  for (int i = 0; i < p->n_sections; ++i) {
    if (p->sections[i] < 0) return fail("%s: a section has %d pairs", what, p->sections[i]);
    pairs += p->sections[i];
  }
  if (pairs > p->D / 2) return fail("%s: the sections take %lld pairs, a head of width %d has %d", what, pairs, p->D, p->D / 2);
  if (p->n_sections > 0) {
    if (!(p->theta > 0.0) || !isfinite(p->theta)) return fail("%s: theta has to be positive and finite", what);
    if (!p->positions && (long long)p->B * p->N > 0) return fail("%s: sections without positions", what);
    if (p->pos_type < SCGG_POS_F32 || p->pos_type > SCGG_POS_I64) return fail("%s: unknown position type", what);
  }
  if ((long long)p->B * p->N > 0x7fffffffLL - 256) return fail("%s: too many tokens for one launch", what);
  const bool norm = p->weight[0] || p->weight[1];
  for (int s = 0; s < 2; ++s) {
    if (p->heads[s] == 0 || p->B == 0 || p->N == 0) continue;
    if (norm && !p->weight[s]) return fail("%s: a norm needs the weights of q and of k", what);
    if (!p->y[s]) return fail("%s: null output", what);
  }
  if (norm && !(p->eps >= 0.f)) return fail("%s: eps has to be at least 0", what);
  return 0;
}

int rope_run(const scgg_rope_args* p, bool bwd, const char* what, void* workspace, size_t workspace_bytes, hipStream_t st) {
  const bool norm = p->weight[0] || p->weight[1];
  for (int s = 0; s < 2 && (long long)p->B * p->N > 0; ++s) {
    if (p->heads[s] == 0) continue;
    if ((!bwd || norm) && !p->x[s]) return fail("%s: null input", what);
    if (bwd && !p->g[s]) return fail("%s: null gradient", what);
  }
  RopePlan plan;
  rope_plan(p, bwd, norm, &plan);
  RopeArgs a = {};
  const long long blocks = plan.blocks[0] + plan.blocks[1];
  for (int s = 0; s < 2; ++s) {
    RopeSide& q = a.side[s];
    q.x = p->x[s]; q.g = p->g[s]; q.y = p->y[s]; q.w = p->weight[s]; q.heads = p->heads[s];
    q.xb = p->x_stride_b[s]; q.xn = p->x_stride_n[s]; q.xh = p->x_stride_h[s];
    q.gb = p->g_stride_b[s]; q.gn = p->g_stride_n[s]; q.gh = p->g_stride_h[s];
    q.tile = plan.tile[s]; q.blocks = (unsigned)plan.blocks[s];
  }
  a.pos = p->positions; a.pb = p->pos_stride_b; a.pn = p->pos_stride_n; a.pa = p->pos_stride_a; a.pos_type = p->pos_type;
  a.N = p->N > 0 ? p->N : 1; a.D = p->D; a.w_f32 = p->weight_f32; a.interleaved = p->interleaved != 0;
  a.lanes = plan.lanes; a.tokens = (unsigned)(p->B * p->N); a.eps = p->eps;
  a.flat = 1;
  for (int s = 0; s < 2; ++s) {
    if (p->heads[s] == 0 || p->B <= 1) continue;
    if (!bwd || norm) a.flat &= p->x_stride_b[s] == p->x_stride_n[s] * p->N;
    if (bwd) a.flat &= p->g_stride_b[s] == p->g_stride_n[s] * p->N;
  }
  if (p->B > 1 && p->n_sections > 0) a.flat &= p->pos_stride_b == p->pos_stride_n * p->N;
  for (int i = 0; i < p->n_sections; ++i) {
    const int n = p->sections[i];
    if (n == 0) continue;
    // theta^(-j / n) (1 / (2 pi)) as a sum of two: 1 / (2 pi) is one, the powers have long double's 64 bits less one step for each factor.
    // theta^(-1 / n): one Newton step on theta r^n = 1 from the 53 bits of pow (powl takes 0.4 us an axis)
    const double pi2 = 0x1.45f306dc9c883p-3, pi2_low = -0x1.6b01ec5417056p-57, root = pow(p->theta, -1.0 / n);
    long double power = 1.0L, square = root, f = 1.0L;
    for (int bit = n; bit > 0; bit >>= 1, square *= square)
      if (bit & 1) power *= square;
    const long double ratio = root + root * (1.0L - (long double)p->theta * power) / n;
    for (int j = 0; j < n; ++j, f *= ratio) {
      const long double t = f * pi2;                                        // exact for j = 0
      a.turn[a.pairs] = (double)t;
      a.turn_low[a.pairs] = (double)(t - a.turn[a.pairs] + f * pi2_low);
      a.axis[a.pairs++] = (uint8_t)i;
    }
  }
  if (a.pairs == 0 && !(bwd && norm)) plan.lds = 0;
  if (bwd && norm) {
    const size_t need = (size_t)blocks * p->D * sizeof(float);
    if (need > 0 && (!workspace || workspace_bytes < need)) return fail("%s: workspace of %zu bytes, %zu are needed", what, workspace_bytes, need);
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail("%s: workspace has to be aligned to 16 bytes", what);
    a.partial = static_cast<float*>(workspace);
  }
  if (blocks > 0) {
    if (p->dtype == SCGG_F32) rope_launch<float>(a, plan.vec, norm, bwd, (unsigned)blocks, plan.lds, st);
    else if (p->dtype == SCGG_BF16) rope_launch<__bf16>(a, plan.vec, norm, bwd, (unsigned)blocks, plan.lds, st);
    else rope_launch<_Float16>(a, plan.vec, norm, bwd, (unsigned)blocks, plan.lds, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail("%s: %s", what, hipGetErrorString(e));
  }
  if (bwd && norm && (p->dweight[0] || p->dweight[1])) {
    const dim3 grid((unsigned)((p->D + 15) / 16), 2);
    const int split = (int)plan.blocks[0], rows = (int)blocks;   // none: the sums are zero
    if (p->dtype == SCGG_F32) hipLaunchKernelGGL(rope_dw_kernel<float>, grid, dim3(1024), 0, st, a.partial, split, rows, p->D, p->weight_f32, p->dweight[0], p->dweight[1]);
    else if (p->dtype == SCGG_BF16) hipLaunchKernelGGL(rope_dw_kernel<__bf16>, grid, dim3(1024), 0, st, a.partial, split, rows, p->D, p->weight_f32, p->dweight[0], p->dweight[1]);
    else hipLaunchKernelGGL(rope_dw_kernel<_Float16>, grid, dim3(1024), 0, st, a.partial, split, rows, p->D, p->weight_f32, p->dweight[0], p->dweight[1]);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail("%s: %s", what, hipGetErrorString(e));
  }
  return 0;
}

}  // namespace
}  // namespace scgg

using namespace scgg;

extern "C" size_t scgg_rope_workspace_bytes(const scgg_rope_args* p) {
  if (rope_check(p, "rope_workspace_bytes")) return 0;
  return (size_t)(ROPE_TRAIN_GROUPS + 2) * p->D * sizeof(float);
}

extern "C" int scgg_rope_forward(const scgg_rope_args* p, void* stream) {
  if (rope_check(p, "rope_forward")) return -1;
  return rope_run(p, false, "rope_forward", nullptr, 0, static_cast<hipStream_t>(stream));
}

extern "C" int scgg_rope_backward(const scgg_rope_args* p, void* workspace, size_t workspace_bytes, void* stream) {
  if (rope_check(p, "rope_backward")) return -1;
  return rope_run(p, true, "rope_backward", workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}
