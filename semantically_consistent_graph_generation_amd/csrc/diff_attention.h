// Differential attention (gfx950): shared parts of the forward and backward kernels.
//
//   out_h = A v,  A = P1 - lambda_h P2,  P_i = softmax(scale q_i k_i^T)
//
// Everything runs on v_mfma_f32_32x32x16: lane l supplies row / column l & 31 and the 8 contraction slots of half l >> 5; the
// result has column l & 31 and rows 8 (r >> 2) + 4 (l >> 5) + (r & 3).  A product whose result feeds the next one is
// formed with the axis that the next one sums over in the rows: the 16 values that a lane then holds are the operand of two
// products over 16 slots each (the slots' order is the rows' order, so the other operand is read in that order).
//
// Types: bf16 and fp16 multiply as they are.  fp32 is split exactly into three bf16 terms (h + m + l) and a product is the six
// leading partial products, which keeps fp32's accuracy at up to 2.7 times the rate of the fp32 matrix instructions (peaks: 2500 / 6 against 157 TFLOP/s).  A tile in LDS has a plane per
// term, so the kernels are the same for all types.
//
// Tiles in LDS: 64 rows (keys, or queries in the dK / dV kernel), read row-wise (b128) and transposed (tr_b64).
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/scgg.h"
#include "kernels.h"

namespace scgg {
namespace diffattn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned long long u64;

constexpr int TILE = 64;          // keys (or queries) per tile: one bit each in a wave-wide ballot
constexpr int THREADS = 256;
constexpr long long MAX_BLOCKS = 0xffffffffll / THREADS;   // a launch counts its threads in 32 bits

struct Args {
  const void *q, *k, *v, *dout;
  const float* lambda;
  const uint8_t* mask;
  void *out, *dq, *dk, *dv;
  float2* stats;                  // [B,H,2,N]: scale log2(e) max, 1 / sum
  float* delta;                   // [B,H,2,N]: sum_j P_i dP
  float* part;                    // partial results of the splits (split_kernel, dq_kernel, dkv_kernel)
  long long qb, qn, qh, kb, kn, kh, vb, vn, vh, gb, gn, gh, mb;
  float scale, c;                 // c = scale log2(e)
  int B, N, M, H, Hkv, d, dv_w, causal;
  int splits, split_tiles;        // forward: workgroups along the keys and the tiles each of them takes; dkv_kernel: along the queries
  int dq_splits;                  // dq_kernel: workgroups along the keys
};

// ------------------------------------------------------------------------------------------------ element types
template <int P>
struct Frag { u32x4 p[P]; };      // 8 contraction slots of a lane, P planes

template <class T>
struct Type;
template <>
struct Type<__bf16> {
  static constexpr int planes = 1;
  static __device__ __forceinline__ f32x16 mma1(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Type<_Float16> {
  static constexpr int planes = 1;
  static __device__ __forceinline__ f32x16 mma1(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Type<float> {
  static constexpr int planes = 3;
  static __device__ __forceinline__ f32x16 mma1(u32x4 a, u32x4 b, f32x16 c) { return Type<__bf16>::mma1(a, b, c); }
};

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// A sum of products over the operands' slots, as a matrix instruction rounds it: fp32's six partial products in one accumulator would be
// six roundings (with a bias of some 1e-3 of a step) of a sum that grows, so the five small ones have an accumulator of their own.
template <class T>
struct Dot {
  f32x16 a = zero16(), small = zero16();
  __device__ __forceinline__ void add(const Frag<Type<T>::planes>& x, const Frag<Type<T>::planes>& y) {
    if constexpr (Type<T>::planes == 1) {
      a = Type<T>::mma1(x.p[0], y.p[0], a);
    } else {
      small = Type<T>::mma1(x.p[2], y.p[0], small);
      small = Type<T>::mma1(x.p[0], y.p[2], small);
      small = Type<T>::mma1(x.p[1], y.p[1], small);
      small = Type<T>::mma1(x.p[1], y.p[0], small);
      small = Type<T>::mma1(x.p[0], y.p[1], small);
      a = Type<T>::mma1(x.p[0], y.p[0], a);
    }
  }
  __device__ __forceinline__ f32x16 sum() const {
    if constexpr (Type<T>::planes == 1) return a;
    else return a + small;
  }
};

// o += x y, for sums over many tiles: fp32's six products are added up from zero and rounded into the long sum once
template <class T>
__device__ __forceinline__ void accumulate(f32x16& o, const Frag<Type<T>::planes>& x, const Frag<Type<T>::planes>& y) {
  if constexpr (Type<T>::planes == 1) {
    o = Type<T>::mma1(x.p[0], y.p[0], o);
  } else {
    f32x16 t = Type<T>::mma1(x.p[2], y.p[0], zero16());       // smallest first
    t = Type<T>::mma1(x.p[0], y.p[2], t);
    t = Type<T>::mma1(x.p[1], y.p[1], t);
    t = Type<T>::mma1(x.p[1], y.p[0], t);
    t = Type<T>::mma1(x.p[0], y.p[1], t);
    t = Type<T>::mma1(x.p[0], y.p[0], t);
    o += t;
  }
}

// two fp32 values into one packed word of each plane
template <class T>
__device__ __forceinline__ void pack2(float x, float y, unsigned (&out)[Type<T>::planes]) {
  if constexpr (Type<T>::planes == 1) {
    typedef T t2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    out[0] = __builtin_bit_cast(unsigned, __builtin_convertvector((f2{x, y}), t2));   // one conversion for both, to nearest
  } else {                         // x = h + m + l by truncation: exact
    unsigned u = __float_as_uint(x), w = __float_as_uint(y);
    out[0] = __builtin_amdgcn_perm(w, u, 0x07060302u);
    x -= __uint_as_float(u & 0xffff0000u);
    y -= __uint_as_float(w & 0xffff0000u);
    u = __float_as_uint(x);
    w = __float_as_uint(y);
    out[1] = __builtin_amdgcn_perm(w, u, 0x07060302u);
    x -= __uint_as_float(u & 0xffff0000u);
    y -= __uint_as_float(w & 0xffff0000u);
    out[2] = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
  }
}

template <class T>
__device__ __forceinline__ Frag<Type<T>::planes> pack8(const float* x) {
  Frag<Type<T>::planes> f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unsigned w[Type<T>::planes];
    pack2<T>(x[2 * i], x[2 * i + 1], w);
#pragma unroll
    for (int p = 0; p < Type<T>::planes; ++p) f.p[p][i] = w[p];
  }
  return f;
}

// 16 bits: A and dS go into their products in two terms, rounded and rest.  Rounded once they add about as much error as the output's own
// rounding does (together 1.41 to 1.67 times that of 32 bits rounded at the end), and a bound on the size, up to which the second term is taken, would
// let a sequence's error depend on its batch.  bf16, forward and training pass, one term / two, us: 4096 causal, 8 heads on 4, 153 / 165, 532 / 585; 2 x 8192,
// 8 heads, 1050 / 1205, 4240 / 5040; 4 x 2048, 16 heads of 32 / 64, 183 / 210, 650 / 796.
template <class T>
constexpr bool TWO_TERMS = Type<T>::planes == 1;

// What pack8 left of x: x - f, rounded in turn.  From the packed words: a conversion of x for itself may be fused with the product that x comes from,
// and then rounds a value near a tie to the other side now and then (fp16), a whole step off.
template <class T>
__device__ __forceinline__ Frag<Type<T>::planes> rest8(const float* x, const Frag<Type<T>::planes>& f) {
  if constexpr (Type<T>::planes == 1) {
    typedef T t2 __attribute__((ext_vector_type(2)));
    float q[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned w = f.p[0][i];
      const t2 h = __builtin_bit_cast(t2, w);
      q[2 * i] = x[2 * i] - (float)h[0];
      q[2 * i + 1] = x[2 * i + 1] - (float)h[1];
    }
    return pack8<T>(q);
  } else {
    return f;                      // nothing is left
  }
}

// Loads of a tile go through a buffer descriptor: a 64-bit base in scalar registers for the tile, a 32-bit byte offset per lane, and
// an offset past the descriptor's 2 GiB gives zeros without a branch.
constexpr unsigned NOWHERE = 0x80000000u;
typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __forceinline__ Buffer buffer(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, 0x7fffffff, 0x00027000);
}
__device__ __forceinline__ u32x4 buffer_load(Buffer b, unsigned at) { return __builtin_amdgcn_raw_buffer_load_b128(b, at, 0, 0); }

// 8 elements as they lie in memory
template <class T>
struct Raw {
  u32x4 a;
  __device__ __forceinline__ void load(const T* p) { a = *reinterpret_cast<const u32x4*>(p); }
  __device__ __forceinline__ void load(Buffer b, unsigned at) { a = buffer_load(b, at); }
  __device__ __forceinline__ void clear() { a = u32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ Frag<1> frag() const { return Frag<1>{{a}}; }
};
template <>
struct Raw<float> {
  f32x4 a, b;
  __device__ __forceinline__ void load(const float* p) { a = *reinterpret_cast<const f32x4*>(p); b = *reinterpret_cast<const f32x4*>(p + 4); }
  __device__ __forceinline__ void load(Buffer f, unsigned at) {
    a = __builtin_bit_cast(f32x4, buffer_load(f, at));
    b = __builtin_bit_cast(f32x4, buffer_load(f, at == NOWHERE ? at : at + 16));
  }
  __device__ __forceinline__ void clear() { a = b = f32x4{0.f, 0.f, 0.f, 0.f}; }
  __device__ __forceinline__ Frag<3> frag() const {
    const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return pack8<float>(x);
  }
};

// ------------------------------------------------------------------------------------------------ tiles in LDS
// A tile of `ROWS` rows and W columns, P planes.  A row is an odd number of 64-byte groups, so four rows in a row start 16 banks
// apart, and the four chunks of a group are permuted by row / 4: 16 rows at one chunk meet every bank once, and so do 4 rows at
// 32 columns.  The permutation stays within a group: all reads of a lane are two addresses and constant offsets.
template <int W, int P, int ROWS = TILE>
struct Tile {
  static constexpr int GROUPS = W / 32, ROW = 64 * (GROUPS % 2 == 0 ? GROUPS + 1 : GROUPS), PLANE = ROWS * ROW, BYTES = P * PLANE;
  static_assert(W % 32 == 0, "rows of whole 64-byte groups");
  static __device__ __forceinline__ int place(int row, int chunk) {    // byte offset of a row's 16-byte chunk
    return row * ROW + 16 * (chunk ^ ((row >> 2) & 3));
  }
  static __device__ __forceinline__ void put(char* base, int row, int chunk, const Frag<P>& f) {
#pragma unroll
    for (int p = 0; p < P; ++p) *reinterpret_cast<u32x4*>(base + p * PLANE + place(row, chunk)) = f.p[p];
  }
  // operand whose row / column index is the tile's row `row0 + (lane & 31)` and whose slots are columns 16 c + 8 g ..
  static __device__ __forceinline__ Frag<P> rows(const char* base, int row0, int c, int lane) {
    const int row = lane & 31, g = lane >> 5, at = row * ROW + 16 * (g ^ ((row >> 2) & 3));
    Frag<P> f;
#pragma unroll
    for (int p = 0; p < P; ++p)
      f.p[p] = *reinterpret_cast<const u32x4*>(base + (at ^ ((c & 1) * 32)) + p * PLANE + row0 * ROW + (c >> 1) * 64);
    return f;
  }
  // operand whose row / column index is the tile's column col0 + (lane & 31) and whose slots are the 16 rows from row0 in
  // the order of a result's rows.  `last`: first column behind the ones that matter; lanes behind it read a neighbour's
  static __device__ __forceinline__ Frag<P> cols(const char* base, int row0, int col0, int lane, int last) {
    const int i = lane & 15, sub = (lane >> 4) & 1, g = lane >> 5;
    Frag<P> f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        int at;
        if (col0 % 32 == 0 && col0 + 32 <= last) {
          const int lane_at = (4 * g + (i >> 2)) * ROW + 16 * ((2 * sub + ((i & 3) >> 1)) ^ g) + 8 * (i & 1);
          at = (lane_at ^ (u * 32)) + (row0 + 8 * u) * ROW + (col0 >> 5) * 64;
        } else {
          const int col = (col0 + 16 * sub >= last ? col0 : col0 + 16 * sub) + 4 * (i & 3), row = 8 * u + 4 * g + (i >> 2);
          at = row0 * ROW + place(row, col >> 3) + 2 * (col & 7);
        }
        const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(base + p * PLANE + at)));
        f.p[p][2 * u] = w[0];
        f.p[p][2 * u + 1] = w[1];
      }
    }
    return f;
  }
};

// ------------------------------------------------------------------------------------------------ which keys are seen
// Bits of the tile that starts at key 64 t: the mask's and those inside M.  The masks' words of a window of tiles are formed at
// once, kept in LDS, and refilled by the whole workgroup when the loop leaves the window.
constexpr int WINDOW = 128;

struct KeyBits {
  const uint8_t* mask;             // of this sequence, or null
  u64* words;                      // LDS [WINDOW]
  int M, first, end;               // window: tiles [first, first + WINDOW); tiles from `end` on are not asked for

  __device__ __forceinline__ void fill(int t, int wave, int lane) {
    __syncthreads();
    for (int i = wave; i < WINDOW; i += THREADS / 64) {
      const long long key = (long long)(t + i) * TILE + lane;
      const bool on = t + i < end && key < M && mask[key] != 0;
      const u64 w = __ballot(on);
      if (lane == 0) words[i] = w;
    }
    first = t;
    __syncthreads();
  }
  __device__ __forceinline__ u64 inside(int t) const {
    const long long left = (long long)M - (long long)t * TILE;
    return left >= TILE ? ~0ull : (1ull << left) - 1;
  }
  // the first tile from t on that has a seen key (or `end`), and its bits; the same for all waves of the workgroup
  __device__ __forceinline__ int next(int t, u64& bits, int wave, int lane) {
    bits = 0;
    if (mask == nullptr) {
      if (t < end) bits = inside(t);
      return t;
    }
    for (; t < end; ++t) {
      if (t >= first + WINDOW) fill(t, wave, lane);
      const u64 w = words[t - first];
      const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)w), hi = __builtin_amdgcn_readfirstlane((unsigned)(w >> 32));
      bits = ((u64)hi << 32) | lo;
      if (bits != 0) break;
    }
    return t;
  }
  __device__ __forceinline__ void start(int t, int wave, int lane) {
    first = t;
    if (mask != nullptr && t < end) fill(t, wave, lane);
  }
};

// bits of a tile for a query that sees keys up to `last` of it (causal)
__device__ __forceinline__ u64 upto(long long last) { return last >= 63 ? ~0ull : last < 0 ? 0ull : (2ull << last) - 1; }

// the scores of the 32-key half `hh` whose keys are not in `bits` become -inf
__device__ __forceinline__ void hide(f32x16& s, u64 bits, int hh, int g) {
  const unsigned w = (unsigned)(bits >> (32 * hh)) >> (4 * g);
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = (w >> (8 * (r >> 2) + (r & 3))) & 1u ? s[r] : -INFINITY;
}

// P = 2^(c s - m) il: one exponent that holds il too where P is rounded to 16 bits (m - log2(il) is off by 2^-24 of itself), the product
// where it is not
template <class T>
struct Prob {
  static constexpr bool folded = Type<T>::planes == 1;
  float m, f;
  __device__ __forceinline__ Prob() {}
  __device__ __forceinline__ Prob(float mc, float il, float factor) {     // factor: a power of two
    m = folded ? (il == 0.f ? INFINITY : mc - __builtin_amdgcn_logf(il * factor)) : mc;
    f = folded ? 1.f : il * factor;
  }
  __device__ __forceinline__ float operator()(float s, float c) const {
    const float e = __builtin_amdgcn_exp2f(fmaf(s, c, -m));
    return folded ? e : e * f;
  }
  __device__ __forceinline__ bool never() const { return folded ? m == INFINITY : f == 0.f; }   // the query sees no key
};

// ------------------------------------------------------------------------------------------------ staging
// A tile's rows into registers, 8 elements a piece, and from there into LDS: the loads of the next tile are under way while
// this one is used.  Rows whose bit is off and columns from `width` on are zeros, whatever memory holds there.
template <class T, int W, int HEADS, int ROWS = TILE>     // HEADS heads of W / HEADS columns side by side in a row
struct Stage {
  static constexpr int PIECES = W / 8, ALL = ROWS * PIECES, PER = (ALL + THREADS - 1) / THREADS, HW = W / HEADS;
  typedef Tile<W, Type<T>::planes, ROWS> tile;
  Raw<T> raw[PER];
  unsigned at[PER];                                        // byte offset of each piece from the tile's first row
  __device__ __forceinline__ void init(long long row_stride, long long head_stride, int width, int tid) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = tid + j * THREADS, row = i / PIECES, pc = i - row * PIECES;
      const int head = HEADS == 1 ? 0 : pc / (HW / 8), col = (pc - head * (HW / 8)) * 8;
      at[j] = i < ALL && col < width ? (unsigned)((row * row_stride + head * head_stride + col) * (long long)sizeof(T)) : NOWHERE;
    }
  }
  __device__ __forceinline__ void load(const T* first_row, u64 bits, int tid) {
    const Buffer b = buffer(first_row);
    if (bits == ~0ull) {
#pragma unroll
      for (int j = 0; j < PER; ++j) raw[j].load(b, at[j]);
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) raw[j].load(b, ((bits >> ((tid + j * THREADS) / PIECES)) & 1) ? at[j] : NOWHERE);
    }
  }
  __device__ __forceinline__ void put(char* lds, int tid) const {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = tid + j * THREADS, row = i / PIECES, pc = i - row * PIECES;
      if (ALL % THREADS == 0 || i < ALL) tile::put(lds, row, pc, raw[j].frag());
    }
  }
};

// 32 rows as operands in registers: lane & 31 is the row, slots 16 c + 8 g ..
template <class T, int W>
__device__ __forceinline__ void load_rows(Frag<Type<T>::planes> (&f)[W / 16], const T* row, bool on, int width, int g) {
#pragma unroll
  for (int c = 0; c < W / 16; ++c) {
    Raw<T> r;
    const int col = 16 * c + 8 * g;
    if (on && col < width) r.load(row + col);
    else r.clear();
    f[c] = r.frag();
  }
}

// four consecutive values of a row, rounded once
template <class T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
  typedef T t4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<t4*>(p) = __builtin_convertvector((f32x4{a, b, c, d}), t4);
}

// Work index -> place: consecutive workgroups go to the 8 dies in turn, so a die takes a contiguous stretch of the work (the tiles
// of one head, whose keys then stay in that die's L2).
__device__ __forceinline__ unsigned die_major(unsigned id, unsigned total) {
  const unsigned per = total >> 3, rest = total & 7, die = id & 7, at = id >> 3;
  return die * per + (die < rest ? die : rest) + at;
}

// widths that a kernel is built for; the smallest pair that holds (d, dv) is taken
#define SCGG_DIFF_WIDTHS(X) X(32, 32) X(32, 64) X(48, 96) X(64, 64) X(64, 128)

template <class T> int run_forward(const Args& a, hipStream_t st);
template <class T> int run_split(const Args& a, hipStream_t st);
template <class T> int run_backward(const Args& a, hipStream_t st);

}  // namespace diffattn
}  // namespace scgg
