// Differential attention: entry points, checks, workspaces and the sum for the gradient of lambda.  The kernels are in
// diff_attention_fwd.h and diff_attention_bwd.h, compiled per element type.
#include "diff_attention.h"

namespace scgg {
namespace diffattn {
namespace {

constexpr int SPLIT_MIN_TILES = 4;     // keys of a split workgroup at least: 4 tiles of 64
constexpr int SPLIT_GROUPS = 1024;     // workgroups that keep the memory busy: 4 on each of 256 CUs (512, 1024, 2048, 4096: one query x 32768 keys
                                       // of 16 x 4 key heads 202, 208, 206, 225 us; 65536 keys of 4 x 4 109, 108, 114, 137)

// dlambda[h] = - sum over sequences and queries of delta_2, in a fixed order: 256 lanes, each a stretch, then a tree
__global__ __launch_bounds__(256) void dlambda_kernel(const float* __restrict__ delta, float* __restrict__ out, int B, int H, int N) {
  __shared__ float red[4];
  const int h = blockIdx.x;
  float v = 0.f;
  for (int b = 0; b < B; ++b) {
    const float* d = delta + (((long long)b * H + h) * 3 + 1) * N;
    for (int n = threadIdx.x; n < N; n += 256) v += d[n];
  }
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0) out[h] = -((red[0] + red[1]) + (red[2] + red[3]));
}

int check_workspace(size_t need, const void* workspace, size_t bytes, const char* what) {
  if (need == 0) return 0;
  if (!workspace || bytes < need) return fail("%s: workspace of %zu bytes, %zu are needed", what, workspace ? bytes : (size_t)0, need);
  if (reinterpret_cast<uintptr_t>(workspace) & 255) return fail("%s: workspace has to be aligned to 256 bytes", what);
  return 0;
}

int check(const scgg_diff_attention_args* p, const char* what) {
  if (!p) return fail("%s: null argument", what);
  if (p->dtype != SCGG_F32 && p->dtype != SCGG_BF16 && p->dtype != SCGG_F16) return fail("%s: unknown dtype %d", what, p->dtype);
  if (p->B < 0 || p->N < 0 || p->M < 0) return fail("%s: bad shape", what);
  if (p->H < 1 || p->Hkv < 1 || p->H % p->Hkv != 0) return fail("%s: %d heads on %d key heads", what, p->H, p->Hkv);
  if (p->d < 8 || p->dv < 8 || p->d % 8 != 0 || p->dv % 8 != 0 || p->d > 64 || p->dv > 128)
    return fail("%s: d = %d, dv = %d: multiples of 8 with d <= 64 and dv <= 128 are supported", what, p->d, p->dv);
  if (!(p->scale > 0.f) || !isfinite(p->scale * 1.44269504088896340736f)) return fail("%s: scale has to be positive and, times log2(e), finite", what);
  if (p->N > 0x7fffffff - 256 || p->M > 0x7fffffff - 256) return fail("%s: too many tokens", what);
  if ((long long)p->B * p->H > 0x7fffffff || (long long)p->B * p->N * p->H > 0x7fffffffLL * 32) return fail("%s: too many rows", what);
  return 0;
}

bool aligned16(const void* base) { return (reinterpret_cast<uintptr_t>(base) & 15) == 0; }

bool aligned(const scgg_diff_attention_args* p, const void* base, int64_t sb, int64_t sn, int64_t sh) {
  const int64_t size = p->dtype == SCGG_F32 ? 4 : 2;
  return ((reinterpret_cast<uintptr_t>(base) | (uintptr_t)((sb | sn | sh) * size)) & 15) == 0;
}

// a tile's rows lie within the 2 GiB that a 32-bit offset reaches
bool near(const scgg_diff_attention_args* p, int64_t sn, int64_t sh, int width) {
  const int64_t size = p->dtype == SCGG_F32 ? 4 : 2;
  return sn >= 0 && sh >= 0 && sn < (1ll << 40) && sh < (1ll << 40) && ((TILE - 1) * sn + sh + width) * size < 0x7fffffffll - 16;
}

int check_inputs(const scgg_diff_attention_args* p, const char* what) {
  const bool queries = p->B > 0 && p->N > 0, keys = p->B > 0 && p->M > 0;
  if ((queries && !p->q) || (keys && (!p->k || !p->v)) || !p->lambda) return fail("%s: null argument", what);
  if ((queries && !aligned(p, p->q, p->q_stride_b, p->q_stride_n, p->q_stride_h)) ||
      (keys && (!aligned(p, p->k, p->k_stride_b, p->k_stride_n, p->k_stride_h) || !aligned(p, p->v, p->v_stride_b, p->v_stride_n, p->v_stride_h))))
    return fail("%s: bases and strides of q, k and v have to be multiples of 16 bytes", what);
  if ((queries && !near(p, p->q_stride_n, p->q_stride_h, p->d)) || (keys && (!near(p, p->k_stride_n, p->k_stride_h, p->d) || !near(p, p->v_stride_n, 0, p->dv))))
    return fail("%s: rows of q, k and v have to lie less than 2 GiB / 64 apart", what);
  return 0;
}

Args make(const scgg_diff_attention_args* p) {
  Args a = {};
  a.q = p->q; a.k = p->k; a.v = p->v; a.dout = p->dout; a.lambda = p->lambda; a.mask = p->key_mask;
  a.out = p->out; a.dq = p->dq; a.dk = p->dk; a.dv = p->dv_out; a.stats = reinterpret_cast<float2*>(p->stats);
  a.qb = p->q_stride_b; a.qn = p->q_stride_n; a.qh = p->q_stride_h;
  a.kb = p->k_stride_b; a.kn = p->k_stride_n; a.kh = p->k_stride_h;
  a.vb = p->v_stride_b; a.vn = p->v_stride_n; a.vh = p->v_stride_h;
  a.gb = p->dout_stride_b; a.gn = p->dout_stride_n; a.gh = p->dout_stride_h; a.mb = p->mask_stride_b;
  a.scale = p->scale; a.c = p->scale * 1.44269504088896340736f;
  a.B = p->B; a.N = p->N; a.M = p->M; a.H = p->H; a.Hkv = p->Hkv; a.d = p->d; a.dv_w = p->dv; a.causal = p->causal != 0;
  return a;
}

// Keys split over workgroups (0: not): for up to 32 rows of a key head, and where the queries give the other kernel, one long chain of tiles on a part of
// the CUs, few workgroups (of 64).  The split kernel does more work per tile and its join costs by the row, so the more workgroups, the more keys it
// takes: up to 4 workgroups per tile of keys, and 160.  us a call not split / split, 8 heads, d = 64, dv = 128, bf16: 10 tiles, 32 workgroups 28 / 26, 64
// 28 / 32; 16 tiles, 64 41 / 35, 96 41 / 48, 120 41 / 55; 32 tiles, 128 73 / 72, 160 73 / 82; 64 tiles, 128 139 / 102, 160 139 / 121, 192 139 / 135;
// 256 tiles, 160 533 / 346.  One query of 16 heads on 4 x 64 x 2048 keys 279 / 55; 60 queries x 8000 keys 260 / 25.  Causal grids too, though the
// split kernel walks the tiles that the mask hides: 2 heads of 4096 147 / 102 (fp32 427 / 313), 4 of 2048 78 / 74 (fp32 220 / 186).
void plan_split(Args& a) {
  const long long rows = (long long)a.N * (a.H / a.Hkv), tiles = (a.M + TILE - 1) / TILE, blocks = (long long)a.B * a.Hkv * ((rows + 31) / 32);
  const long long others = (long long)a.B * a.H * (((long long)a.N + 63) / 64), most = tiles < 40 ? 4 * tiles : 160;
  a.splits = 0;
  if ((rows > 32 && others > most) || tiles < 2 * SPLIT_MIN_TILES || blocks == 0) return;
  long long s = SPLIT_GROUPS / blocks;
  if (s > tiles / SPLIT_MIN_TILES) s = tiles / SPLIT_MIN_TILES;
  if (s < 1) s = 1;
  a.split_tiles = (int)((tiles + s - 1) / s);
  a.splits = (int)((tiles + a.split_tiles - 1) / a.split_tiles);
}

size_t part_bytes(const Args& a) {
  return a.splits == 0 ? 0 : (size_t)a.B * a.H * a.N * 2 * a.splits * (2 * a.dv_w + 4) * sizeof(float);
}
// Queries split over workgroups in the dK / dV kernel: where the keys alone give fewer than two workgroups to each CU, and there are tiles to
// split.  Each split writes its sums in 32 bits and they are read again, so there are four at most.  Training pass with 1, 2, 4, 8 splits allowed:
// 4096 causal, 8 heads on 4, 1053, 711, 551, 550 us; not causal 1172, 838, 756, 756; 16 heads of 2048 433, 413, 412, 414.
void plan_dkv(Args& a) {
  const long long blocks = (long long)a.B * a.Hkv * ((a.M + 127) / 128), tiles = (long long)((a.N + TILE - 1) / TILE) * (a.H / a.Hkv);
  long long s = blocks > 0 ? 512 / blocks : 1;
  if (s > 4) s = 4;
  if (s > tiles / 4) s = tiles / 4;
  a.splits = s < 1 ? 1 : (int)s;
}
// Keys split over workgroups in the dQ kernel, where the queries (64 to a workgroup) fill about half of the GPU or less.  The splits' dQ and the
// sweeps' second launch cost about as much as eight tiles.  Training pass, not split / split, 8 heads: 128 workgroups, 16 tiles, fp32, d = 64 417 / 346 us (bf16
// 177 / 180), 64 tiles, bf16 386 / 297; 160 workgroups, 16 tiles, fp32 440 / 464, 32 tiles 836 / 754 (bf16 256 / 227).  Causal grids of up to two workgroups
// per CU are split in two: all of them run at once, so the longest is the time, and halving it is worth the join (4096 causal, 8 heads on 4, training pass:
// 575 -> 551 us; not causal it would cost 757 -> 780).
void plan_dq(Args& a) {
  const long long blocks = (long long)a.B * a.H * (((long long)a.N + 63) / 64), tiles = (a.M + TILE - 1) / TILE;
  long long s = blocks == 0 ? 1 : blocks <= (tiles < 32 ? 128 : 160) ? 512 / blocks : a.causal && blocks <= 512 ? 2 : 1;
  if (s > 16) s = 16;
  if (s > tiles / 8) s = tiles / 8;
  a.dq_splits = s < 1 ? 1 : (int)s;
}
size_t dq_part_bytes(const Args& a) {
  return a.dq_splits <= 1 ? 0 : (size_t)a.dq_splits * a.B * a.H * a.N * 2 * a.d * sizeof(float);
}
size_t dkv_part_bytes(const Args& a) {
  return a.splits <= 1 ? 0 : (size_t)a.splits * a.B * a.M * a.Hkv * (2 * a.d + a.dv_w) * sizeof(float);
}
size_t delta_bytes(const Args& a) { return ((size_t)a.B * a.H * 3 * a.N * sizeof(float) + 255) / 256 * 256; }

// the deltas, and the splits' parts of one kernel after the other
size_t backward_bytes(Args& a) {
  plan_dq(a);
  plan_dkv(a);
  const size_t q = dq_part_bytes(a), kv = dkv_part_bytes(a);
  return delta_bytes(a) + (q > kv ? q : kv);
}

int done(int rc, const char* what) {
  if (rc == -3) return fail("%s: too many tokens for one launch", what);
  if (rc != 0) return fail("%s: the kernel's shared memory could not be set up", what);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail("%s: %s", what, hipGetErrorString(e));
}

}  // namespace
}  // namespace diffattn
}  // namespace scgg

using namespace scgg;
using namespace scgg::diffattn;

extern "C" size_t scgg_diff_attention_forward_workspace_bytes(const scgg_diff_attention_args* p) {
  if (check(p, "diff_attention_forward_workspace_bytes")) return 0;
  Args a = make(p);
  plan_split(a);
  return part_bytes(a);
}

extern "C" size_t scgg_diff_attention_backward_workspace_bytes(const scgg_diff_attention_args* p) {
  if (check(p, "diff_attention_backward_workspace_bytes")) return 0;
  Args a = make(p);
  return backward_bytes(a);
}

extern "C" int scgg_diff_attention_forward(const scgg_diff_attention_args* p, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "diff_attention_forward";
  if (check(p, what) || check_inputs(p, what)) return -1;
  if (p->B == 0 || p->N == 0) return 0;
  if (!p->out) return fail("%s: null output", what);
  if (!aligned16(p->out) || !aligned16(p->stats)) return fail("%s: out and stats have to be aligned to 16 bytes", what);
  Args a = make(p);
  plan_split(a);
  const size_t need = part_bytes(a);
  if (check_workspace(need, workspace, workspace_bytes, what)) return -1;
  a.part = static_cast<float*>(workspace);
  hipStream_t st = static_cast<hipStream_t>(stream);
  int rc;
  if (a.splits > 0) rc = p->dtype == SCGG_F32 ? run_split<float>(a, st) : p->dtype == SCGG_BF16 ? run_split<__bf16>(a, st) : run_split<_Float16>(a, st);
  else rc = p->dtype == SCGG_F32 ? run_forward<float>(a, st) : p->dtype == SCGG_BF16 ? run_forward<__bf16>(a, st) : run_forward<_Float16>(a, st);
  return done(rc, what);
}

extern "C" int scgg_diff_attention_backward(const scgg_diff_attention_args* p, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "diff_attention_backward";
  if (check(p, what) || check_inputs(p, what)) return -1;
  const bool queries = p->B > 0 && p->N > 0, keys = p->B > 0 && p->M > 0;
  if ((queries && (!p->dout || !p->dq || !p->stats)) || (keys && (!p->dk || !p->dv_out)) || !p->dlambda) return fail("%s: null argument", what);
  if (queries && !aligned(p, p->dout, p->dout_stride_b, p->dout_stride_n, p->dout_stride_h))
    return fail("%s: base and strides of dout have to be multiples of 16 bytes", what);
  if (queries && !near(p, p->dout_stride_n, 0, p->dv)) return fail("%s: rows of dout have to lie less than 2 GiB / 64 apart", what);
  if (!aligned16(p->dq) || !aligned16(p->dk) || !aligned16(p->dv_out) || !aligned16(p->stats))
    return fail("%s: dq, dk, dv_out and stats have to be aligned to 16 bytes", what);
  Args a = make(p);
  const size_t need = backward_bytes(a);
  if (check_workspace(need, workspace, workspace_bytes, what)) return -1;
  a.delta = static_cast<float*>(workspace);
  a.part = workspace ? reinterpret_cast<float*>(static_cast<char*>(workspace) + delta_bytes(a)) : nullptr;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int rc = p->dtype == SCGG_F32 ? run_backward<float>(a, st) : p->dtype == SCGG_BF16 ? run_backward<__bf16>(a, st) : run_backward<_Float16>(a, st);
  if (rc == 0) hipLaunchKernelGGL(dlambda_kernel, dim3((unsigned)p->H), dim3(256), 0, st, a.delta, p->dlambda, p->B, p->H, p->N);
  return done(rc, what);
}
