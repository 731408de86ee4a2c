// bp_kv_attend.cu -- attention of one new token per sequence over the paged
// b-posit key-value cache (bp_paged_attention): the entry points, and the kernel
// that finishes what k_kv_attend (bp_kv_attend.cuh) leaves in parts.
#include <math.h>

#include "bp_kv_attend.cuh"

namespace bp {
namespace {

constexpr int kJoinParts = 256;     // CTAs of one launch, at most
constexpr int kJoinWarps = 4, kJoinBatch = 8;   // warps of a block, parts that a warp loads at once

// Joins the parts of a row that several CTAs of k_kv_attend worked on: block
// (c, h) takes head h of the row that starts in CTA c's range and goes on behind
// it.  Every warp reads all parts' statistics (a lane every 32nd, all at once) and
// sums the outputs of every fourth part, eight in flight together, so that a row
// of 74 parts (131071 entries of one sequence) waits for memory five times.
// Launched early (programmatic dependent launch), its start hides behind the
// main kernel.
template <typename T>
__device__ __forceinline__ void join_row(const AttendParams &p, int cta, int h) {
  __shared__ float sums[kJoinWarps][128];
  const int2 open = p.cta_row[cta];
  if (open.x < 0) return;
  const int D = p.c.dim, rec = kHeadsPerRow * D, parts = open.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t head = head_of(p, row_id(p, open.x), h);
  // the first part is the CTA's second record (a row that starts there), the others are first records
  const float *base = p.cta_rec + cta * 2 * (rec + 16) + lane;
  auto part = [&](int k) { return base + (k ? k * 2 : 1) * (rec + 16); };
  float m[kJoinParts / 32], l[kJoinParts / 32], M = -INFINITY, L = 0.0f;
#pragma unroll
  for (int i = 0; i < kJoinParts / 32; ++i) {
    const int k = min(i * 32 + lane, parts - 1);       // (past the last part: the last one again, with weight 0)
    m[i] = i * 32 < parts ? part(k)[rec + h - lane] : -INFINITY;
    l[i] = i * 32 < parts ? part(k)[rec + 8 + h - lane] : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < kJoinParts / 32; ++i) M = fmaxf(M, m[i]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, d));
  const float at = finite_max(M);
#pragma unroll
  for (int i = 0; i < kJoinParts / 32; ++i) {
    m[i] = i * 32 + lane < parts ? ex2(m[i] - at) : 0.0f;      // the part's weight from here on
    L = i * 32 + lane < parts ? fmaf(l[i], m[i], L) : L;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) L += __shfl_xor_sync(~0u, L, d);
  float O[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < kJoinParts / 32; ++i) {
    if (i * 32 >= parts) break;
    float x[kJoinBatch][4];
#pragma unroll
    for (int j = 0; j < kJoinBatch; ++j) {
      const float *r = part(min(i * 32 + j * kJoinWarps + warp, parts - 1)) + h * D;
#pragma unroll
      for (int y = 0; y < 4; ++y) x[j][y] = y * 32 < D ? r[y * 32] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < kJoinBatch; ++j) {
      const float f = __shfl_sync(~0u, m[i], j * kJoinWarps + warp);
#pragma unroll
      for (int y = 0; y < 4; ++y) O[y] = i * 32 + j * kJoinWarps + warp < parts ? fmaf(x[j][y], f, O[y]) : O[y];
    }
  }
  static_assert(kJoinWarps * kJoinBatch == 32, "32 parts a round");
#pragma unroll
  for (int y = 0; y < 4; ++y) sums[warp][y * 32 + lane] = O[y];
  __syncthreads();
  // (the score blocks beside this one work the logarithm out for themselves)
  if (threadIdx.x == 0 && p.lse && head >= 0) p.lse[head] = (M + log2f(L)) * 0.6931471805599453f;
  const int d = threadIdx.x;
  if (head >= 0 && d < D)
    ((T *)p.out)[head * D + d] = from_f32<T>(((sums[0][d] + sums[1][d]) + (sums[2][d] + sums[3][d])) / L);
}

// scores[b, hk, i] += sum over the query heads of kv head hk of 2^(raw - lse2),
// for kScoreEntries entries: one thread per entry, so the sum has one order and
// needs no atomics.  A row that k_kv_attend left in parts has its logarithms
// worked out here from the parts' statistics, a head per warp in turn.
constexpr int kScoreEntries = 256;
__device__ __forceinline__ void add_scores(const AttendParams &p, int bk, int chunk) {
  __shared__ float lse[kHeadsPerRow];
  const int b = bk / p.c.kv_heads, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = min(p.c.length(b), p.max_len), first = chunk * kScoreEntries;
  if (first >= n) return;
  constexpr int PER = kScoreEntries / (kJoinWarps * 32);
  float w[PER] = {};
  bool lost = false;
  for (int ch = 0; ch < p.chunks; ++ch) {
    const int row = bk * p.chunks + ch, heads = min(kHeadsPerRow, p.group - ch * kHeadsPerRow);
    const int2 at = p.row_parts[row];
    for (int h = warp; h < heads; h += kJoinWarps) {
      float y;
      if (at.y == 0) {
        y = p.lse2[(int64_t)row * kHeadsPerRow + h];
      } else {
        const int rec = kHeadsPerRow * p.c.dim;
        const float *base = p.cta_rec + at.x * 2 * (rec + 16) + rec + h;
        float M = -INFINITY, L = 0.0f;
        for (int k = lane; k < at.y; k += 32) M = fmaxf(M, base[(k ? k * 2 : 1) * (rec + 16)]);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, d));
        const float from = finite_max(M);
        for (int k = lane; k < at.y; k += 32) {
          const float *r = base + (k ? k * 2 : 1) * (rec + 16);
          L = fmaf(r[8], ex2(r[0] - from), L);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) L += __shfl_xor_sync(~0u, L, d);
        y = M + log2f(L);
      }
      if (lane == 0) lse[h] = y;
    }
    __syncthreads();
    // (NaN: a page outside the pool, or a query that is not finite; -inf: every score is.  Either way the softmax is
    // NaN and the kv head keeps its scores)
    for (int h = 0; h < heads; ++h) lost = lost || !(lse[h] > -INFINITY);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = first + j * kJoinWarps * 32 + threadIdx.x;
      if (i < n) {
        const float *raw = p.raw + ((int64_t)row * p.max_len + i) * p.gp;
        for (int h = 0; h < heads; h += 2) {
          const float2 s = *reinterpret_cast<const float2 *>(raw + h);
          w[j] += ex2(s.x - lse[h]);
          if (h + 1 < heads) w[j] += ex2(s.y - lse[h + 1]);
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = first + j * kJoinWarps * 32 + threadIdx.x;
    if (i < n && !lost) p.c.scores[(int64_t)bk * p.c.cap + i] += w[j];
  }
}

// What is left after k_kv_attend: `joins` blocks join rows, the others add scores.
template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) k_kv_finish(AttendParams p, int joins, int chunks) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int i = blockIdx.x;
  if (i < joins) join_row<T>(p, i / kHeadsPerRow, i % kHeadsPerRow);
  else add_scores(p, (i - joins) / chunks, (i - joins) % chunks);
}

// CTAs of the main kernel: one per SM.
int attend_grid() {
  const int n = sm_count();
  return n < kJoinParts ? n : kJoinParts;
}

// Workspace layout; every part starts on 256 bytes.
struct Layout {
  size_t warp_rec, cta_rec, cta_row, lse2, row_parts, raw, bytes;
};
Layout layout_of(const KvView &c, int heads, int max_len, bool accumulate, int grid) {
  const int group = heads / c.kv_heads, chunks = (group + kHeadsPerRow - 1) / kHeadsPerRow;
  const int64_t rows = (int64_t)c.batch * c.kv_heads * chunks;
  const size_t rec = (size_t)kHeadsPerRow * c.dim;
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  Layout l;
  l.warp_rec = 0;
  l.cta_rec = up((size_t)grid * kMaxWarps * rec * 4);
  l.cta_row = l.cta_rec + up((size_t)grid * 2 * (rec + 16) * 4);
  l.lse2 = l.cta_row + up((size_t)grid * sizeof(int2));
  l.row_parts = l.lse2 + (accumulate ? up(rows * kHeadsPerRow * 4) : 0);
  l.raw = l.row_parts + (accumulate ? up(rows * sizeof(int2)) : 0);
  l.bytes = l.raw + (accumulate ? up((size_t)rows * max_len * raw_heads(group) * 4) : 0);
  return l;
}

int attend_check(const bp_kv_cache *cache, int layer, int heads, int max_length, int accumulate, const char *what,
                 KvView *c, int *max_len) {
  int rc = kv_check(cache, layer, what, c);
  if (rc != kOk) return rc;
  if (heads < 1 || heads > 65536 || heads % cache->kv_heads)
    return set_error(kEInval, "%s: %d heads do not divide over %d kv heads", what, heads, cache->kv_heads);
  if (max_length < 0) return set_error(kEInval, "%s: negative max_length", what);
  if (accumulate && !cache->scores) return set_error(kEInval, "%s: the cache keeps no scores", what);
  *max_len = max_length && max_length < c->cap ? max_length : c->cap;
  const int64_t rows = (int64_t)cache->batch * cache->kv_heads * ((heads / cache->kv_heads + 7) / 8);
  if (rows * ((*max_len + 15) / 16 + kRowUnits) > 0x7FFFFF00 ||
      (accumulate && (int64_t)cache->batch * cache->kv_heads * ((*max_len + 255) / 256) > 0x7FFF0000))
    return set_error(kERange, "%s: more work than the call can number", what);
  return kOk;
}

}  // namespace
}  // namespace bp

using namespace bp;

extern "C" size_t bp_paged_attention_workspace_size(const bp_kv_cache *cache, int heads, int max_length,
                                                    int accumulate) {
  KvView c;
  int max_len = 0;
  clear_error();
  if (attend_check(cache, 0, heads, max_length, accumulate, "bp_paged_attention_workspace_size", &c, &max_len) != kOk)
    return 0;
  return layout_of(c, heads, max_len, accumulate != 0, attend_grid()).bytes;
}

extern "C" int bp_paged_attention(const bp_kv_cache *cache, int layer, int dtype, int heads, const void *q,
                                  int64_t q_stride, void *out, float *lse, float scale, int max_length,
                                  int accumulate, void *workspace, size_t workspace_bytes, void *stream) {
  static const char *const what = "bp_paged_attention";
  clear_error();
  AttendParams p{};
  int rc = attend_check(cache, layer, heads, max_length, accumulate, what, &p.c, &p.max_len);
  if (rc != kOk) return rc;
  if (dtype < BP_F32 || dtype > BP_F16) return set_error(kEFmt, "%s: unknown dtype %d", what, dtype);
  if (cache->batch == 0) return kOk;
  if (!q || !out) return set_error(kEInval, "%s: null pointer", what);
  const int per = dtype == BP_F32 ? 4 : 8;
  if (q_stride < (int64_t)heads * cache->head_dim)
    return set_error(kEInval, "%s: the batch stride of q is smaller than its rows", what);
  if (!aligned16(q) || !aligned16(out) || q_stride % per)
    return set_error(kEAlign, "%s: pointers and strides must be multiples of 16 bytes", what);
  if (crosses(q, q_stride, out, cache->batch, (int64_t)heads * cache->head_dim, 16 / per))
    return set_error(kEInval, "%s: out lies on q, but not row for row", what);
  if (workspace && ((uintptr_t)workspace & 255u)) return set_error(kEAlign, "%s: workspace not 256-byte aligned", what);
  rc = check_device();
  const int grid = attend_grid();
  const Layout l = layout_of(p.c, heads, p.max_len, accumulate != 0, grid);
  if (workspace && workspace_bytes < l.bytes)
    return set_error(kEWorkspace, "%s: workspace %zu bytes < %zu needed", what, workspace_bytes, l.bytes);
  if (rc != kOk) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  void *ws = workspace;
  if (!ws) {
    cudaError_t e = cudaMallocAsync(&ws, l.bytes, s);
    if (e != cudaSuccess) return set_error(kECuda, "%s: workspace allocation: %s", what, cudaGetErrorString(e));
  }
  uint8_t *base = (uint8_t *)ws;
  p.heads = heads; p.group = heads / cache->kv_heads;
  p.chunks = (p.group + kHeadsPerRow - 1) / kHeadsPerRow;
  p.q = q; p.qs = q_stride; p.out = out; p.lse = lse;
  p.scale = scale * 1.4426950408889634f;
  p.warp_rec = (float *)(base + l.warp_rec);
  p.cta_rec = (float *)(base + l.cta_rec);
  p.cta_row = (int2 *)(base + l.cta_row);
  p.lse2 = accumulate ? (float *)(base + l.lse2) : nullptr;
  p.row_parts = accumulate ? (int2 *)(base + l.row_parts) : nullptr;
  p.raw = accumulate ? (float *)(base + l.raw) : nullptr;
  p.gp = raw_heads(p.group);
  rc = p.c.fmt == 8 ? launch_kv_attend8(p, dtype, grid, s) : launch_kv_attend16(p, dtype, grid, s);
  // (a batch of at most kOneCta units is one CTA's, and no row of it is in parts)
  const int64_t units = (int64_t)cache->batch * cache->kv_heads * p.chunks * ((p.max_len + 15) / 16 + kRowUnits);
  const int joins = units > kOneCta ? grid * kHeadsPerRow : 0;
  const int chunks = accumulate ? (p.max_len + kScoreEntries - 1) / kScoreEntries : 0;
  const int64_t blocks = joins + (int64_t)chunks * cache->batch * cache->kv_heads;
  if (rc == kOk && blocks) {
    const dim3 g((unsigned)blocks);
    const auto kernel = dtype == BP_F32 ? k_kv_finish<float>
                                        : (dtype == BP_BF16 ? k_kv_finish<__nv_bfloat16> : k_kv_finish<__half>);
    rc = launch_early(kernel, g, kJoinWarps * 32, 0, s, "k_kv_finish", p, joins, chunks);
  }
  if (!workspace) {
    cudaError_t f = cudaFreeAsync(ws, s);
    if (rc == kOk && f != cudaSuccess) rc = set_error(kECuda, "%s: workspace free: %s", what, cudaGetErrorString(f));
  }
  return rc;
}
