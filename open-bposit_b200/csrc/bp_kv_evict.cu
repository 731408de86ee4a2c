// bp_kv_evict.cu -- cuts the rows of the paged key-value cache down to their
// best entries, in place (bp_kv_evict).
#include "bp_kv.cuh"

namespace bp {
namespace {

struct EvictParams {
  KvView c;                  // layer 0
  const float *weights;      // [layers, batch, kv_heads, cap]
  int budget, recent, sinks;
  int32_t *keep;             // optional [layers, batch, kv_heads, budget]
};

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kQueue = 2 * kThreads;   // places given up that wait for a mover

// Weights as unsigned integers of the same order: NaN lowest, -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float w, bool guarded) {
  if (guarded) return 0xFF800000u;                     // +inf
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);        // -0 + 0 = +0
  return (u >> 31) ? ~u : u | 0x80000000u;
}

struct Scan {
  int warp_sum[kWarps];
};

// Exclusive prefix count of `flag` over the block's threads; *total: their sum.
__device__ __forceinline__ int block_rank(bool flag, Scan &s, int *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t mask = __ballot_sync(~0u, flag);
  if (lane == 0) s.warp_sum[warp] = __popc(mask);
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const int n = s.warp_sum[w];
    before += w < warp ? n : 0;
    all += n;
  }
  __syncthreads();
  *total = all;
  return before + __popc(mask & ((1u << lane) - 1u));
}

// One block per (layer, sequence, kv head).  A radix select over the ordered
// weights (8 bits a pass) finds the budget-th largest; entries above it are
// kept, and of those equal to it the first ones.  Then two scans run towards
// each other's ends: the front scan (places < budget) queues the places given
// up, the back scan (places >= budget) moves its kept entries into them, both
// in order, so that a chunk's moves never write a place that is still to be
// read: a place is queued only after it was scanned, and movers are read from
// behind the budget, which nothing writes.
__global__ void __launch_bounds__(kThreads) k_kv_evict(EvictParams p) {
  const KvView &c = p.c;
  const int64_t r = blockIdx.x;
  const int hk = (int)(r % c.kv_heads), b = (int)(r / c.kv_heads % c.batch);
  const int layer = (int)(r / c.kv_heads / c.batch);
  const int n = c.length(b), M = p.budget, tid = threadIdx.x;
  int32_t *keep = p.keep ? p.keep + r * M : nullptr;
  if (n <= M) {
    if (keep)
      for (int i = tid; i < M; i += kThreads) keep[i] = i < n ? i : -1;
    return;
  }
  __shared__ Scan scan;
  __shared__ int hist[256], s_bin, s_above, s_front;
  __shared__ int32_t queue[kQueue], src[kThreads], dst[kThreads];
  __shared__ int newest_w[kWarps];
  const float *w = p.weights + r * c.cap;
  int32_t *pos = c.positions + r * c.cap;
  float *scores = c.scores ? c.scores + r * c.cap : nullptr;

  int newest = INT_MIN;
  for (int i = tid; i < n; i += kThreads) newest = max(newest, pos[i]);
  newest = __reduce_max_sync(~0u, newest);
  if ((tid & 31) == 0) newest_w[tid >> 5] = newest;
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) newest = max(newest, newest_w[i]);
  const long long guard = (long long)newest - p.recent;
  auto key_of = [&](int i) { return order_key(w[i], pos[i] < p.sinks || pos[i] > guard); };

  uint32_t prefix = 0;
  int need = M;              // how many of the entries that match the prefix so far are kept
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
      const uint32_t k = key_of(i);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int above = 0, bin = 255;
      while (bin > 0 && above + hist[bin] < need) above += hist[bin--];
      s_bin = bin;
      s_above = above;
    }
    __syncthreads();
    prefix |= (uint32_t)s_bin << shift;
    need -= s_above;
  }
  // entries with key == prefix before place M
  if (tid == 0) s_front = 0;
  __syncthreads();
  int mine = 0;
  for (int i = tid; i < M; i += kThreads) mine += key_of(i) == prefix;
  if (mine) atomicAdd(&s_front, mine);
  __syncthreads();

  int fp = 0, bp = M, ties_f = 0, ties_b = s_front, head = 0, held = 0;
  const int nb = c.fmt / 8, vecs = c.dim * nb / 16;      // 16-byte pieces of one row
  while (bp < n) {
    int total;
    if (held <= kQueue - kThreads && fp < M) {
      const int i = fp + tid;
      const bool in = i < M;
      const uint32_t k = in ? key_of(i) : 0u;
      const bool tie = in && k == prefix;
      const int rank = ties_f + block_rank(tie, scan, &total);
      ties_f += total;
      const bool kept = in && (k > prefix || (tie && rank < need));
      if (kept && keep) keep[i] = i;
      const bool hole = in && !kept;
      const int at = block_rank(hole, scan, &total);
      if (hole) queue[(head + held + at) % kQueue] = i;
      held += total;
      fp += kThreads;
      __syncthreads();
      continue;
    }
    const int i = bp + tid;
    const bool in = i < n;
    const uint32_t k = in ? key_of(i) : 0u;
    const bool tie = in && k == prefix;
    const int rank = ties_b + block_rank(tie, scan, &total);
    ties_b += total;
    const bool kept = in && (k > prefix || (tie && rank < need));
    const int at = block_rank(kept, scan, &total);
    if (kept) {
      src[at] = i;
      dst[at] = queue[(head + at) % kQueue];
    }
    __syncthreads();
    head += total;
    held -= total;
    bp += kThreads;
    const int64_t layer_rows = layer * c.layer_rows;
    for (int j = tid; j < total * 2 * vecs; j += kThreads) {
      const int e = j / (2 * vecs), piece = j % (2 * vecs);
      const int pf = c.page_of(b, src[e]), pt = c.page_of(b, dst[e]);
      if (pf < 0 || pt < 0) continue;
      const int64_t from = layer_rows + c.row(pf, hk, src[e]), to = layer_rows + c.row(pt, hk, dst[e]);
      uint8_t *pool = piece < vecs ? c.k : c.v;
      const int x = piece < vecs ? piece : piece - vecs;
      reinterpret_cast<uint4 *>(pool)[to * vecs + x] = reinterpret_cast<const uint4 *>(pool)[from * vecs + x];
      if (x == 0 && c.k_exp) {
        int8_t *ex = piece < vecs ? c.k_exp : c.v_exp;
        ex[to] = ex[from];
      }
    }
    if (tid < total) {
      pos[dst[tid]] = pos[src[tid]];
      if (scores) scores[dst[tid]] = scores[src[tid]];
      if (keep) keep[dst[tid]] = src[tid];
    }
    __syncthreads();
  }
  // front places behind the last one scanned: the back scan found no more movers, all are kept
  if (keep)
    for (int i = fp + tid; i < M; i += kThreads) keep[i] = i;
}

}  // namespace
}  // namespace bp

using namespace bp;

extern "C" int bp_kv_evict(const bp_kv_cache *cache, const float *weights, int budget, int recent, int sinks,
                           int32_t *keep, void *stream) {
  static const char *const what = "bp_kv_evict";
  clear_error();
  EvictParams p{};
  int rc = kv_check(cache, 0, what, &p.c);
  if (rc != kOk) return rc;
  if (budget < 1 || recent < 0 || sinks < 0)
    return set_error(kEInval, "%s: budget must be positive, recent and sinks not negative", what);
  if (!cache->positions || (!weights && !cache->scores))
    return set_error(kEInval, "%s: the cache keeps no positions, or there are no weights", what);
  const int64_t rows = (int64_t)cache->layers * cache->batch * cache->kv_heads;
  if (rows > 0x7FFFFFFF) return set_error(kERange, "%s: too many rows", what);
  if (rows == 0) return kOk;
  rc = check_device();
  if (rc != kOk) return rc;
  p.weights = weights ? weights : cache->scores;
  p.budget = budget; p.recent = recent; p.sinks = sinks; p.keep = keep;
  k_kv_evict<<<(unsigned)rows, kThreads, 0, (cudaStream_t)stream>>>(p);
  return check_launch("k_kv_evict");
}
