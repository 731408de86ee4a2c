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

constexpr int kThreads = 1024, kWarps = kThreads / 32;  // of the streaming form
constexpr int kBatch = 4;              // entries that one of its threads reads at once
constexpr int kQueue = 2 * kThreads;   // places given up that wait for a mover
constexpr int kBins = 2048;            // of a histogram of weights
constexpr uint32_t kTop = 0xFF800000u; // order_key of +inf

// Weights as unsigned integers of the same order: NaN lowest, -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float w, bool guarded) {
  if (guarded) return kTop;
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);        // -0 + 0 = +0
  return (u >> 31) ? ~u : u | 0x80000000u;
}

// The bin of `hist`, from the top down, in which the count passes `need`:
// found = {bin, entries in bins above it, entries in it}.
template <int NT>
__device__ __forceinline__ void find_bin(const int *hist, int need, int *warp_sum, uint32_t *found) {
  constexpr int PER = kBins / NT;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int bin[PER], mine = 0;
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    bin[q] = hist[kBins - 1 - (tid * PER + q)];
    mine += bin[q];
  }
  int incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(~0u, incl, d);
    if (lane >= d) incl += y;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int above = incl - mine + __reduce_add_sync(~0u, lane < warp ? warp_sum[lane] : 0);
  if (above < need && above + mine >= need) {
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      if (above < need && above + bin[q] >= need) {
        found[0] = kBins - 1 - (tid * PER + q);
        found[1] = above;
        found[2] = bin[q];
        break;
      }
      above += bin[q];
    }
  }
  __syncthreads();
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
  static_assert(kWarps == 32, "a warp's sum per lane");
  const int n = s.warp_sum[lane], before = __reduce_add_sync(~0u, lane < warp ? n : 0);
  *total = __reduce_add_sync(~0u, n);
  __syncthreads();
  return before + __popc(mask & ((1u << lane) - 1u));
}

// Moves `moves` entries of a row from places src to places dst, NT at a time: a
// thread per entry looks up the pages and moves exponents, position and score,
// then all threads copy the codes, 16 bytes each, several on their way at once.
// 192 rows of 8192 64-wide bp8 entries cut to 2048, about 1500 entries moved in
// each: 37 us, 27 of them for the moves, whose scattered 32-byte sectors are 120
// MB (43 us when each of an entry's threads looked up its pages).
constexpr uint32_t kNone = ~0u;        // row of an entry whose page is outside the pool; pools have fewer rows
template <int NT, typename Index>
__device__ __forceinline__ void move_entries(const EvictParams &p, int64_t r, int b, int hk, int64_t layer_rows,
                                             const Index *src, const Index *dst, int moves, uint2 *rows) {
  const KvView &c = p.c;
  const int tid = threadIdx.x, vecs = c.dim * (c.fmt / 8) / 16, per = 2 * vecs;
  const int first = tid / per, piece = tid - first * per, step = NT / per;
  const bool value = piece >= vecs;
  uint4 *pool = reinterpret_cast<uint4 *>(value ? c.v : c.k) + layer_rows * vecs + (value ? piece - vecs : piece);
  int8_t *ke = c.k_exp + layer_rows, *ve = c.v_exp + layer_rows;
  int32_t *pos = c.positions + r * c.cap;
  float *scores = c.scores ? c.scores + r * c.cap : nullptr;
  int32_t *keep = p.keep ? p.keep + r * p.budget : nullptr;
  for (int base = 0; base < moves; base += NT) {
    if (base + tid < moves) {
      const int s = src[base + tid], d = dst[base + tid];
      const int pf = c.page_of(b, s), pt = c.page_of(b, d), ps = pos[s];
      const float score = scores ? scores[s] : 0.0f;
      uint2 row = make_uint2(kNone, kNone);
      if (pf >= 0 && pt >= 0) {
        row = make_uint2((uint32_t)c.row(pf, hk, s), (uint32_t)c.row(pt, hk, d));
        if (c.fmt == 8) {
          const int8_t x = ke[row.x], y = ve[row.x];
          ke[row.y] = x;
          ve[row.y] = y;
        }
      }
      pos[d] = ps;
      if (scores) scores[d] = score;
      if (keep) keep[d] = s;
      rows[tid] = row;
    }
    __syncthreads();
    const int n = min(NT, moves - base);
    if (first < step)
      for (int e = first; e < n; e += 4 * step) {
        uint4 code[4];
        uint2 row[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          row[j] = e + j * step < n ? rows[e + j * step] : make_uint2(kNone, kNone);
          if (row[j].y != kNone) code[j] = pool[(int64_t)row[j].x * vecs];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (row[j].y != kNone) pool[(int64_t)row[j].y * vecs] = code[j];
      }
    __syncthreads();
  }
}

// One block per (layer, sequence, kv head) with all its weights in registers,
// thread t holding entries t, t + NT, ...  What bounds it is latency: the loads
// of lengths, weights and positions, then block barriers, then the moves; so
// the passes are few and work on registers.
//  * The budget-th largest weight: a histogram of 2048 bins over the range that
//    the weights have (+inf apart), then over the bin that holds it, until the
//    bin is one value or all of it is kept -- two or three passes.
//  * Kept entries behind the budget go, in order, to the places in front that
//    were given up: every (chunk of NT entries, warp) counts both kinds by
//    ballot, one scan of the counts gives everyone's rank.
template <int NT, int KPT>
__global__ void __launch_bounds__(NT) k_kv_evict_row(EvictParams p) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int NW = NT / 32, E = NW * KPT;
  const KvView &c = p.c;
  const int r = blockIdx.x;
  const int hk = r % c.kv_heads, lb = r / c.kv_heads, b = lb % c.batch, layer = lb / c.batch;
  const int n = c.length(b), M = p.budget, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int32_t *keep = p.keep ? p.keep + (int64_t)r * M : nullptr;
  if (n <= M) {
    if (keep)
      for (int i = tid; i < M; i += NT) keep[i] = i < n ? i : -1;
    return;
  }
  __shared__ __align__(8) int hist[kBins];          // and then the rows of entries that move
  static_assert(NT * 8 <= kBins * 4, "a pair of rows per thread");
  __shared__ int count[E + 1], warp_sum[32];
  __shared__ uint32_t red[3][32], found[3];
  __shared__ uint16_t src[NT * KPT / 2], dst[NT * KPT / 2];
  const float *w = p.weights + (int64_t)r * c.cap;
  const int32_t *pos = c.positions + (int64_t)r * c.cap;

  uint32_t key[KPT];
  {
    float wv[KPT];
    int ps[KPT], newest = INT_MIN;
#pragma unroll
    for (int j = 0; j < KPT; ++j) {
      const int i = j * NT + tid;
      wv[j] = i < n ? w[i] : 0.0f;
      ps[j] = i < n ? pos[i] : INT_MIN;
    }
#pragma unroll
    for (int j = 0; j < KPT; ++j) newest = max(newest, ps[j]);
    newest = __reduce_max_sync(~0u, newest);
    if (lane == 0) warp_sum[warp] = newest;
    __syncthreads();
    newest = __reduce_max_sync(~0u, lane < NW ? warp_sum[lane] : INT_MIN);
    const long long guard = (long long)newest - p.recent;
#pragma unroll
    for (int j = 0; j < KPT; ++j) key[j] = order_key(wv[j], ps[j] < p.sinks || ps[j] > guard);
  }
  auto in = [&](int j) { return j * NT + tid < n; };

  // ---- thr, with the entries kept: key > thr, and `need` of those with key == thr (all of them if !ties) ----
  uint32_t thr = kTop, lo = ~0u, hi = 0;
  int need = M, top = 0;
#pragma unroll
  for (int j = 0; j < KPT; ++j)
    if (in(j)) {
      if (key[j] == kTop) ++top;
      else {
        lo = min(lo, key[j]);
        hi = max(hi, key[j]);
      }
    }
  top = __reduce_add_sync(~0u, top);
  lo = __reduce_min_sync(~0u, lo);
  hi = __reduce_max_sync(~0u, hi);
  if (lane == 0) {
    red[0][warp] = top;
    red[1][warp] = lo;
    red[2][warp] = hi;
  }
  __syncthreads();
  top = __reduce_add_sync(~0u, lane < NW ? red[0][lane] : 0u);
  lo = __reduce_min_sync(~0u, lane < NW ? red[1][lane] : ~0u);
  hi = __reduce_max_sync(~0u, lane < NW ? red[2][lane] : 0u);
  bool ties = top > M;
  if (top < M) {
    need = M - top;
    while (true) {
      const int shift = max(0, 32 - __clz(hi - lo) - 11);
      for (int i = tid; i < kBins; i += NT) hist[i] = 0;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < KPT; ++j)
        if (in(j) && key[j] >= lo && key[j] <= hi) atomicAdd(&hist[(key[j] - lo) >> shift], 1);
      __syncthreads();
      find_bin<NT>(hist, need, warp_sum, found);
      need -= (int)found[1];
      const int held = (int)found[2];
      const uint32_t width = (1u << shift) - 1u;
      lo += found[0] << shift;
      hi = hi - lo < width ? hi : lo + width;
      if (shift == 0 || held == need) {
        thr = lo;
        ties = held > need;
        break;
      }
    }
  }
  // exclusive ranks of flagged entries in entry order, from the counts per (chunk, warp) in `count`; returns the total
  auto scan_counts = [&]() {
    __syncthreads();
    const int mine = tid < E ? count[tid] : 0;
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(~0u, incl, d);
      if (lane >= d) incl += y;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    const int base = __reduce_add_sync(~0u, lane < warp ? warp_sum[lane] : 0);
    if (tid < E) count[tid] = base + incl - mine;
    if (tid == NT - 1) count[E] = base + incl;
    __syncthreads();
  };
  static_assert(E <= NT, "a count per thread");
  uint32_t kept = 0;
#pragma unroll
  for (int j = 0; j < KPT; ++j)
    if (in(j) && (ties ? key[j] > thr : key[j] >= thr)) kept |= 1u << j;
  const uint32_t below = (1u << lane) - 1u;
  if (ties) {                // the first `need` of the entries at the threshold
#pragma unroll
    for (int j = 0; j < KPT; ++j) {
      const uint32_t m = __ballot_sync(~0u, in(j) && key[j] == thr);
      if (lane == 0) count[j * NW + warp] = __popc(m);
    }
    scan_counts();
#pragma unroll
    for (int j = 0; j < KPT; ++j) {
      const bool tie = in(j) && key[j] == thr;
      const uint32_t m = __ballot_sync(~0u, tie);
      if (tie && count[j * NW + warp] + __popc(m & below) < need) kept |= 1u << j;
    }
    __syncthreads();
  }
  // holes in the low half of a count, movers in the high half: fewer than 2^15 of each
#pragma unroll
  for (int j = 0; j < KPT; ++j) {
    const int i = j * NT + tid;
    const bool k = kept >> j & 1;
    const uint32_t holes = __ballot_sync(~0u, i < M && !k), movers = __ballot_sync(~0u, i >= M && k);
    if (lane == 0) count[j * NW + warp] = __popc(holes) | __popc(movers) << 16;
  }
  scan_counts();
#pragma unroll
  for (int j = 0; j < KPT; ++j) {
    const int i = j * NT + tid;
    const bool k = kept >> j & 1;
    const uint32_t holes = __ballot_sync(~0u, i < M && !k), movers = __ballot_sync(~0u, i >= M && k);
    const int at = count[j * NW + warp];
    if (i < M && !k) dst[(at & 0xFFFF) + __popc(holes & below)] = (uint16_t)i;
    if (i >= M && k) src[(at >> 16) + __popc(movers & below)] = (uint16_t)i;
    if (i < M && k && keep) keep[i] = i;
  }
  __syncthreads();
  move_entries<NT>(p, r, b, hk, layer * c.layer_rows, src, dst, count[E] >> 16, reinterpret_cast<uint2 *>(hist));
}

// The same for rows that do not fit a block's registers: the weights are read
// once per pass.  A radix select over the ordered weights (11, 11 and 10 bits) finds
// the budget-th largest.  Then two scans run towards each other's ends: the front
// scan (places < budget) queues the places given up, the back scan (places >=
// budget) moves its kept entries into them, both in order, so that a chunk's
// moves never write a place that is still to be read: a place is queued only
// after it was scanned, and movers are read from behind the budget, which nothing
// writes.
__global__ void __launch_bounds__(kThreads) k_kv_evict_long(EvictParams p) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
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
  __shared__ __align__(8) int hist[kBins];          // and then the rows of entries that move
  __shared__ int warp_sum[kWarps], s_front;
  __shared__ uint32_t found[3];
  __shared__ int32_t queue[kQueue], src[kThreads], dst[kThreads];
  const float *w = p.weights + r * c.cap;
  const int32_t *pos = c.positions + r * c.cap;

  int newest = INT_MIN;
#pragma unroll 4
  for (int i = tid; i < n; i += kThreads) newest = max(newest, pos[i]);
  newest = __reduce_max_sync(~0u, newest);
  if ((tid & 31) == 0) warp_sum[tid >> 5] = newest;
  __syncthreads();
  newest = __reduce_max_sync(~0u, warp_sum[tid & 31]);
  const long long guard = (long long)newest - p.recent;
  auto key_of = [&](int i) { return order_key(w[i], pos[i] < p.sinks || pos[i] > guard); };
  // each(i, key) for this thread's entries below `end`, kBatch loads in flight
  auto for_keys = [&](int end, auto each) {
    for (int i = tid; i < end; i += kBatch * kThreads) {
      uint32_t k[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) k[j] = i + j * kThreads < end ? key_of(i + j * kThreads) : 0u;
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i + j * kThreads < end) each(k[j]);
    }
  };

  uint32_t prefix = 0;
  int need = M;              // how many of the entries that match the prefix so far are kept
  for (int shift = 21; shift >= 0; shift = shift > 10 ? shift - 11 : shift - 10) {
    for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
    __syncthreads();
    const int width = shift ? 11 : 10;
    const uint32_t above = shift == 21 ? 0u : ~0u << (shift + width), bins = (1u << width) - 1u;
    for_keys(n, [&](uint32_t k) {
      if (((k ^ prefix) & above) == 0) atomicAdd(&hist[(k >> shift) & bins], 1);
    });
    __syncthreads();
    find_bin<kThreads>(hist, need, warp_sum, found);
    prefix |= found[0] << shift;
    need -= (int)found[1];
  }
  // entries with key == prefix before place M
  if (tid == 0) s_front = 0;
  __syncthreads();
  int mine = 0;
  for_keys(M, [&](uint32_t k) { mine += k == prefix; });
  if (mine) atomicAdd(&s_front, mine);
  __syncthreads();

  int fp = 0, bp = M, ties_f = 0, ties_b = s_front, head = 0, held = 0;
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
    move_entries<kThreads>(p, r, b, hk, layer * c.layer_rows, src, dst, total, reinterpret_cast<uint2 *>(hist));
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
  cudaStream_t s = (cudaStream_t)stream;
  const dim3 grid((unsigned)rows);
  // The smallest block that holds a row's weights in its registers; longer rows stream them.  us for 384 rows (one row)
  // of 64-wide bp8 heads cut by half, at each limit and in the next larger form, where few entries move:
  //   1024: 4.1 (2.8) and 7.4 (3.5)     2048: 7.8 (3.7) and 15.5 (6.6)     8192: 19.3 (7.1) and 34.9 (11.0)
  //   16384: 36.8 (11.4) and 89.8 (28.2); streamed, 32768: 202 (52)
  // A quarter of the entries moved as well, in the form that is taken:
  //   1024: 14.5 (6.3)     2048: 26.9 (8.0)     8192: 79 (19.5)     16384: 156 (32)     32768: 563 (120)
  static const char *const name = "k_kv_evict";
  if (p.c.cap <= 256 * 4) return launch_early(k_kv_evict_row<256, 4>, grid, 256, 0, s, name, p);
  if (p.c.cap <= 512 * 4) return launch_early(k_kv_evict_row<512, 4>, grid, 512, 0, s, name, p);
  if (p.c.cap <= 512 * 16) return launch_early(k_kv_evict_row<512, 16>, grid, 512, 0, s, name, p);
  if (p.c.cap <= 1024 * 16) return launch_early(k_kv_evict_row<1024, 16>, grid, 1024, 0, s, name, p);
  return launch_early(k_kv_evict_long, grid, kThreads, 0, s, name, p);
}
