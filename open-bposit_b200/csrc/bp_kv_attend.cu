// bp_kv_attend.cu -- attention of one new token per sequence over the paged
// b-posit key-value cache (bp_paged_attention).
#include <math.h>

#include "bp_kv.cuh"

namespace bp {
namespace {

struct AttendParams {
  KvView c;
  int heads, group;          // query heads, query heads per kv head
  int max_len;
  const void *q;
  int64_t qs;                // batch stride of q, elements
  void *out;
  float *lse;
  float scale;               // of the scores, times log2(e)
  float *raw;                // workspace: lse2 [batch, heads] when scores are accumulated
};

__device__ __forceinline__ float code_value(const KvView &c, const uint8_t *pool, int64_t at) {
  return __uint_as_float(c.fmt == 8 ? posit_to_f32_bits<8, 2>(pool[at])
                                    : bp16_to_f32_bits(reinterpret_cast<const uint16_t *>(pool)[at]));
}

// One block per (sequence, head); its warps take entries in turn, a warp's
// lanes share an entry's dot product, and the warps' running maxima, sums and
// outputs are joined at the end.
template <typename T, int D>
__global__ void __launch_bounds__(128) k_attend_simple(AttendParams p) {
  constexpr int E = D / 32;
  const KvView &c = p.c;
  const int h = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = min(c.length(b), p.max_len), hk = h / p.group;
  __shared__ float s_m[4], s_l[4], s_o[4][D];
  float q[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    q[i] = to_f32(((const T *)p.q)[b * p.qs + h * D + lane * E + i]);
    o[i] = 0.0f;
  }
  bool bad = false;
  for (int i = warp; i < n; i += 4) {
    const int page = c.page_of(b, i);
    if (page < 0) {
      bad = true;
      continue;
    }
    const int64_t row = c.row(page, hk, i);
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < E; ++j) s = fmaf(q[j], code_value(c, c.k, row * D + lane * E + j), s);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
    s *= p.scale;
    if (c.k_exp) s *= exp2_int(c.k_exp[row]);
    const float mn = fmaxf(m, s), a = exp2f(m - mn), w = exp2f(s - mn);
    const float wv = c.v_exp ? w * exp2_int(c.v_exp[row]) : w;
    m = mn;
    l = fmaf(l, a, w);
#pragma unroll
    for (int j = 0; j < E; ++j) o[j] = fmaf(o[j], a, wv * code_value(c, c.v, row * D + lane * E + j));
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int j = 0; j < E; ++j) s_o[warp][lane * E + j] = o[j];
  bad = __syncthreads_or(bad);
  const float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  float den = 0.0f, a[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    a[w] = s_m[w] == -INFINITY && s_l[w] == 0.0f ? 0.0f : exp2f(s_m[w] - top);
    den = fmaf(s_l[w], a[w], den);
  }
  for (int d = threadIdx.x; d < D; d += 128) {
    float x = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) x = fmaf(s_o[w][d], a[w], x);
    x = n == 0 ? 0.0f : x / den;
    if (bad) x = NAN;
    ((T *)p.out)[((int64_t)b * p.heads + h) * D + d] = from_f32<T>(x);
  }
  if (threadIdx.x == 0) {
    const float lse2 = bad ? NAN : (n == 0 ? -INFINITY : top + log2f(den));
    if (p.lse) p.lse[b * p.heads + h] = lse2 * 0.6931471805599453f;
    if (p.raw) p.raw[b * p.heads + h] = lse2;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(128) k_scores_simple(AttendParams p) {
  const KvView &c = p.c;
  const int hk = blockIdx.x, b = blockIdx.y;
  const int n = min(c.length(b), p.max_len);
  if (n == 0 || isnan(p.raw[b * p.heads + hk * p.group])) return;
  for (int i = threadIdx.x; i < n; i += 128) {
    const int page = c.page_of(b, i);
    if (page < 0) continue;
    const int64_t row = c.row(page, hk, i);
    const float ke = c.k_exp ? exp2_int(c.k_exp[row]) : 1.0f;
    float w = 0.0f;
    for (int g = 0; g < p.group; ++g) {
      const T *q = (const T *)p.q + b * p.qs + (hk * p.group + g) * D;
      float s = 0.0f;
      for (int d = 0; d < D; ++d) s = fmaf(to_f32(q[d]), code_value(c, c.k, row * D + d), s);
      w += exp2f(s * p.scale * ke - p.raw[b * p.heads + hk * p.group + g]);
    }
    c.scores[((int64_t)b * c.kv_heads + hk) * c.cap + i] += w;
  }
}

template <typename T, int D>
int launch_attend(const AttendParams &p, cudaStream_t s) {
  k_attend_simple<T, D><<<dim3(p.heads, p.c.batch), 128, 0, s>>>(p);
  int rc = check_launch("k_attend_simple");
  if (rc != kOk || !p.raw) return rc;
  k_scores_simple<T, D><<<dim3(p.c.kv_heads, p.c.batch), 128, 0, s>>>(p);
  return check_launch("k_scores_simple");
}

template <typename T>
int launch_attend_dim(const AttendParams &p, cudaStream_t s) {
  switch (p.c.dim) {
    case 32: return launch_attend<T, 32>(p, s);
    case 64: return launch_attend<T, 64>(p, s);
    case 96: return launch_attend<T, 96>(p, s);
    default: return launch_attend<T, 128>(p, s);
  }
}

size_t workspace_bytes_of(const KvView &c, int heads, int max_len, bool accumulate) {
  return accumulate ? (size_t)c.batch * heads * 4 : 0;
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
  return kOk;
}

}  // namespace
}  // namespace bp

using namespace bp;

extern "C" size_t bp_paged_attention_workspace_size(const bp_kv_cache *cache, int heads, int max_length,
                                                    int accumulate) {
  KvView c;
  int max_len;
  clear_error();
  if (attend_check(cache, 0, heads, max_length, accumulate, "bp_paged_attention_workspace_size", &c, &max_len) != kOk)
    return 0;
  return workspace_bytes_of(c, heads, max_len, accumulate != 0);
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
  if (workspace && ((uintptr_t)workspace & 255u)) return set_error(kEAlign, "%s: workspace not 256-byte aligned", what);
  const size_t need = workspace_bytes_of(p.c, heads, p.max_len, accumulate != 0);
  if (workspace && workspace_bytes < need)
    return set_error(kEWorkspace, "%s: workspace %zu bytes < %zu needed", what, workspace_bytes, need);
  rc = check_device();
  if (rc != kOk) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  void *ws = workspace;
  if (!ws && need) {
    cudaError_t e = cudaMallocAsync(&ws, need, s);
    if (e != cudaSuccess) return set_error(kECuda, "%s: workspace allocation: %s", what, cudaGetErrorString(e));
  }
  p.heads = heads; p.group = heads / cache->kv_heads;
  p.q = q; p.qs = q_stride; p.out = out; p.lse = lse;
  p.scale = scale * 1.4426950408889634f;
  p.raw = accumulate ? (float *)ws : nullptr;
  if (dtype == BP_F32) rc = launch_attend_dim<float>(p, s);
  else if (dtype == BP_BF16) rc = launch_attend_dim<__nv_bfloat16>(p, s);
  else rc = launch_attend_dim<__half>(p, s);
  if (!workspace && ws) {
    cudaError_t f = cudaFreeAsync(ws, s);
    if (rc == kOk && f != cudaSuccess) rc = set_error(kECuda, "%s: workspace free: %s", what, cudaGetErrorString(f));
  }
  return rc;
}
