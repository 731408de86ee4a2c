// bp_kv_append.cu -- writes new tokens into the paged key-value cache
// (bp_kv_append) and holds the argument checks that the cache's calls share.
#include <math.h>

#include "bp_kv.cuh"

namespace bp {

int kv_check(const bp_kv_cache *c, int layer, const char *what, KvView *view) {
  if (!c) return set_error(kEInval, "%s: null cache", what);
  if (c->fmt != 8 && c->fmt != 16) return set_error(kEFmt, "%s: fmt must be 8 or 16 (got %d)", what, c->fmt);
  if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 96 && c->head_dim != 128)
    return set_error(kERange, "%s: head_dim must be 32, 64, 96 or 128 (got %d)", what, c->head_dim);
  if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)))
    return set_error(kERange, "%s: page_size must be a power of two from 16 to 1024 (got %d)", what, c->page_size);
  if (c->layers < 1 || c->kv_heads < 1 || c->pages < 0 || c->batch < 0 || c->max_pages < 0)
    return set_error(kEInval, "%s: bad cache sizes", what);
  if (layer < 0 || layer >= c->layers)
    return set_error(kEInval, "%s: layer %d outside [0, %d)", what, layer, c->layers);
  if (c->batch > 2048) return set_error(kERange, "%s: batch of at most 2048 sequences (got %d)", what, c->batch);
  if (c->kv_heads > 1024) return set_error(kERange, "%s: at most 1024 kv heads (got %d)", what, c->kv_heads);
  if ((int64_t)c->max_pages * c->page_size > (1 << 30))
    return set_error(kERange, "%s: capacity of at most 2^30 entries", what);
  if ((int64_t)c->pages * c->kv_heads >= 0xFFFFFFF0LL / c->page_size)
    return set_error(kERange, "%s: 2^32 or more rows in a layer of the pools", what);
  if (c->pages && (!c->k || !c->v)) return set_error(kEInval, "%s: null pool", what);
  if ((c->batch && !c->lengths) || (c->batch && c->max_pages && !c->page_table))
    return set_error(kEInval, "%s: null page table or lengths", what);
  if (c->fmt == 8 ? c->pages && (!c->k_exp || !c->v_exp) : c->k_exp || c->v_exp)
    return set_error(kEInval, "%s: fmt 8 needs both exponent arrays, fmt 16 takes none", what);
  if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_exp) || !aligned16(c->v_exp))
    return set_error(kEAlign, "%s: pools must be 16-byte aligned", what);
  KvView w{};
  w.fmt = c->fmt; w.layers = c->layers; w.pages = c->pages; w.kv_heads = c->kv_heads; w.dim = c->head_dim;
  w.batch = c->batch; w.max_pages = c->max_pages; w.cap = c->max_pages * c->page_size;
  while ((1 << w.page_shift) < c->page_size) ++w.page_shift;
  w.layer_rows = (int64_t)c->pages * c->kv_heads * c->page_size;
  const int64_t bytes = w.layer_rows * c->head_dim * (c->fmt / 8);
  w.k = (uint8_t *)c->k + layer * bytes;
  w.v = (uint8_t *)c->v + layer * bytes;
  w.k_exp = c->k_exp ? c->k_exp + layer * w.layer_rows : nullptr;
  w.v_exp = c->v_exp ? c->v_exp + layer * w.layer_rows : nullptr;
  w.table = c->page_table; w.lengths = c->lengths;
  const int64_t track = (int64_t)layer * c->batch * c->kv_heads * w.cap;
  w.positions = c->positions ? c->positions + track : nullptr;
  w.scores = c->scores ? c->scores + track : nullptr;
  *view = w;
  return kOk;
}

namespace {

struct AppendParams {
  KvView c;
  int tokens, heads, rope_rows;
  int q_warps;               // warps of one token that take queries; the others take keys and values
  const void *k, *v, *q;
  int64_t ks, vs, qs;        // token strides, elements
  const float *cos, *sin;
  const int32_t *positions, *seqs, *places;
  void *q_out;
};

constexpr int kAppendThreads = 128;

// Four consecutive activations as fp32.
__device__ __forceinline__ void load4(const float *p, float *x) {
  const float4 f = *reinterpret_cast<const float4 *>(p);
  x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
}
template <typename T>
__device__ __forceinline__ void load4(const T *p, float *x) {
  const uint2 w = *reinterpret_cast<const uint2 *>(p);
  T t[4];
  memcpy(t, &w, 8);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = to_f32(t[i]);
}
__device__ __forceinline__ void store4(float *p, const float *x) {
  *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
template <typename T>
__device__ __forceinline__ void store4(T *p, const float *x) {
  T t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = from_f32<T>(x[i]);
  uint2 w;
  memcpy(&w, t, 8);
  *reinterpret_cast<uint2 *>(p) = w;
}

// Codes of eight values of a row (bp8: of x / 2^e), four to a word or two.
__device__ __noinline__ void encode_any(const float *x, int e, int fmt, uint32_t *o) {
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = __float_as_uint(x[i]);
    if (fmt == 8) o[i >> 2] |= bp8_encode_exp(u, e) << 8 * (i & 3);
    else o[i >> 1] |= bp16_encode_bits(u, true) << 16 * (i & 1);
  }
}
template <int FMT>
__device__ __forceinline__ void encode8(const float (&x)[8], int e, uint32_t (&o)[FMT / 4]) {
  bool easy = true;
  uint32_t m[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = __float_as_uint(x[i]) & 0x7FFFFFFFu;
    const uint32_t V = FMT == 8 ? a - ((uint32_t)e << 23) : a;
    // (a bound on `a` too: subtracting e from an exponent of zero could wrap into the range)
    easy = easy && (FMT == 8 ? bp8_in_range(V) && a - 0x00800000u < 0x7F000000u : bp16_in_range(V));
    m[i] = FMT == 8 ? bp8_encode_near(V) : bp16_encode_near(V);
    m[i] = __float_as_uint(x[i]) >> 31 ? 0u - m[i] : m[i];
  }
  if (FMT == 8) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      o[i] = __byte_perm(__byte_perm(m[4 * i], m[4 * i + 1], 0x0040), __byte_perm(m[4 * i + 2], m[4 * i + 3], 0x0040), 0x5410);
  } else {
#pragma unroll
    for (int i = 0; i < FMT / 4; ++i) o[i] = __byte_perm(m[(2 * i) & 7], m[(2 * i + 1) & 7], 0x5410);
  }
  if (!easy) {             // zeros, very small values, infinities, NaN
    float y[8];
    uint32_t w[FMT / 4];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i];
#pragma unroll
    for (int i = 0; i < FMT / 4; ++i) w[i] = 0;
    encode_any(y, e, FMT, w);
#pragma unroll
    for (int i = 0; i < FMT / 4; ++i) o[i] = w[i];
  }
}

// Rows of keys or values that a group takes at a time, with U rows of queries: two where there are many tokens (16384
// fp32 tokens of 32 and 8 heads of 128 into bp16: 122 us, 6.0 TB/s, against 133 with one; 20001 bf16 tokens of 9 and 3
// heads of 64 into bp16: 26.3 against 28.0, where rotation and encoding take 60% of the issue slots).
constexpr int kv_unroll(int U) { return U > 1 ? 2 : 1; }

// A warp works on rows of one token, either keys and values or queries (a row is
// a head): a group of GW lanes takes a row, a lane four pairs (i, i + D/2) of it,
// so that loads and stores are 16 bytes (fp32) and a row's maximum is a shuffle
// within the group.  Keys are rotated in float64: both products are exact there,
// so the result is the exact sum rounded to float64 and then to fp32 whatever
// the order of evaluation, and the codes that are stored do not depend on it.
// Queries are rotated in fp32 (a product and an fma): converting all their values
// to float64 and back took the conversion unit longer than the memory needs for
// them.  With many tokens a group takes U rows of queries (two of keys or values)
// at a time, all loaded before the first is worked on.
template <typename T, int D, int FMT, int U>
__global__ void __launch_bounds__(kAppendThreads) k_kv_append(AppendParams p) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int GL = D / 8, GW = GL <= 4 ? 4 : (GL <= 8 ? 8 : 16), RPW = 32 / GW, KU = kv_unroll(U);
  const KvView &c = p.c;
  const int t = blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, sub = lane & (GW - 1), grp = lane / GW;
  if (t >= p.tokens) return;
  const bool on = sub < GL, queries = (int)blockIdx.y < p.q_warps;
  const int chunk = queries ? blockIdx.y : blockIdx.y - p.q_warps;
  const int kv_rows = 2 * c.kv_heads;
  int b = t, place;
  if (p.places) {
    b = p.seqs[t];
    place = p.places[t];
  } else {
    place = max(c.lengths[t], 0) - 1;      // not cut to the capacity: a token behind it is dropped
  }
  const int at = p.positions ? p.positions[t] : place;
  const int r0 = chunk * RPW * (queries ? U : KU) + grp;
  const bool turn = p.cos && (queries || r0 < c.kv_heads);      // some row is rotated: r0 is, if any
  float cs[4], sn[4];
  auto angles = [&]() {
    const bool known = (unsigned)at < (unsigned)p.rope_rows;
#pragma unroll
    for (int i = 0; i < 4; ++i) cs[i] = sn[i] = NAN;
    if (known && on) {
      load4(p.cos + (int64_t)at * (D / 2) + sub * 4, cs);
      load4(p.sin + (int64_t)at * (D / 2) + sub * 4, sn);
    }
  };

  if (queries) {
    float x[U][8];
    const T *src = (const T *)p.q + t * p.qs + r0 * D + sub * 4;
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (on && r0 + i * RPW < p.heads) {
        load4(src + i * RPW * D, x[i]);
        load4(src + i * RPW * D + D / 2, x[i] + 4);
      }
    angles();
    T *dst = (T *)p.q_out + ((int64_t)t * p.heads + r0) * D + sub * 4;
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (on && r0 + i * RPW < p.heads) {
        float y[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          y[j] = __fmaf_rn(x[i][j], cs[j], -__fmul_rn(x[i][4 + j], sn[j]));
          y[4 + j] = __fmaf_rn(x[i][4 + j], cs[j], __fmul_rn(x[i][j], sn[j]));
        }
        store4(dst + i * RPW * D, y);
        store4(dst + i * RPW * D + D / 2, y + 4);
      }
    return;
  }
  float x[KU][8];
#pragma unroll
  for (int k = 0; k < KU; ++k) {
    const int r = r0 + k * RPW;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[k][i] = 0.0f;
    const T *src = r < c.kv_heads ? (const T *)p.k + t * p.ks + r * D : (const T *)p.v + t * p.vs + (r - c.kv_heads) * D;
    if (on && r < kv_rows) {
      load4(src + sub * 4, x[k]);
      load4(src + sub * 4 + D / 2, x[k] + 4);
    }
  }
  if (turn) angles();
  const bool placed = on && (unsigned)b < (unsigned)c.batch && (unsigned)place < (unsigned)c.cap;
  const int page = placed ? c.page_of(b, place) : -1;
#pragma unroll
  for (int k = 0; k < KU; ++k) {
    const int r = r0 + k * RPW;
    const bool key = r < c.kv_heads;
    if (key && p.cos) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const double u = x[k][i], w = x[k][4 + i], cc = cs[i], ss = sn[i];
        x[k][i] = (float)__fma_rn(u, cc, -__dmul_rn(w, ss));
        x[k][4 + i] = (float)__fma_rn(w, cc, __dmul_rn(u, ss));
      }
    }
    int e = 0;
    if (FMT == 8) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t a = __float_as_uint(x[k][i]) & 0x7FFFFFFFu;
        top = a < 0x7F800000u && a > top ? a : top;
      }
#pragma unroll
      for (int d = GW / 2; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(~0u, top, d));
      e = top ? max(f32_floor_log2(top) - 3, -126) : 0;
    }
    if (page < 0 || r >= kv_rows) continue;
    const int h = key ? r : r - c.kv_heads;
    const int64_t row = c.row(page, h, place);
    uint8_t *pool = (key ? c.k : c.v) + row * (D * FMT / 8);
    uint32_t o[FMT / 4];
    encode8<FMT>(x[k], e, o);
    if (FMT == 8) {
      reinterpret_cast<uint32_t *>(pool)[sub] = o[0];
      reinterpret_cast<uint32_t *>(pool)[D / 8 + sub] = o[1];
      if (sub == 0) (key ? c.k_exp : c.v_exp)[row] = (int8_t)e;
    } else {
      reinterpret_cast<uint2 *>(pool)[sub] = make_uint2(o[0], o[1]);
      reinterpret_cast<uint2 *>(pool)[D / 8 + sub] = make_uint2(o[FMT / 4 - 2], o[FMT / 4 - 1]);
    }
    if (key && sub == 0) {
      const int64_t i = ((int64_t)b * c.kv_heads + h) * c.cap + place;
      if (c.positions) c.positions[i] = at;
      if (c.scores) c.scores[i] = 0.0f;
    }
  }
}

template <typename T, int D, int FMT>
int launch_append(AppendParams p, cudaStream_t s) {
  constexpr int GL = D / 8, GW = GL <= 4 ? 4 : (GL <= 8 ? 8 : 16), RPW = 32 / GW, U = 4;
  const int heads = p.q ? p.heads : 0;
  const unsigned blocks = (p.tokens + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
  // A group of lanes rotates one row of queries while there are few, so that they spread over the SMs, and U rows on
  // from there, which reads a token's angles once for all of them: 256 tokens of 32 heads of 128 take 3.3 us against
  // 4.2 with U rows, 4096 bf16 tokens of 14 heads of 64 take 8.4 against 6.6; 1024 to 2048 tokens are within 15%.
  // Without queries a group takes one row however many tokens there are (16384 fp32 tokens of 8 heads of 128 into bp16:
  // 46 us; 8192 tokens of 2 heads of 64 into bp8: 5.9).
  const bool few = (int64_t)p.tokens * ((heads + RPW - 1) / RPW) < (int64_t)sm_count() * 48;
  const int rows = few ? RPW : RPW * U;
  p.q_warps = (heads + rows - 1) / rows;
  const int kv = RPW * (few ? 1 : kv_unroll(U));
  const dim3 grid(blocks, p.q_warps + (2 * p.c.kv_heads + kv - 1) / kv);
  return few ? launch_early(k_kv_append<T, D, FMT, 1>, grid, kAppendThreads, 0, s, "k_kv_append", p)
             : launch_early(k_kv_append<T, D, FMT, U>, grid, kAppendThreads, 0, s, "k_kv_append", p);
}

template <typename T, int FMT>
int launch_append_dim(const AppendParams &p, cudaStream_t s) {
  switch (p.c.dim) {
    case 32: return launch_append<T, 32, FMT>(p, s);
    case 64: return launch_append<T, 64, FMT>(p, s);
    case 96: return launch_append<T, 96, FMT>(p, s);
    default: return launch_append<T, 128, FMT>(p, s);
  }
}
template <typename T>
int launch_append_fmt(const AppendParams &p, cudaStream_t s) {
  return p.c.fmt == 8 ? launch_append_dim<T, 8>(p, s) : launch_append_dim<T, 16>(p, s);
}

}  // namespace
}  // namespace bp

using namespace bp;

extern "C" int bp_kv_append(const bp_kv_cache *cache, int layer, int dtype, int tokens, const void *k,
                            int64_t k_stride, const void *v, int64_t v_stride, const void *q, int heads,
                            int64_t q_stride, const float *cos, const float *sin, int rope_rows,
                            const int32_t *positions, const int32_t *seqs, const int32_t *places, void *q_out,
                            void *stream) {
  static const char *const what = "bp_kv_append";
  clear_error();
  AppendParams p{};
  int rc = kv_check(cache, layer, what, &p.c);
  if (rc != kOk) return rc;
  if (dtype < BP_F32 || dtype > BP_F16) return set_error(kEFmt, "%s: unknown dtype %d", what, dtype);
  if (tokens < 0 || (q && heads < 1) || heads > 65536) return set_error(kEInval, "%s: bad token or head count", what);
  if (!seqs != !places) return set_error(kEInval, "%s: seqs and places come together", what);
  if (!places && tokens && tokens != cache->batch)   // (no tokens: the lists are null too)
    return set_error(kEInval, "%s: %d tokens for %d sequences (give seqs and places)", what, tokens, cache->batch);
  if (!cos != !sin || (cos && rope_rows < 1) || (q && !cos))
    return set_error(kEInval, "%s: q and the rotation need both tables", what);
  if (tokens == 0) return kOk;
  if (!k || !v || (q && !q_out)) return set_error(kEInval, "%s: null pointer", what);
  const int es = dtype == BP_F32 ? 4 : 2, per = 16 / es;
  const int64_t kvw = (int64_t)cache->kv_heads * cache->head_dim, qw = (int64_t)heads * cache->head_dim;
  if (k_stride < kvw || v_stride < kvw || (q && q_stride < qw))
    return set_error(kEInval, "%s: a token stride is smaller than its rows", what);
  if (!aligned16(k) || !aligned16(v) || !aligned16(q) || !aligned16(q_out) || k_stride % per || v_stride % per ||
      (q && q_stride % per))
    return set_error(kEAlign, "%s: pointers and strides must be multiples of 16 bytes", what);
  if (q && crosses(q, q_stride, q_out, tokens, qw, es))
    return set_error(kEInval, "%s: q_out lies on q, but not row for row", what);
  if (!aligned16(cos) || !aligned16(sin)) return set_error(kEAlign, "%s: tables must be 16-byte aligned", what);
  rc = check_device();
  if (rc != kOk) return rc;
  p.tokens = tokens; p.heads = heads; p.rope_rows = rope_rows;
  p.k = k; p.v = v; p.q = q; p.ks = k_stride; p.vs = v_stride; p.qs = q_stride;
  p.cos = cos; p.sin = sin; p.positions = positions; p.seqs = seqs; p.places = places; p.q_out = q_out;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == BP_F32) return launch_append_fmt<float>(p, s);
  if (dtype == BP_BF16) return launch_append_fmt<__nv_bfloat16>(p, s);
  return launch_append_fmt<__half>(p, s);
}
