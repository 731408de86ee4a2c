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

// A warp works on one token: groups of GW lanes take its rows (a head of k, v or
// q) in turn, a lane four pairs (i, i + D/2) of a row, so that loads and stores
// are 16 bytes (fp32) and a row's maximum is a shuffle within the group.  The
// rotation is in float64: both products are exact there, so the result is the
// exact sum rounded to float64 and then to fp32 whatever the order of
// evaluation; the table's row is converted once per token.  The next row is
// loaded while one is worked on.  gridDim.y warps share a token when there are
// few tokens.
template <typename T, int D, int FMT>
__global__ void __launch_bounds__(kAppendThreads) k_kv_append(AppendParams p) {
  constexpr int GL = D / 8, GW = GL <= 4 ? 4 : (GL <= 8 ? 8 : 16), RPW = 32 / GW;
  const KvView &c = p.c;
  const int rows = 2 * c.kv_heads + (p.q ? p.heads : 0);
  const int t = blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, sub = lane & (GW - 1);
  if (t >= p.tokens) return;
  const int step = gridDim.y * RPW, first = blockIdx.y * RPW + lane / GW;

  auto load = [&](int r, float *x) {     // row r of the token: k, v, then q heads
    const T *src = r < c.kv_heads       ? (const T *)p.k + t * p.ks + r * D
                   : r < 2 * c.kv_heads ? (const T *)p.v + t * p.vs + (r - c.kv_heads) * D
                                        : (const T *)p.q + t * p.qs + (r - 2 * c.kv_heads) * D;
    src += sub * 4;
    load4(src, x);
    load4(src + D / 2, x + 4);
  };
  float x[8], y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = y[i] = 0.0f;
  if (first < rows && sub < GL) load(first, x);
  int b = t, place;
  if (p.places) {
    b = p.seqs[t];
    place = p.places[t];
  } else {
    place = c.length(t) - 1;
  }
  const int at = p.positions ? p.positions[t] : place;
  double cc[4], ss[4];
  if (p.cos) {
    const bool known = (unsigned)at < (unsigned)p.rope_rows;
    float cs[4] = {NAN, NAN, NAN, NAN}, sn[4] = {NAN, NAN, NAN, NAN};
    if (known && sub < GL) {
      load4(p.cos + (int64_t)at * (D / 2) + sub * 4, cs);
      load4(p.sin + (int64_t)at * (D / 2) + sub * 4, sn);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      cc[i] = cs[i];
      ss[i] = sn[i];
    }
  }
  int page = -1;
  if ((unsigned)b < (unsigned)c.batch && (unsigned)place < (unsigned)c.cap) page = c.page_of(b, place);

  // (whole warps stay in the loop for the shuffles: a group without a row of its own has `on` false)
  for (int r = first; r - lane / GW < rows; r += step) {
    const bool on = r < rows && sub < GL;
    if (r + step < rows && sub < GL) load(r + step, y);
    const int part = r < c.kv_heads ? 0 : (r < 2 * c.kv_heads ? 1 : 2);
    if (part != 1 && p.cos) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const double u = x[i], w = x[4 + i];
        x[i] = (float)__fma_rn(u, cc[i], -__dmul_rn(w, ss[i]));
        x[4 + i] = (float)__fma_rn(w, cc[i], __dmul_rn(u, ss[i]));
      }
    }
    if (part == 2) {
      if (on) {
        T *dst = (T *)p.q_out + ((int64_t)t * p.heads + r - 2 * c.kv_heads) * D + sub * 4;
        store4(dst, x);
        store4(dst + D / 2, x + 4);
      }
    }
    if (__any_sync(~0u, part != 2)) {
      int e = 0;
      if (FMT == 8) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t a = __float_as_uint(x[i]) & 0x7FFFFFFFu;
          top = a < 0x7F800000u && a > top ? a : top;
        }
#pragma unroll
        for (int d = GW / 2; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(~0u, top, d));
        e = top ? max(f32_floor_log2(top) - 3, -126) : 0;
      }
      if (on && part != 2 && page >= 0) {
        const int h = part == 0 ? r : r - c.kv_heads;
        const int64_t row = c.row(page, h, place);
        uint8_t *pool = part == 0 ? c.k : c.v;
        if (FMT == 8) {
          uint32_t lo = 0, hi = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            lo |= bp8_encode_exp(__float_as_uint(x[i]), e) << (8 * i);
            hi |= bp8_encode_exp(__float_as_uint(x[4 + i]), e) << (8 * i);
          }
          *reinterpret_cast<uint32_t *>(pool + row * D + sub * 4) = lo;
          *reinterpret_cast<uint32_t *>(pool + row * D + D / 2 + sub * 4) = hi;
          if (sub == 0) (part == 0 ? c.k_exp : c.v_exp)[row] = (int8_t)e;
        } else {
          uint32_t o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            o[i] = bp16_encode_rtne(__float_as_uint(x[2 * i])) |
                   (bp16_encode_rtne(__float_as_uint(x[2 * i + 1])) << 16);
          uint16_t *dst = (uint16_t *)pool + row * D + sub * 4;
          *reinterpret_cast<uint2 *>(dst) = make_uint2(o[0], o[1]);
          *reinterpret_cast<uint2 *>(dst + D / 2) = make_uint2(o[2], o[3]);
        }
        if (part == 0 && sub == 0) {
          const int64_t i = ((int64_t)b * c.kv_heads + h) * c.cap + place;
          if (c.positions) c.positions[i] = at;
          if (c.scores) c.scores[i] = 0.0f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = y[i];
  }
}

template <typename T, int D>
int launch_append(const AppendParams &p, cudaStream_t s) {
  constexpr int GL = D / 8, GW = GL <= 4 ? 4 : (GL <= 8 ? 8 : 16), RPW = 32 / GW;
  const int rows = 2 * p.c.kv_heads + (p.q ? p.heads : 0);
  const unsigned blocks = (p.tokens + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
  // one warp a token once that fills the GPU (16 warps an SM); below, as many as the token has rows for
  const int most = (rows + RPW - 1) / RPW;
  int share = (int)(((int64_t)sm_count() * 16 + p.tokens - 1) / p.tokens);
  share = share < most ? share : most;
  const dim3 grid(blocks, share);
  if (p.c.fmt == 8) k_kv_append<T, D, 8><<<grid, kAppendThreads, 0, s>>>(p);
  else k_kv_append<T, D, 16><<<grid, kAppendThreads, 0, s>>>(p);
  return check_launch("k_kv_append");
}

template <typename T>
int launch_append_dim(const AppendParams &p, cudaStream_t s) {
  switch (p.c.dim) {
    case 32: return launch_append<T, 32>(p, s);
    case 64: return launch_append<T, 64>(p, s);
    case 96: return launch_append<T, 96>(p, s);
    default: return launch_append<T, 128>(p, s);
  }
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
  if (!places && tokens != cache->batch)
    return set_error(kEInval, "%s: %d tokens for %d sequences (give seqs and places)", what, tokens, cache->batch);
  if (!cos != !sin || (cos && rope_rows < 1) || (q && !cos))
    return set_error(kEInval, "%s: q and the rotation need both tables", what);
  if (tokens == 0) return kOk;
  if (!k || !v || (q && !q_out)) return set_error(kEInval, "%s: null pointer", what);
  const int es = dtype == BP_F32 ? 4 : 2, per = 16 / es;
  const int64_t kvw = (int64_t)cache->kv_heads * cache->head_dim, qw = (int64_t)heads * cache->head_dim;
  if (k_stride < kvw || v_stride < kvw || (q && q_stride < qw))
    return set_error(kEInval, "%s: a token stride is smaller than its rows", what);
  if (!aligned16(k) || !aligned16(v) || !aligned16(q) || !aligned16(q_out) || !aligned16(cos) || !aligned16(sin) ||
      k_stride % per || v_stride % per || (q && q_stride % per))
    return set_error(kEAlign, "%s: pointers and strides must be multiples of 16 bytes", what);
  rc = check_device();
  if (rc != kOk) return rc;
  p.tokens = tokens; p.heads = heads; p.rope_rows = rope_rows;
  p.k = k; p.v = v; p.q = q; p.ks = k_stride; p.vs = v_stride; p.qs = q_stride;
  p.cos = cos; p.sin = sin; p.positions = positions; p.seqs = seqs; p.places = places; p.q_out = q_out;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == BP_F32) return launch_append_dim<float>(p, s);
  if (dtype == BP_BF16) return launch_append_dim<__nv_bfloat16>(p, s);
  return launch_append_dim<__half>(p, s);
}
