// bp_kv_attend.cuh -- the one-token attention kernel over the paged b-posit
// cache, instantiated by bp_kv_attend8.cu (bp8) and bp_kv_attend16.cu (bp16) and
// launched by bp_kv_attend.cu.
//
// Per (sequence, kv head) row, with G query heads sharing the keys and values:
//   s[i, h] = scale * 2^ke[i] * sum_d K[i, d] q[h, d],   i < length
//   o[h, d] = sum_i e^(s[i, h] - m) 2^ve[i] V[i, d] / sum_i e^(s[i, h] - m)
// in one pass over the entries with a running maximum m, sum l and output o.
//
// Bound: the codes are read once from memory (2 D bytes per entry and kv head
// in bp8) and every code has to be decoded, which at the memory's rate is about
// 23 codes per clock and SM -- so decoding, not arithmetic on the decoded
// values, is what the layout is built around:
//  * Both products run on the tensor cores (mma.sync; tcgen05 would need the
//    decoded operands written back to shared memory, 2 to 4 bytes per code,
//    for an N of 8) with the cache as the wide operand: S^T = K q^T and
//    O^T = V^T P^T.  The K dimension of an MMA and the order of its rows are
//    free, so each thread's fragment is a contiguous piece of the rows in
//    shared memory and is decoded in registers, without a transpose.
//  * bp8 codes have at most 4 significant bits and a binade in [-24, 24]: exact
//    in bf16.  A 256-entry table holds, per code and lane, the bf16 value in the
//    low and in the high half of a word (64 KB: bank = lane, so no conflicts,
//    and one byte permute makes the address).  bp16 codes have at most 11
//    significant bits: exact in tf32; their fp32 bits are piecewise linear in
//    the code (see decode16).
//  * q and the softmax weights are fp32 and are split exactly into bf16 terms
//    (8 bits each), or nearly so into two tf32 terms, so every product keeps
//    fp32 accuracy; each tile's MMA sum is added to the running output by an
//    fp32 fma (the tensor cores truncate their sums, which would drift over
//    thousands of tiles).
//
// Work split: rows are cut into tiles of TT entries; the tiles of all rows, in
// order, are dealt to the CTAs (one per SM) in equal contiguous ranges and
// within a CTA to its warps, whatever the lengths are.  A warp fetches its
// tiles by bulk copies (one per page and operand) into its own stage and needs
// no other warp until its range ends.  A row that lies within one warp's range
// is finished by that warp; parts of a row are joined first over the CTA's warps
// in shared memory, then over CTAs by k_kv_join.
#pragma once
#include <math.h>

#include "bp_kv.cuh"

namespace bp {

constexpr long long kKvWaitLimit = 4000000000LL;   // cycles (~2 s) before a wait gives up
constexpr long long kKvDrainLimit = 200000000LL;   // cycles (~0.1 s) for copies in flight after that
constexpr int kHeadsPerRow = 8;                     // query heads of one work row (N of the MMAs)

struct AttendParams {
  KvView c;
  int heads, group, chunks;  // query heads, per kv head, and work rows per kv head
  int max_len;
  const void *q;
  int64_t qs;                // batch stride of q, elements
  void *out;
  float *lse;                // optional output, natural logarithm
  float scale;               // of the scores, times log2(e)
  // workspace
  float *warp_rec;           // [CTA][warp][8 D]: parts that ended inside a warp's range
  float *cta_rec;            // [CTA][2][8 D + 16]: o, m, l of rows that cross CTAs
  int4 *cta_row;             // [CTA]: {row that starts here and goes on or -1, CTAs that share it, -, -}
  float *lse2;               // [rows][8], base 2; null unless scores are accumulated
  float *raw;                // [rows][max_len][gp] scores, base 2; null unless accumulated
  int gp;                    // heads kept per entry in raw (even)
  int *error;
};

constexpr int kMaxWarps = 16;

// Query heads kept per entry and work row in `raw`, even so that pairs are one access.
inline int raw_heads(int group) { return group >= kHeadsPerRow ? kHeadsPerRow : (group + 1) & ~1; }

// Tile and launch shape of one instance.
template <int FMT, int D>
struct AttendCfg {
  static constexpr int BYTES = FMT / 8;
  static constexpr int ROWB = D * BYTES;
  static constexpr int TT = FMT == 8 ? (D <= 64 ? 64 : 32) : (D <= 32 ? 64 : 32);   // entries per tile
  static constexpr int NW = FMT == 8 ? (D <= 64 ? 16 : 8) : (D <= 64 ? 12 : 8);
  static constexpr int TILEB = TT * ROWB;
  static constexpr int STAGE = 2 * TILEB + (FMT == 8 ? 2 * TT : 0);
  static constexpr int LUT = FMT == 8 ? 65536 : 0;
  static constexpr int REC = kHeadsPerRow * D;                   // floats of one part's output
  // table, stages, part statistics [NW][2][16], part rows [NW][2], barriers [NW][2], scan [NW + 1], tiles before
  // each sequence [batch + 1]
  static constexpr int META = LUT + NW * STAGE;
  static constexpr int FIXED = META + NW * 2 * 64 + NW * 2 * 4 + NW * 2 * 8 + (NW + 2) * 4;
  static size_t smem(int batch) { return FIXED + (size_t)(batch + 1) * 4; }
  static_assert(REC * 4 <= STAGE, "a part's output fits the stage");
  static_assert(STAGE % 16 == 0, "stages stay 16-byte aligned");
};

namespace {

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bar_init(uint64_t *bar) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_addr(bar)));
}
__device__ __forceinline__ void bar_expect(uint64_t *bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t *bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait of a whole warp; false (and the error word set) if it gave up.
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity, int *error) {
  if (__all_sync(~0u, bar_try(bar, parity))) return true;
  const long long t0 = clock64();
  while (true) {
    if (__all_sync(~0u, bar_try(bar, parity))) return true;
    if (__any_sync(~0u, clock64() - t0 > kKvWaitLimit)) {
      if ((threadIdx.x & 31) == 0) atomicOr(error, 64);
      return false;
    }
  }
}
__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_addr(dst)),
      "l"(src), "r"(bytes), "r"(smem_addr(bar))
      : "memory");
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t to_tf32(float x) {
  uint32_t y;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(y) : "f"(x));
  return y;
}

// Terms that q and the weights are split into: fp32 exactly into three bf16
// terms, or into two tf32 terms (relative error 2^-22); bf16 and fp16 queries
// need one and two (one in tf32).  Weights for a 16-bit output take two terms
// (2^-16 of each weight, far below the output's half step).
template <int FMT, typename T>
struct Terms {
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr bool BF16 = !F32 && __is_same(T, __nv_bfloat16);
  static constexpr int Q = FMT == 8 ? (F32 ? 3 : (BF16 ? 1 : 2)) : (F32 ? 2 : 1);
  static constexpr int P = FMT == 8 ? (F32 ? 3 : 2) : 2;
};

__device__ __forceinline__ uint32_t top_bits(uint32_t x) { return x & 0xFFFF0000u; }
// (a's high half) | (b's high half) << 16
__device__ __forceinline__ uint32_t pack_high(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }

// x and y as N packed pairs of bf16 terms, largest first: each term is the
// rest's top 8 bits (truncated, so nothing overflows), the last of two or more
// takes what is left (exact for three terms, rounded for fewer).
template <int N>
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t (&out)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (n == N - 1 && N == 2) {
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(out[n]) : "f"(y), "f"(x));
    } else {
      out[n] = pack_high(__float_as_uint(x), __float_as_uint(y));
      if (n < N - 1) {
        x -= __uint_as_float(top_bits(__float_as_uint(x)));
        y -= __uint_as_float(top_bits(__float_as_uint(y)));
      }
    }
  }
}
template <int N>
__device__ __forceinline__ void split_tf32(float x, uint32_t (&out)[N]) {
  out[0] = __float_as_uint(x) & 0xFFFFE000u;
  if (N == 2) out[N - 1] = to_tf32(x - __uint_as_float(out[0]));
}

// fp32 bits of a bp16 code's value; `u` is 2^23 + 2^15 + the signed code as a
// float.  Below 1 the value's exponent and fraction, read as one fixed-point
// number, are 8 times those of the code's magnitude as a float (es = 3: a
// regime step is a binade of the magnitude and 8 of the value, and the exponent
// and fraction bits that follow line up), less a constant; above 1 they
// mirror those of 2^15 - magnitude.  Zero and NaR (magnitudes 0 and 2^15) give 0.
__device__ __forceinline__ uint32_t decode16(float u) {
  const float x = u - 8421376.0f;              // 2^23 + 2^15
  const float t = fabsf(x) - 16384.0f;
  const float w = 16384.0f - fabsf(t);         // min(magnitude, 2^15 - magnitude)
  uint32_t v = __float_as_uint(w) * 8u - (8u * ((127u + 14u) << 23) - (127u << 23));
  v = t > 0.0f ? (254u << 23) - v : v;
  v = w == 0.0f ? 0u : v;
  return v | (__float_as_uint(x) & 0x80000000u);
}

template <typename T>
__device__ __forceinline__ void write_out(const AttendParams &p, int64_t row, int h, int d, int D, float x) {
  const int ch = (int)(row % p.chunks);
  const int64_t bk = row / p.chunks;
  const int hk = (int)(bk % p.c.kv_heads), b = (int)(bk / p.c.kv_heads);
  const int g = ch * kHeadsPerRow + h;
  if (g < p.group) ((T *)p.out)[((int64_t)b * p.heads + hk * p.group + g) * D + d] = from_f32<T>(x);
}
__device__ __forceinline__ void write_lse(const AttendParams &p, int64_t row, int h, float lse2) {
  if (p.lse2) p.lse2[row * kHeadsPerRow + h] = lse2;
  if (!p.lse) return;
  const int ch = (int)(row % p.chunks);
  const int64_t bk = row / p.chunks;
  const int g = ch * kHeadsPerRow + h;
  if (g < p.group)
    p.lse[bk / p.c.kv_heads * p.heads + bk % p.c.kv_heads * p.group + g] = lse2 * 0.6931471805599453f;
}

// CTAs that take part: at least kMinTiles tiles each, so that short batches are
// not cut into parts that cost more to join than to read.
constexpr int kMinTiles = 8;
__device__ __forceinline__ int active_ctas(int tiles, int grid) {
  const int n = (tiles + kMinTiles - 1) / kMinTiles;
  return n < grid ? n : grid;
}

template <int FMT, int D, typename T>
__global__ void __launch_bounds__(AttendCfg<FMT, D>::NW * 32, 1) k_kv_attend(AttendParams p) {
  using C = AttendCfg<FMT, D>;
  using N = Terms<FMT, T>;
  constexpr int TT = C::TT, NW = C::NW, MT = TT / 16, MD = D / 16, NT = NW * 32;
  constexpr int QS = FMT == 8 ? D / 16 : D / 8;          // MMA steps along D
  extern __shared__ __align__(128) uint8_t smem[];
  float *const rec_ml = reinterpret_cast<float *>(smem + C::META);          // [NW][2][m 8, l 8]
  int *const rec_row = reinterpret_cast<int *>(rec_ml + NW * 32);           // [NW][2]
  uint64_t *const bars = reinterpret_cast<uint64_t *>(rec_row + NW * 2);    // [NW][K, V]
  int *const scan = reinterpret_cast<int *>(bars + NW * 2);
  int *const before = scan + NW + 2;                                        // [batch + 1]
  const KvView &c = p.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int per_seq = c.kv_heads * p.chunks;             // work rows of one sequence
  asm volatile("griddepcontrol.launch_dependents;");

  auto length = [&](int b) { return min(c.length(b), p.max_len); };
  // tiles before each sequence
  {
    const int each = (c.batch + NT - 1) / NT;
    int mine = 0;
    for (int i = 0; i < each; ++i) {
      const int b = tid * each + i;
      if (b < c.batch) mine += (length(b) + TT - 1) / TT * per_seq;
    }
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(~0u, incl, d);
      if (lane >= d) incl += x;
    }
    if (lane == 31) scan[warp] = incl;
    if (tid < NW * 2) {
      rec_row[tid] = -1;
      bar_init(&bars[tid]);
    }
    if (tid == 0) asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();
    int at = incl - mine;
    for (int w = 0; w < warp; ++w) at += scan[w];
    for (int i = 0; i < each; ++i) {
      const int b = tid * each + i;
      if (b < c.batch) {
        before[b] = at;
        at += (length(b) + TT - 1) / TT * per_seq;
      }
    }
    if (tid == NT - 1) before[c.batch] = at;
    __syncthreads();
  }
  const int total = before[c.batch];
  // empty sequences: zeros, and -inf for the logarithm
  for (int b = blockIdx.x; b < c.batch; b += gridDim.x)
    if (before[b + 1] == before[b]) {
      T *o = (T *)p.out + (int64_t)b * p.heads * D;
      for (int i = tid; i < p.heads * D; i += NT) o[i] = from_f32<T>(0.0f);
      if (p.lse)
        for (int i = tid; i < p.heads; i += NT) p.lse[(int64_t)b * p.heads + i] = -INFINITY;
    }
  const int ctas = active_ctas(total, gridDim.x);
  const int cta = blockIdx.x;
  if (cta >= ctas) {
    if (tid == 0) p.cta_row[cta] = make_int4(-1, 0, 0, 0);
    return;
  }
  const int lo = (int)((int64_t)total * cta / ctas), hi = (int)((int64_t)total * (cta + 1) / ctas);
  const int wlo = lo + (int)((int64_t)(hi - lo) * warp / NW), whi = lo + (int)((int64_t)(hi - lo) * (warp + 1) / NW);

  uint8_t *const stage = smem + C::LUT + warp * C::STAGE;
  uint8_t *const sk = stage, *const sv = stage + C::TILEB;
  int8_t *const ske = reinterpret_cast<int8_t *>(stage + 2 * C::TILEB), *const sve = ske + TT;
  uint64_t *const kbar = &bars[warp * 2], *const vbar = kbar + 1;

  // ---- the tile that is fetched next: x = its number, and where it lies ----
  int nx = wlo, nb = 0, nrow = 0, ntile = 0, nn = 0, npage = -1;
  auto locate = [&]() {       // sequence of tile nx by bisection
    int a = 0, z = c.batch;
    while (z - a > 1) {
      const int m = (a + z) >> 1;
      if (before[m] <= nx) a = m;
      else z = m;
    }
    nb = a;
    nn = length(nb);
    const int nt = (nn + TT - 1) / TT, r = nx - before[nb];
    nrow = nt ? r / nt : 0;
    ntile = nt ? r % nt : 0;
  };
  const int seg = min(TT, 1 << c.page_shift);            // entries per copy
  auto pages = [&]() {        // this lane's page of the tile; its entries in it
    const int i = ntile * TT + lane * seg;
    npage = lane * seg < TT && i < nn ? c.page_of(nb, i) : -2;
  };
  uint32_t fetched[2] = {0, 0};
  auto fetch = [&](bool value) {
    ++fetched[value];
    const int i = ntile * TT + lane * seg;
    const int cnt = npage == -2 ? 0 : min(seg, nn - i);
    const bool ok = npage >= 0;
    const uint32_t bytes = ok ? cnt * C::ROWB : 0, ebytes = FMT == 8 && ok ? (cnt + 15) & ~15 : 0;
    const uint32_t all = __reduce_add_sync(~0u, bytes + ebytes);
    uint64_t *bar = value ? vbar : kbar;
    if (lane == 0) bar_expect(bar, all);
    __syncwarp();
    if (ok) {
      const int64_t row = c.row(npage, nrow / p.chunks, i);
      bulk_load((value ? sv : sk) + lane * seg * C::ROWB, (value ? c.v : c.k) + row * C::ROWB, bytes, bar);
      if (FMT == 8) bulk_load((value ? sve : ske) + lane * seg, (value ? c.v_exp : c.k_exp) + row, ebytes, bar);
    }
  };

  if (wlo < whi) {
    locate();
    pages();
    fetch(false);
    fetch(true);
  }
  if (FMT == 8) {
    // the decode table: word 64 code + lane (value in the low half) and + 32 (in the high half)
    for (int i = tid; i < 512; i += NT) {
      const int code = i & 255;
      const uint32_t v = posit_to_f32_bits<8, 2>(code);
      uint32_t *row = reinterpret_cast<uint32_t *>(smem) + code * 64;
      const int half = (i >> 8) * 32;
#pragma unroll 8
      for (int j = 0; j < 32; ++j) row[half + ((j + i) & 31)] = half ? v : v >> 16;
    }
  }
  __syncthreads();
  const uint32_t lane4 = lane * 4;
  // bytes ka of a and kb of b as a pair of bf16 values
  auto pair8 = [&](uint32_t a, int ka, uint32_t b, int kb) {
    const uint32_t x = __byte_perm(a, lane4, 0x5504 | ka << 4), y = __byte_perm(b, lane4, 0x5504 | kb << 4);
    return *reinterpret_cast<const uint32_t *>(smem + x) | *reinterpret_cast<const uint32_t *>(smem + 128 + y);
  };

  uint32_t qf[QS][N::Q][2];
  float o[MD][4], m[2], l[2];
  bool dead = false;
  // entry of an S tile's row g (and, + 8, of row g + 8): see the header on the free order
  const int er = (g & 1) ? 4 + ((g >> 1) ^ 1) : g >> 1;

  for (int x = wlo; x < whi; ++x) {
    const int b = nb, row = nrow, tile = ntile, n = nn, nt = (n + TT - 1) / TT;
    const int64_t grow = (int64_t)b * per_seq + row;
    const int valid = min(TT, n - tile * TT);
    const uint32_t parity = (x - wlo) & 1;
    const bool lost = __any_sync(~0u, npage == -1);
    if (x == wlo || tile == 0) {       // a new row: its queries, and an empty state
      const int hk = row / p.chunks, h = (row % p.chunks) * kHeadsPerRow + g;
      const T *q = (const T *)p.q + b * p.qs + (int64_t)(hk * p.group + h) * D + t * (D / 4);
#pragma unroll
      for (int s = 0; s < QS; ++s) {
        constexpr int per = FMT == 8 ? 4 : 2;
        float f[per];
#pragma unroll
        for (int j = 0; j < per; ++j) f[j] = h < p.group ? to_f32(q[s * per + j]) : 0.0f;
        if (FMT == 8) {
          uint32_t u[N::Q], w[N::Q];
          split_bf16<N::Q>(f[0], f[1], u);
          split_bf16<N::Q>(f[per - 2], f[per - 1], w);
#pragma unroll
          for (int i = 0; i < N::Q; ++i) {
            qf[s][i][0] = u[i];
            qf[s][i][1] = w[i];
          }
        } else {
          uint32_t u[N::Q], w[N::Q];
          split_tf32<N::Q>(f[0], u);
          split_tf32<N::Q>(f[1], w);
#pragma unroll
          for (int i = 0; i < N::Q; ++i) {
            qf[s][i][0] = u[i];
            qf[s][i][1] = w[i];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < MD; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.0f;
    }
    // ---- scores: S^T[entry, head] ----
    if (!dead) dead = !bar_wait(kbar, parity, p.error);
    float s[MT][4];
    float kscale[MT][2];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.0f;
      const int e = i * 16 + er;
      kscale[i][0] = FMT == 8 ? exp2_int(ske[e]) * p.scale : p.scale;
      kscale[i][1] = FMT == 8 ? exp2_int(ske[e + 8]) * p.scale : p.scale;
      if (FMT == 8) {
        uint32_t a0[D / 16], a1[D / 16];
        const uint8_t *r0 = sk + e * C::ROWB + t * (D / 4), *r1 = r0 + 8 * C::ROWB;
        if constexpr (D % 64 == 0) {
#pragma unroll
          for (int w = 0; w < D / 64; ++w) {
            *reinterpret_cast<uint4 *>(a0 + 4 * w) = reinterpret_cast<const uint4 *>(r0)[w];
            *reinterpret_cast<uint4 *>(a1 + 4 * w) = reinterpret_cast<const uint4 *>(r1)[w];
          }
        } else {
#pragma unroll
          for (int w = 0; w < D / 32; ++w) {
            *reinterpret_cast<uint2 *>(a0 + 2 * w) = reinterpret_cast<const uint2 *>(r0)[w];
            *reinterpret_cast<uint2 *>(a1 + 2 * w) = reinterpret_cast<const uint2 *>(r1)[w];
          }
        }
#pragma unroll
        for (int w = 0; w < QS; ++w) {
          const uint32_t a[4] = {pair8(a0[w], 0, a0[w], 1), pair8(a1[w], 0, a1[w], 1), pair8(a0[w], 2, a0[w], 3),
                                 pair8(a1[w], 2, a1[w], 3)};
#pragma unroll
          for (int j = N::Q - 1; j >= 0; --j) mma_bf16(s[i], a, qf[w][j][0], qf[w][j][1]);
        }
      } else {
        const uint8_t *r0 = sk + e * C::ROWB + t * (D / 2), *r1 = r0 + 8 * C::ROWB;
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {      // 8 codes of each row
          const uint4 x0 = reinterpret_cast<const uint4 *>(r0)[w], x1 = reinterpret_cast<const uint4 *>(r1)[w];
          const uint32_t y0[4] = {x0.x, x0.y, x0.z, x0.w}, y1[4] = {x1.x, x1.y, x1.z, x1.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t u0 = y0[k] ^ 0x80008000u, u1 = y1[k] ^ 0x80008000u;
            const uint32_t a[4] = {decode16(__uint_as_float(__byte_perm(u0, 0x4B00u, 0x5410))),
                                   decode16(__uint_as_float(__byte_perm(u1, 0x4B00u, 0x5410))),
                                   decode16(__uint_as_float(__byte_perm(u0, 0x4B00u, 0x5432))),
                                   decode16(__uint_as_float(__byte_perm(u1, 0x4B00u, 0x5432)))};
#pragma unroll
            for (int j = N::Q - 1; j >= 0; --j) mma_tf32(s[i], a, qf[w * 4 + k][j][0], qf[w * 4 + k][j][1]);
          }
        }
      }
    }
    __syncwarp();
    // ---- the next tile's keys ----
    const bool more = x + 1 < whi;
    if (more) {
      ++nx;
      ++ntile;
      if (ntile == nt) {
        ntile = 0;
        if (++nrow == per_seq) {
          nrow = 0;
          do ++nb;
          while (before[nb + 1] == before[nb]);
          nn = length(nb);
        }
      }
      pages();
      if (!dead) fetch(false);
    }
    // ---- weights ----
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = i * 16 + er + (j >> 1) * 8;
        s[i][j] = e < valid ? s[i][j] * kscale[i][j >> 1] : -INFINITY;
        mx[j & 1] = fmaxf(mx[j & 1], s[i][j]);
      }
    if (p.raw) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int e = i * 16 + er + j * 8;
          if (e < valid && 2 * t < p.gp)
            *reinterpret_cast<float2 *>(p.raw + ((grow * p.max_len + tile * TT + e) * p.gp + 2 * t)) =
                make_float2(s[i][2 * j], s[i][2 * j + 1]);
        }
    }
    float alpha[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) mx[j] = fmaxf(mx[j], __shfl_xor_sync(~0u, mx[j], d));
      const float mn = fmaxf(m[j], mx[j]);
      // nothing but -inf so far: weigh it with 0
      const float at = mn == -INFINITY ? 0.0f : mn;
      alpha[j] = ex2(m[j] - at);
      l[j] *= alpha[j];
      m[j] = mn;
      mx[j] = at;
    }
    if (!dead) dead = !bar_wait(vbar, parity, p.error);
    if (lost || dead) l[0] = l[1] = NAN;
    // ---- O^T += V^T P^T ----
    float acc[MD][4];
#pragma unroll
    for (int i = 0; i < MD; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      float w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = ex2(s[i][j] - mx[j & 1]);
        l[j & 1] += w[j];
      }
      if (FMT == 8) {
        const int e = i * 16 + er;
        const float v0 = exp2_int(sve[e]), v1 = exp2_int(sve[e + 8]);
        // (entries behind the length have weight 0 and any exponent: 0 times a finite power)
        uint32_t u0[N::P], u1[N::P];
        split_bf16<N::P>(w[0] * v0, w[1] * v0, u0);
        split_bf16<N::P>(w[2] * v1, w[3] * v1, u1);
#pragma unroll
        for (int j = 0; j < N::P; ++j) {
          u0[j] = transpose8x8(u0[j]);
          u1[j] = transpose8x8(u1[j]);
        }
        // this thread's entries of the 16: t, 4 + (t ^ 1), 8 + t, 12 + (t ^ 1)
        uint32_t a[4][D / 32];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint8_t *r = sv + (i * 16 + k * 4 + ((k & 1) ? t ^ 1 : t)) * C::ROWB + g * (D / 8);
          if constexpr (D == 128) *reinterpret_cast<uint4 *>(a[k]) = *reinterpret_cast<const uint4 *>(r);
          else if constexpr (D == 64) *reinterpret_cast<uint2 *>(a[k]) = *reinterpret_cast<const uint2 *>(r);
          else
#pragma unroll
            for (int y = 0; y < D / 32; ++y) a[k][y] = reinterpret_cast<const uint32_t *>(r)[y];
        }
#pragma unroll
        for (int d = 0; d < MD; ++d) {
          const int y = d >> 1, k = (d & 1) * 2;
          const uint32_t v[4] = {pair8(a[0][y], k, a[1][y], k), pair8(a[0][y], k + 1, a[1][y], k + 1),
                                 pair8(a[2][y], k, a[3][y], k), pair8(a[2][y], k + 1, a[3][y], k + 1)};
#pragma unroll
          for (int j = N::P - 1; j >= 0; --j) mma_bf16(acc[d], v, u0[j], u1[j]);
        }
      } else {
#pragma unroll
        for (int half = 0; half < 2; ++half) {        // rows 0-7 and 8-15: one MMA step of 8 entries each
          const uint32_t lo16 = transpose8x8(__byte_perm(__float_as_uint(w[2 * half]), __float_as_uint(w[2 * half + 1]), 0x5410));
          const uint32_t hi16 = transpose8x8(pack_high(__float_as_uint(w[2 * half]), __float_as_uint(w[2 * half + 1])));
          uint32_t u0[N::P], u1[N::P];
          split_tf32<N::P>(__uint_as_float(__byte_perm(lo16, hi16, 0x5410)), u0);
          split_tf32<N::P>(__uint_as_float(__byte_perm(lo16, hi16, 0x7632)), u1);
          uint32_t a[2][D / 16];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint8_t *r = sv + (i * 16 + half * 8 + (k ? 4 + (t ^ 1) : t)) * C::ROWB + g * (D / 4);
            if constexpr (D % 64 == 0) {
#pragma unroll
              for (int y = 0; y < D / 64; ++y)
                *reinterpret_cast<uint4 *>(a[k] + 4 * y) = reinterpret_cast<const uint4 *>(r)[y];
            } else {
#pragma unroll
              for (int y = 0; y < D / 32; ++y)
                *reinterpret_cast<uint2 *>(a[k] + 2 * y) = reinterpret_cast<const uint2 *>(r)[y];
            }
          }
#pragma unroll
          for (int d = 0; d < MD; ++d) {
            const uint32_t x0 = a[0][d] ^ 0x80008000u, x1 = a[1][d] ^ 0x80008000u;
            const uint32_t v[4] = {decode16(__uint_as_float(__byte_perm(x0, 0x4B00u, 0x5410))),
                                   decode16(__uint_as_float(__byte_perm(x0, 0x4B00u, 0x5432))),
                                   decode16(__uint_as_float(__byte_perm(x1, 0x4B00u, 0x5410))),
                                   decode16(__uint_as_float(__byte_perm(x1, 0x4B00u, 0x5432)))};
#pragma unroll
            for (int j = N::P - 1; j >= 0; --j) mma_tf32(acc[d], v, u0[j], u1[j]);
          }
        }
      }
    }
#pragma unroll
    for (int d = 0; d < MD; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[d][j] = fmaf(o[d][j], alpha[j & 1], acc[d][j]);
    __syncwarp();
    if (more && !dead) fetch(true);

    // ---- the end of a row, or of this warp's range ----
    if (tile + 1 == nt || !more) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[j] += __shfl_xor_sync(~0u, l[j], d);
      const bool begun = x - tile >= wlo, ended = tile + 1 == nt;
      if (begun && ended) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int h = 2 * t + j, ch = row % p.chunks, gh = ch * kHeadsPerRow + h;
          if (gh < p.group) {
            T *out = (T *)p.out + ((int64_t)b * p.heads + (row / p.chunks) * p.group + gh) * D + g * (D / 8);
            const float inv = 1.0f / l[j];
#pragma unroll
            for (int d = 0; d < MD; ++d) {
              out[2 * d] = from_f32<T>(o[d][j] * inv);
              out[2 * d + 1] = from_f32<T>(o[d][2 + j] * inv);
            }
          }
          if (g == 0) write_lse(p, grow, h, m[j] + log2f(l[j]));
        }
      } else {
        // a part: inside the range it goes to the workspace (the stage holds the next tile), at its end to the stage
        const int slot = more ? 0 : 1;
        float *rec = more ? p.warp_rec + ((int64_t)cta * NW + warp) * C::REC : reinterpret_cast<float *>(stage);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float *r = rec + (2 * t + j) * D + g * (D / 8);
#pragma unroll
          for (int d = 0; d < MD; ++d) {
            r[2 * d] = o[d][j];
            r[2 * d + 1] = o[d][2 + j];
          }
          if (g == 0) {
            rec_ml[(warp * 2 + slot) * 16 + 2 * t + j] = m[j];
            rec_ml[(warp * 2 + slot) * 16 + 8 + 2 * t + j] = l[j];
          }
        }
        if (lane == 0) rec_row[warp * 2 + slot] = (int)grow;
      }
    }
  }
  if (dead) {      // the copies in flight may still land: wait for them, with a limit
    const long long t0 = clock64();
    while (clock64() - t0 < kKvDrainLimit)
      if (bar_try(kbar, (fetched[0] - 1) & 1) && bar_try(vbar, (fetched[1] - 1) & 1)) break;
  }
  __syncthreads();

  // ---- join the parts of this CTA's rows ----
  int4 open = make_int4(-1, 0, 0, 0);
  for (int i = 0; i < NW * 2;) {
    const int row = rec_row[i];
    if (row < 0) {
      ++i;
      continue;
    }
    int z = i + 1;
    while (z < NW * 2 && (rec_row[z] == row || rec_row[z] < 0)) ++z;
    const int b = row / per_seq, nt = (before[b + 1] - before[b]) / per_seq;
    const int x0 = before[b] + (row - b * per_seq) * nt, x1 = x0 + nt;
    const bool whole = x0 >= lo && x1 <= hi;
    float *out = p.cta_rec + ((int64_t)cta * 2 + (x0 >= lo)) * (C::REC + 16);
    for (int e = tid; e < C::REC; e += NT) {
      const int h = e / D;
      float M = -INFINITY, L = 0.0f, O = 0.0f;
      for (int k = i; k < z; ++k)
        if (rec_row[k] == row) M = fmaxf(M, rec_ml[k * 16 + h]);
      for (int k = i; k < z; ++k)
        if (rec_row[k] == row) {
          const float a = ex2(rec_ml[k * 16 + h] - M);
          const float *rec = (k & 1) ? reinterpret_cast<const float *>(smem + C::LUT + (k >> 1) * C::STAGE)
                                     : p.warp_rec + ((int64_t)cta * NW + (k >> 1)) * C::REC;
          L = fmaf(rec_ml[k * 16 + 8 + h], a, L);
          O = fmaf(rec[e], a, O);
        }
      if (whole) {
        write_out<T>(p, row, h, e - h * D, D, O / L);
        if (e % D == 0) write_lse(p, row, h, M + log2f(L));
      } else {
        out[e] = O;
        if (e % D == 0) {
          out[C::REC + h] = M;
          out[C::REC + 8 + h] = L;
        }
      }
    }
    if (x0 >= lo && x1 > hi) {
      // the CTA that holds tile x1 - 1 is the last one of this row
      const int last = (int)(((int64_t)x1 * ctas - 1) / total);
      open = make_int4(row, last - cta + 1, 0, 0);
    }
    i = z;
  }
  if (tid == 0) p.cta_row[cta] = open;
}

}  // namespace

// Launches the instance for (fmt, D, dtype) on `grid` CTAs.
int launch_kv_attend8(const AttendParams &p, int dtype, int grid, cudaStream_t s);
int launch_kv_attend16(const AttendParams &p, int dtype, int grid, cudaStream_t s);

template <int FMT, int D, typename T>
int launch_kv_attend_one(const AttendParams &p, int grid, cudaStream_t s) {
  using C = AttendCfg<FMT, D>;
  const size_t bytes = C::smem(p.c.batch);
  static_assert(C::FIXED + 4 * 4097 <= 232448, "shared memory per CTA");
  cudaError_t e = cudaFuncSetAttribute(k_kv_attend<FMT, D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != cudaSuccess) return set_error(kECuda, "k_kv_attend: %s", cudaGetErrorString(e));
  k_kv_attend<FMT, D, T><<<grid, C::NW * 32, bytes, s>>>(p);
  return check_launch("k_kv_attend");
}
template <int FMT, typename T>
int launch_kv_attend_dim(const AttendParams &p, int grid, cudaStream_t s) {
  switch (p.c.dim) {
    case 32: return launch_kv_attend_one<FMT, 32, T>(p, grid, s);
    case 64: return launch_kv_attend_one<FMT, 64, T>(p, grid, s);
    case 96: return launch_kv_attend_one<FMT, 96, T>(p, grid, s);
    default: return launch_kv_attend_one<FMT, 128, T>(p, grid, s);
  }
}
template <int FMT>
int launch_kv_attend_fmt(const AttendParams &p, int dtype, int grid, cudaStream_t s) {
  if (dtype == BP_F32) return launch_kv_attend_dim<FMT, float>(p, grid, s);
  if (dtype == BP_BF16) return launch_kv_attend_dim<FMT, __nv_bfloat16>(p, grid, s);
  return launch_kv_attend_dim<FMT, __half>(p, grid, s);
}

}  // namespace bp
