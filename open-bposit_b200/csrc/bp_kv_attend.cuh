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
//  * Both products run on the tensor cores (mma.sync m16n8k8, tf32; tcgen05
//    would need the decoded operands written back to shared memory, 4 bytes
//    per code, for 8 rows of queries).  The cache is the B operand, whose K
//    order and column order are free, so each thread's fragments are contiguous
//    pieces of the rows in shared memory, decoded in registers without a
//    transpose; and S^T's accumulators are P's A fragment as they are.
//  * Codes are exact in tf32: bp8 values have at most 4 significant bits, bp16
//    values at most 11.  Both go through a table with a copy of every entry for
//    each lane (bank = lane, so no conflicts, and one byte permute makes the
//    address): for bp8 the fp32 value of the code, for bp16 the value of the
//    upper byte's first code and the step to the next one, so that a permute, a
//    look-up, a permute, a sign extension and a multiply-add decode a code (11
//    instructions without the table: decode16, which the rare codes take that
//    are not linear in the lower byte).
//  * The rows of the A operand are 8 query heads twice: the upper 11 bits of q
//    (or of the softmax weight), and what is left of it, 11 bits more.  The two
//    sums are added in fp32, so products keep fp32 accuracy.  Each tile's sum
//    is added to the running output by an fp32 fma: the tensor cores truncate
//    their sums, which would drift over thousands of tiles.
//
// Work split: rows are cut into units of 16 entries; the units of all rows, in
// order and with some more for every row's start, are dealt to the CTAs (one per
// SM) in equal contiguous ranges and within a CTA to its warps, whatever the
// lengths are.  A warp takes its units
// four at a time (a tile; single ones at the end of a row or of its range),
// fetches tiles into its own stage (cp.async, 16 bytes a lane: a page table look-up per
// page and no address work per row) and needs no other warp until its range
// ends; the next tile's keys are fetched while this one's values are used, and
// the other way round.  Rows lie in the stage with their 16-byte pieces permuted
// (Swizzle) so that no fragment load has bank conflicts.  A row that lies within
// one warp's range is finished by that warp; parts of a row are joined first
// over the CTA's warps in shared memory, then over CTAs by k_kv_finish.
#pragma once
#include <math.h>

#include <atomic>
#include <type_traits>

#include "bp_kv.cuh"

namespace bp {

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
  int2 *cta_row;             // [CTA]: {row that starts here and goes on behind it, or -1; CTAs that share it}
  float *lse2;               // [rows][8], base 2; null unless scores are accumulated
  int2 *row_parts;           // [rows]: {first CTA, parts} of a row that crosses CTAs, {-, 0}: its lse2 is there; or null
  float *raw;                // [rows][max_len][gp] scores, base 2; null unless accumulated
  int gp;                    // heads kept per entry in raw (even)
};

constexpr int kMaxWarps = 8;                        // warps of a CTA
constexpr int kMaxBatch = 2048;
constexpr int kTableAt = 65536;                     // shared address of the bp8 decode table
constexpr int kSharedReserved = 1024;               // shared address where a block's own memory starts

// Query heads kept per entry and work row in `raw`, even so that pairs are one access.
inline int raw_heads(int group) { return group >= kHeadsPerRow ? kHeadsPerRow : (group + 1) & ~1; }

// Tile and launch shape of one instance.
template <int FMT, int D, typename T>
struct AttendCfg {
  static constexpr int BYTES = FMT / 8;
  static constexpr int ROWB = D * BYTES;
  // Entries per tile, warps, and parts that an output's columns are worked on in.  Wide bp16 rows
  // take single units, whose unrolled steps fit the instruction cache (32 entries at D = 128: 84 us, a quarter of it
  // waiting for instructions, where single units take 48 us).
  static constexpr bool WIDE = FMT == 16 && D > 64;
  static constexpr int TT = FMT == 8 ? (D <= 64 ? 64 : 32) : (D <= 32 ? 64 : (D <= 64 ? 32 : 16));
  static constexpr int NW = kMaxWarps;
  static constexpr int PARTS = WIDE ? 2 : 1;
  static constexpr int TILEB = TT * ROWB;
  // 2^exponent of a tile's keys and values as fp32, [t][n][2] in the order that thread t of a quad needs them, with
  // a row stride that keeps the four rows in different banks
  static constexpr int POWROW = TT / 4 + 8;
  static constexpr int POWB = FMT == 8 ? 2 * 4 * POWROW * 4 : 0;
  static constexpr int STAGE = 2 * TILEB + (FMT == 8 ? 2 * TT : 0) + POWB;   // keys, values, exponents, powers
  static constexpr int REC = kHeadsPerRow * D;                   // floats of one part's output
  // Shared memory: the decode table at shared addresses 64 K .. 128 K, so that an entry's address is the bytes {lane,
  // code, 1, 0}; FRONT stages below it, the others above.  The table's entries fill half of its 256-byte rows; the
  // other halves hold the units before each sequence and the lengths (kMaxBatch of each).
  static constexpr int FRONT = (kTableAt - kSharedReserved) / STAGE;
  static constexpr int BACK = NW - (FRONT < NW ? FRONT : NW);
  // offset of what follows the table, from shared address kSharedReserved
  static constexpr int AFTER = 2 * kTableAt - kSharedReserved;
  // part statistics [NW][2][16], part rows and their sequences [NW][2], scan [NW + 2]
  static constexpr int META = AFTER + BACK * STAGE;
  static constexpr int SMEM = META + NW * 2 * 64 + NW * 2 * 8 + (NW + 2) * 4;
  static __device__ __forceinline__ int stage_at(int warp) {
    return warp < FRONT ? warp * STAGE : AFTER + (warp - FRONT) * STAGE;
  }
  static_assert(REC * 4 <= STAGE, "a part's output fits the stage");
  static_assert(FMT == 16 || TT % 32 == 0, "a lane converts TT / 32 exponents");
  static_assert(STAGE % 16 == 0, "stages stay 16-byte aligned");
};

namespace {

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 16 bytes from global to shared memory, asynchronously; groups complete in order.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All groups but the last N are complete, for the whole warp.
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
  __syncwarp();
}

// Offset of 16-byte piece c of row r of a tile.  A fragment load takes the same
// pieces of several rows at once: keys pieces of rows {0, 5}, {1, 4}, {2, 7} or
// {3, 6} (two rows a quarter warp), values of rows 0-3 or 4-7 (four rows).  The
// permutation puts those into different banks; rows of 96 and 192 bytes differ
// enough by themselves.
template <int ROWB>
__device__ __forceinline__ int swizzle(int r, int c) {
  int s = 0, lane = c;
  if (ROWB == 32) {            // 4 rows in 128 bytes
    lane = (r & 3) * 2 + c;
    s = (r >> 2 & 1) * 4;
    return (r >> 2) * 128 + (lane ^ s) * 16;
  }
  if (ROWB == 64) {            // 2 rows
    lane = (r & 1) * 4 + c;
    s = (r >> 1 & 1) * 2;
    return (r >> 1) * 128 + (lane ^ s) * 16;
  }
  if (ROWB == 128) s = (r & 3) * 2 ^ (r & 1);
  if (ROWB == 256) s = ((r & 1) | (r >> 1 & 1) * 4) ^ (c >> 3) * 2;
  return r * ROWB + (c ^ s) * 16;
}
// N words at word `at` of row r; they lie within 16-byte pieces.
template <int ROWB, int N>
__device__ __forceinline__ void load_words(const uint8_t *tile, int r, int at, uint32_t (&x)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
      *reinterpret_cast<uint4 *>(x + 4 * i) =
          *reinterpret_cast<const uint4 *>(tile + swizzle<ROWB>(r, at / 4 + i));
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i)
      *reinterpret_cast<uint2 *>(x + 2 * i) = *reinterpret_cast<const uint2 *>(
          tile + swizzle<ROWB>(r, (at + 2 * i) / 4) + (at + 2 * i) % 4 * 4);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      x[i] = *reinterpret_cast<const uint32_t *>(tile + swizzle<ROWB>(r, (at + i) / 4) + (at + i) % 4 * 4);
  }
}

// c += a b, and the same from a zero accumulator.
__device__ __forceinline__ void mma_tf32_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Entry of the decode table by shared address.
__device__ __forceinline__ uint32_t table_entry(uint32_t at) {
  uint32_t y;
  asm("ld.shared.b32 %0, [%1];" : "=r"(y) : "r"(at));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// What scores and parts are weighed against: where there is nothing but -inf so
// far, any number gives them the weight 0.
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ uint32_t to_tf32(float x) {
  uint32_t y;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(y) : "f"(x));
  return y;
}

// The upper 11 bits of x, and the rest of it as tf32.
__device__ __forceinline__ uint32_t tf32_high(float x) { return __float_as_uint(x) & 0xFFFFE000u; }

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

// Word i of the decode table's free halves: the units before sequence i, and
// from kMaxBatch + 1 on the lengths.
__device__ __forceinline__ int &spare_word(uint8_t *table, int i) {
  return *reinterpret_cast<int *>(table + (i >> 5) * 256 + 128 + (i & 31) * 4);
}

// tf32 bits of code k of a word; `entry`: lane * 4 and the table's address.
// bp16: the fp32 bits are linear in the code within blocks of 256 codes, but in
// the first and last block of each sign; a code of those leaves a 1 in `odd`,
// and the step is done again with EXACT.  (The table's low 13 bits ride along:
// they are not part of a tf32 operand.)
template <int FMT, bool EXACT>
__device__ __forceinline__ uint32_t decode_code(uint32_t entry, uint32_t w, int k, uint32_t &odd) {
  if (FMT == 8) return table_entry(__byte_perm(w, entry, 0x6504 | k << 4));
  if (EXACT) return decode16(__uint_as_float(__byte_perm(w ^ 0x80008000u, 0x4B00u, k ? 0x5432 : 0x5410)));
  const uint32_t e = table_entry(__byte_perm(w, entry, 0x6504 | (2 * k + 1) << 4));
  int step;
  asm("bfe.s32 %0, %1, 0, 13;" : "=r"(step) : "r"(e));
  odd |= e;
  return __byte_perm(w, 0, 0x4404 | (2 * k) << 4) * (uint32_t)step + e;
}

// A work row: 8 (or fewer) query heads of one kv head of one sequence.
struct RowId {
  int b, hk, ch;
};
__device__ __forceinline__ RowId row_id(const AttendParams &p, int row) {
  const int bk = row / p.chunks, b = bk / p.c.kv_heads;
  return {b, bk - b * p.c.kv_heads, row - bk * p.chunks};
}
// Query head h of the row as an index into [batch, heads]; -1 for a head that pads the row.
__device__ __forceinline__ int64_t head_of(const AttendParams &p, const RowId &r, int h) {
  const int g = r.ch * kHeadsPerRow + h;
  return g < p.group ? (int64_t)r.b * p.heads + r.hk * p.group + g : -1;
}
__device__ __forceinline__ void write_lse(const AttendParams &p, int row, int h, int64_t head, float lse2) {
  if (p.lse2) {
    p.lse2[(int64_t)row * kHeadsPerRow + h] = lse2;
    if (h == 0) p.row_parts[row] = make_int2(0, 0);
  }
  if (p.lse && head >= 0) p.lse[head] = lse2 * 0.6931471805599453f;
}

// The units 0 .. total - 1 over `parts`: the first total % parts of them have one more.
struct Deal {
  int each, more;
  __device__ __forceinline__ Deal(int total, int parts) : each(total / parts), more(total - each * parts) {}
  __device__ __forceinline__ int begin(int part) const { return part * each + min(part, more); }
  __device__ __forceinline__ int part_of(int unit) const {
    const int front = more * (each + 1);
    return unit < front ? unit / (each + 1) : more + (unit - front) / each;
  }
};
// CTAs that take part: at least kMinUnits units each, so that short batches are
// not cut into parts that cost more to join than to read (8 sequences of 1 to
// 1500 entries, 14 and 2 heads of 64, bp8: 8.5 us with 4 units, 8.7 with 8, 9.5
// with 16, 10.8 with 32; longer batches use every CTA with any of them).  What
// fits kOneCta units stays in one CTA and needs no second
// kernel (one sequence of 17 entries: 5.3 us, against 5.9 in two).
constexpr int kMinUnits = 8, kOneCta = 16;
// Units that a row counts for besides its own, in front of them, when work is
// dealt: its end and the next one's start leave the pipeline of fetches empty
// (64 sequences of up to 16384 entries: 52.5 us with 0, 51.4 with 1, 50.6 to 50.9
// with 2 to 6, 51.0 with 8; 16 sequences of up to 4096 entries of 8 x 128 in bp16:
// 49.8 with 0, 47.4 with 1, 47.7 with 2 and 3, 48.3 with 6; 16 x 4096 with scores:
// 16.5 with 0, 15.8 with 1, 15.4 from 3 to 6).
constexpr int kRowUnits = 3;
__device__ __forceinline__ int active_ctas(int units, int grid) {
  return units <= kOneCta ? min(units, 1) : min((units + kMinUnits - 1) / kMinUnits, grid);
}

template <int FMT, int D, typename T>
__global__ void __launch_bounds__(AttendCfg<FMT, D, T>::NW * 32, 1) k_kv_attend(AttendParams p) {
  using C = AttendCfg<FMT, D, T>;
  constexpr int TT = C::TT, NW = C::NW, NT = NW * 32;
  constexpr int TU = TT / 16;           // units per tile
  constexpr int DN = D / 8;             // 8-wide columns of O, and MMA steps along D
  constexpr int KW = C::ROWB / 16;      // words of a key row that one thread holds
  constexpr int VW = C::ROWB / 32;      // words of a value row that one thread holds
  constexpr bool F32 = sizeof(T) == 4;
  extern __shared__ __align__(128) uint8_t smem[];
  float *const rec_ml = reinterpret_cast<float *>(smem + C::META);          // [NW][2][m 8, l 8]
  int2 *const rec_row = reinterpret_cast<int2 *>(rec_ml + NW * 32);         // [NW][2]: row, sequence
  int *const scan = reinterpret_cast<int *>(rec_row + NW * 2);
  uint8_t *const table = smem + (kTableAt - kSharedReserved);
  auto before = [=](int b) -> int & { return spare_word(table, b); };
  auto lens = [=](int b) -> int & { return spare_word(table, kMaxBatch + 1 + b); };
  static_assert(2 * kMaxBatch + 1 <= 256 * 32, "words in the free halves");
  const KvView &c = p.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int per_seq = c.kv_heads * p.chunks;             // work rows of one sequence
  // the decode table: word 64 i + lane
  for (int i = tid; i < 256; i += NT) {
    uint32_t v;
    if (FMT == 8) {
      v = posit_to_f32_bits<8, 2>(i);
    } else {
      // bits of code 256 i's value, and the step per code within the block (down for negative codes) over 2^8 as a
      // signed 13-bit number; 1 for the blocks in which the steps differ
      const bool neg = i >= 128;
      const uint32_t m = (neg ? 256 - i : i) * 256, m1 = neg ? m - 1 : m + 1;
      const int32_t step = (int32_t)(bp16_to_f32_bits(m1) - bp16_to_f32_bits(m)) >> 8;
      v = i == 0 || i == 127 || i == 128 || i == 255 ? 1u
                                                     : bp16_to_f32_bits(m) | (neg ? 0x80000000u : 0u) | (step & 0x1FFF);
    }
    uint4 *row = reinterpret_cast<uint4 *>(table) + i * 16;
#pragma unroll
    for (int j = 0; j < 8; ++j) row[(j + i) & 7] = make_uint4(v, v, v, v);
  }
  // (all of the above may run before the kernels ahead in the stream have finished)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  auto length = [&](int b) { return min(c.length(b), p.max_len); };
  auto row_cost = [](int n) { return n > 0 ? (n + 15) / 16 + kRowUnits : 0; };
  // units before each sequence
  {
    const int each = (c.batch + NT - 1) / NT;
    int mine = 0;
    for (int i = 0; i < each; ++i) {
      const int b = tid * each + i;
      if (b < c.batch) {
        const int n = length(b);
        lens(b) = n;
        mine += row_cost(n) * per_seq;
      }
    }
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(~0u, incl, d);
      if (lane >= d) incl += x;
    }
    if (lane == 31) scan[warp] = incl;
    if (tid < NW * 2) rec_row[tid] = make_int2(-1, 0);
    __syncthreads();
    int at = incl - mine;
    for (int w = 0; w < warp; ++w) at += scan[w];
    for (int i = 0; i < each; ++i) {
      const int b = tid * each + i;
      if (b < c.batch) {
        before(b) = at;
        at += row_cost(lens(b)) * per_seq;
      }
    }
    if (tid == NT - 1) before(c.batch) = at;
    __syncthreads();
  }
  const int total = before(c.batch);
  // empty sequences: zeros, and -inf for the logarithm
  for (int b = blockIdx.x; b < c.batch; b += gridDim.x)
    if (before(b + 1) == before(b)) {
      T *o = (T *)p.out + (int64_t)b * p.heads * D;
      for (int i = tid; i < p.heads * D; i += NT) o[i] = from_f32<T>(0.0f);
      if (p.lse)
        for (int i = tid; i < p.heads; i += NT) p.lse[(int64_t)b * p.heads + i] = -INFINITY;
    }
  const int ctas = active_ctas(total, gridDim.x);
  const int cta = blockIdx.x;
  if (cta >= ctas) {
    if (tid == 0) p.cta_row[cta] = make_int2(-1, 0);
    return;
  }
  const Deal deal(total, ctas);
  const int lo = deal.begin(cta), hi = deal.begin(cta + 1);
  const Deal share(hi - lo, NW);
  const int wlo = lo + share.begin(warp), whi = lo + share.begin(warp + 1);

  uint8_t *const stage = smem + C::stage_at(warp);
  uint8_t *const sk = stage, *const sv = stage + C::TILEB;
  int8_t *const ske = reinterpret_cast<int8_t *>(stage + 2 * C::TILEB), *const sve = ske + TT;
  float *const kpow = reinterpret_cast<float *>(stage + 2 * C::TILEB + 2 * TT), *const vpow = kpow + 4 * C::POWROW;
  // ---- where tiles lie: units u .. u + count - 1 of a work row ----
  struct Place {
    int b, row, hk, ch, u, count, n;       // sequence, work row of it (hk * chunks + ch), units, entries of the row
  };
  auto units_of = [](int n) { return (n + 15) / 16; };
  int ax = whi;                // where the tile that is fetched next lies in all the work; from whi on: there is none
  // from tile w, at ax, to the next one
  auto advance = [&](Place &w) {
    ax += w.count;
    w.u += w.count;
    const bool next = w.u >= units_of(w.n);
    if (next) ax += kRowUnits;
    if (ax >= whi) return;
    if (next) {
      w.u = 0;
      ++w.row;
      if (++w.ch == p.chunks) {
        w.ch = 0;
        ++w.hk;
      }
      if (w.row == per_seq) {
        w.row = w.hk = 0;
        do ++w.b;
        while (before(w.b + 1) == before(w.b));
        w.n = lens(w.b);
      }
    }
    w.count = min(min(TU, units_of(w.n) - w.u), whi - ax);
  };
  // Page of the tile's unit `lane` (-1: the tile has no such unit).
  auto page_of = [&](const Place &w) {
    return lane < w.count ? c.table[(int64_t)w.b * c.max_pages + ((w.u + lane) * 16 >> c.page_shift)] : -1;
  };
  const uint32_t stage_s = smem_addr(stage);
  constexpr int CPR = C::ROWB / 16;        // 16-byte pieces per row
  constexpr int PJ = CPR / 2;              // pieces per lane of 16 rows
  // piece `lane` of 16 rows; piece j * 32 + lane lies 512 j behind it, permuted alike (see below for 256-byte rows)
  const uint32_t to = swizzle<C::ROWB>(lane / CPR, lane % CPR);
  // A tile's place in the pools: the rows of its units (the look-up of the pages, this, and the copies are apart, so
  // that none of them waits for the one before).
  struct Rows {
    uint32_t mine, unit[TU];               // this lane's unit's row, and all of them; kNone for a page outside the pool
    bool plain;                            // a whole tile, all of whose pages are there
  };
  constexpr uint32_t kNone = ~0u;          // pools have fewer rows
  auto rows_of = [&](const Place &w, int page, Rows &r) {
    r.mine = (unsigned)page < (unsigned)c.pages ? (uint32_t)c.row(page, w.hk, (w.u + lane) * 16) : kNone;
#pragma unroll
    for (int i = 0; i < TU; ++i) r.unit[i] = __shfl_sync(~0u, r.mine, i);
    bool all = w.n - w.u * 16 >= TT;
#pragma unroll
    for (int i = 0; i < TU; ++i) all = all && r.unit[i] != kNone;
    r.plain = all;
  };
  auto fetch = [&](const Place &w, const Rows &r, bool value) {
    const uint8_t *pool = (value ? c.v : c.k) + lane * 16;
    const uint32_t dst = stage_s + (value ? C::TILEB : 0) + to;
    if (r.plain) {
#pragma unroll
      for (int i = 0; i < TU; ++i) {
        const uint8_t *src = pool + (uint64_t)r.unit[i] * C::ROWB;
#pragma unroll
        for (int j = 0; j < PJ; ++j) {
          const uint32_t d = dst + i * 16 * C::ROWB + j * 512;
          copy16(CPR == 16 && (j & 1) ? d ^ 64 : d, src + j * 512);
        }
      }
    } else {
      const int valid = w.n - w.u * 16;
#pragma unroll 1
      for (int i = 0; i < w.count; ++i) {
        const uint32_t row = __shfl_sync(~0u, r.mine, i);
        const uint8_t *src = pool + (uint64_t)row * C::ROWB;
#pragma unroll
        for (int j = 0; j < PJ; ++j) {
          const uint32_t d = dst + i * 16 * C::ROWB + j * 512;
          if (row != kNone && i * 16 + (j * 32 + lane) / CPR < valid) copy16(CPR == 16 && (j & 1) ? d ^ 64 : d, src + j * 512);
        }
      }
    }
    if (FMT == 8 && r.mine != kNone)
      copy16(stage_s + 2 * C::TILEB + (value ? TT : 0) + lane * 16, (value ? c.v_exp : c.k_exp) + r.mine);
    copy_commit();
  };

  Place cur{}, ahead{};        // this tile, and the next to be fetched
  Rows rows{};
  int page = -1;
  bool bad = false;            // a page of the tile is outside the pool
  auto is_bad = [&](const Place &w, int pg) { return __any_sync(~0u, lane < w.count && (unsigned)pg >= (unsigned)c.pages); };
  bool first = false;          // there is a tile, and it is the first one
  if (wlo < whi) {
    int a = 0, z = c.batch;                // sequence of the first unit, by bisection
    while (z - a > 1) {
      const int half = (a + z) >> 1;
      if (before(half) <= wlo) a = half;
      else z = half;
    }
    cur.b = a;
    cur.n = lens(a);
    const int r = wlo - before(a), nu = units_of(cur.n);
    cur.row = r / (nu + kRowUnits);
    const int in_row = r - cur.row * (nu + kRowUnits) - kRowUnits;
    cur.u = max(in_row, 0);
    ax = wlo + max(-in_row, 0);
    first = ax < whi;
    cur.hk = p.chunks == 1 ? cur.row : cur.row / p.chunks;
    cur.ch = cur.row - cur.hk * p.chunks;
    cur.count = min(min(TU, nu - cur.u), whi - ax);
  }
  if (first) {
    ahead = cur;
    page = page_of(ahead);
    rows_of(ahead, page, rows);
    bad = is_bad(ahead, page);
    fetch(ahead, rows, false);
    fetch(ahead, rows, true);
    advance(ahead);
  }
  __syncthreads();
  const uint32_t entry = lane * 4 | (kTableAt >> 16) << 8;
  constexpr int CW = 4 / C::BYTES;      // codes per word

  // The thread's place in the fragments: head g of A and of the accumulators; column g of S is entry `er` of its 8
  // entries, and the accumulators' columns 2t and 2t + 1 (K of the second product: t and t + 4) are entries t and
  // 4 + (t ^ 1) -- an order in which neighbouring quads read rows of different banks.
  const int er = (g & 1) ? 4 + ((g >> 1) ^ 1) : g >> 1;
  const int e0 = t, e1 = 4 + (t ^ 1);
  uint32_t qf[DN][F32 ? 4 : 2];
  float o[DN][2], m = -INFINITY, l = 0.0f;

  bool lost = false;
  int at_row = 0;                          // first unit of the current row that this warp has

  // The three stages of a step over U units, from unit i0 of the stage on.
  // S[head, entry] = q K^T
  auto scores_with = [&](auto exact, auto &s, int i0) {
    uint32_t odd = 0;
    constexpr int SN = sizeof(s) / sizeof(s[0]);
    // four columns at a time: an MMA waits for the one before it in its sum
    constexpr int G = SN < 4 ? SN : 4;
#pragma unroll
    for (int i = 0; i < SN; i += G) {
      uint32_t kw[G][KW];
      float c4[G][4];
#pragma unroll
      for (int k = 0; k < G; ++k) load_words<C::ROWB>(sk + (i0 * 16 + (i + k) * 8) * C::ROWB, er, t * KW, kw[k]);
#pragma unroll
      for (int w = 0; w < DN; ++w) {
        const uint32_t a[4] = {qf[w][0], F32 ? qf[w][1] : 0u, qf[w][F32 ? 2 : 1], F32 ? qf[w][F32 ? 3 : 0] : 0u};
#pragma unroll
        for (int k = 0; k < G; ++k) {
          const uint32_t b0 = decode_code<FMT, decltype(exact)::value>(entry, kw[k][2 * w / CW], 2 * w % CW, odd);
          const uint32_t b1 = decode_code<FMT, decltype(exact)::value>(entry, kw[k][2 * w / CW], 2 * w % CW + 1, odd);
          if (w == 0) mma_tf32_first(c4[k], a, b0, b1);
          else mma_tf32(c4[k], a, b0, b1);
        }
      }
#pragma unroll
      for (int k = 0; k < G; ++k) {
        s[i + k][0] = F32 ? c4[k][0] + c4[k][2] : c4[k][0];
        s[i + k][1] = F32 ? c4[k][1] + c4[k][3] : c4[k][1];
      }
    }
    return odd;
  };
  auto scores = [&](auto &s, int i0) {
    const uint32_t odd = scores_with(std::false_type{}, s, i0);
    if (FMT == 16 && __any_sync(~0u, odd & 1u)) scores_with(std::true_type{}, s, i0);
  };
  // S becomes e^(S - maximum), maximum and sum move on; returns the factor for what was summed before
  auto weights = [&](auto &s, int i0, int valid) {
    constexpr int SN = sizeof(s) / sizeof(s[0]);
#pragma unroll
    for (int i = 0; i < SN; i += 2) {
      float4 f = make_float4(p.scale, p.scale, p.scale, p.scale);
      if (FMT == 8) f = *reinterpret_cast<const float4 *>(kpow + t * C::POWROW + 4 * i0 + 2 * i);
      s[i][0] *= f.x;
      s[i][1] *= f.y;
      s[i + 1][0] *= f.z;
      s[i + 1][1] *= f.w;
    }
    if (SN == 2) {             // only a unit by itself can end behind the length
#pragma unroll
      for (int i = 0; i < SN; ++i) {
        if (i * 8 + e0 >= valid) s[i][0] = -INFINITY;
        if (i * 8 + e1 >= valid) s[i][1] = -INFINITY;
      }
    }
    if (p.raw && g < p.gp) {
      float *raw = p.raw + (((int64_t)cur.b * per_seq + cur.row) * p.max_len + (cur.u + i0) * 16) * p.gp + g;
#pragma unroll
      for (int i = 0; i < SN; ++i) {
        if (SN > 2 || i * 8 + e0 < valid) raw[(i * 8 + e0) * p.gp] = s[i][0];
        if (SN > 2 || i * 8 + e1 < valid) raw[(i * 8 + e1) * p.gp] = s[i][1];
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < SN; i += 2) mx = fmaxf(mx, fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i + 1][0], s[i + 1][1])));
    mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 2));
    mx = fmaxf(m, mx);
    const float at = finite_max(mx);
    const float alpha = ex2(m - at);
    m = mx;
    float sum[4] = {l * alpha, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < SN; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s[i][j] = ex2(s[i][j] - at);
        sum[(2 * i + j) & 3] += s[i][j];
      }
    l = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    return alpha;
  };
  // O[head, d] = alpha O + P V
  // (columns part * DH .. of each thread's DN: wide rows in two parts, for fewer registers)
  constexpr int DH = DN / C::PARTS, VH = VW / C::PARTS;
  auto values_with = [&](auto exact, const auto &s, int i0, int part, auto &acc) {
    uint32_t odd = 0;
    constexpr int SN = sizeof(s) / sizeof(s[0]);
#pragma unroll
    for (int i = 0; i < SN; ++i) {
      float w0 = s[i][0], w1 = s[i][1];
      if (FMT == 8) {      // (entries behind the length have weight 0 and any exponent: 0 times a finite power)
        const float2 f = *reinterpret_cast<const float2 *>(vpow + t * C::POWROW + 4 * i0 + 2 * i);
        w0 *= f.x;
        w1 *= f.y;
      }
      const uint32_t a[4] = {tf32_high(w0), tf32_high(w0 - __uint_as_float(tf32_high(w0))), tf32_high(w1),
                             tf32_high(w1 - __uint_as_float(tf32_high(w1)))};
      uint32_t v0[VH], v1[VH];
      const uint8_t *r = sv + (i0 * 16 + i * 8) * C::ROWB;
      load_words<C::ROWB>(r, e0, g * VW + part * VH, v0);
      load_words<C::ROWB>(r, e1, g * VW + part * VH, v1);
#pragma unroll
      for (int d = 0; d < DH; ++d) {
        const uint32_t b0 = decode_code<FMT, decltype(exact)::value>(entry, v0[d / CW], d % CW, odd);
        const uint32_t b1 = decode_code<FMT, decltype(exact)::value>(entry, v1[d / CW], d % CW, odd);
        if (i == 0) mma_tf32_first(acc[d], a, b0, b1);
        else mma_tf32(acc[d], a, b0, b1);
      }
    }
    return odd;
  };
  auto values = [&](const auto &s, int i0, float alpha) {
#pragma unroll
    for (int part = 0; part < C::PARTS; ++part) {
      float acc[DH][4];
      const uint32_t odd = values_with(std::false_type{}, s, i0, part, acc);
      if (FMT == 16 && __any_sync(~0u, odd & 1u)) values_with(std::true_type{}, s, i0, part, acc);
#pragma unroll
      for (int d = 0; d < DH; ++d) {
        float *out = o[part * DH + d];
        out[0] = fmaf(out[0], alpha, acc[d][0] + acc[d][2]);
        out[1] = fmaf(out[1], alpha, acc[d][1] + acc[d][3]);
      }
    }
  };
  // each exponent of the tile is turned into a power of two once, and read back by the four threads that need it
  auto powers = [&](const int8_t *exps, float *pow, float scale) {
    if constexpr (FMT == 8) {
#pragma unroll
      for (int i = 0; i < TT / 32; ++i) {
        const int e = i * 32 + lane, y = e & 7;
        pow[(y < 4 ? y : (y - 4) ^ 1) * C::POWROW + (e >> 3) * 2 + (y >> 2)] = exp2_int(exps[e]) * scale;
      }
    }
  };

  for (bool go = first; go;) {
    // the pages of the tile to be fetched are looked up while this one's keys are worked on
    const bool more = ax < whi;
    if (more) page = page_of(ahead);
    lost |= bad;
    if (first || cur.u == 0) {             // a new row: its queries (while its keys are on their way), an empty state
      const uint4 *q = reinterpret_cast<const uint4 *>(
          (const T *)p.q + cur.b * p.qs + (int64_t)(cur.hk * p.group + cur.ch * kHeadsPerRow + g) * D + t * (D / 4));
      constexpr int QV = D / 4 * sizeof(T) / 16;
      const bool real = cur.ch * kHeadsPerRow + g < p.group;
      uint4 raw[QV];
#pragma unroll
      for (int i = 0; i < QV; ++i) raw[i] = real ? q[i] : make_uint4(0, 0, 0, 0);
      T f[D / 4];
      memcpy(f, raw, sizeof f);
#pragma unroll
      for (int s = 0; s < DN; ++s)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float y = to_f32(f[2 * s + j]);
          if (F32) {
            qf[s][2 * j] = tf32_high(y);
            qf[s][2 * j + 1] = to_tf32(y - __uint_as_float(tf32_high(y)));
          } else {
            qf[s][j] = __float_as_uint(y);     // bf16 and fp16 are tf32 values
          }
        }
#pragma unroll
      for (int i = 0; i < DN; ++i) o[i][0] = o[i][1] = 0.0f;
      m = -INFINITY;
      l = 0.0f;
      at_row = cur.u;
      lost = bad;
    }
    copy_wait<1>();
    const int valid = cur.n - cur.u * 16;
    if (TU == 1 || (cur.count == TU && valid >= TT)) {
      float s[TT / 8][2];
      scores(s, 0);
      if (more) rows_of(ahead, page, rows);
      copy_wait<0>();
      powers(ske, kpow, p.scale);
      powers(sve, vpow, 1.0f);
      __syncwarp();
      if (more) fetch(ahead, rows, false);
      else copy_commit();
      values(s, 0, weights(s, 0, valid));
      __syncwarp();
      if (more) fetch(ahead, rows, true);
      else copy_commit();
    } else {
      copy_wait<0>();
      powers(ske, kpow, p.scale);
      powers(sve, vpow, 1.0f);
      __syncwarp();
#pragma unroll 1
      for (int i = 0; i < cur.count; ++i) {
        float s[2][2];
        scores(s, i);
        values(s, i, weights(s, i, valid - i * 16));
      }
      __syncwarp();
      if (more) {
        rows_of(ahead, page, rows);
        fetch(ahead, rows, false);
        fetch(ahead, rows, true);
      }
    }

    // ---- the end of a row, or of this warp's range ----
    const bool ended = cur.u + cur.count == units_of(cur.n);
    if (ended || !more) {
      l += __shfl_xor_sync(~0u, l, 1);
      l += __shfl_xor_sync(~0u, l, 2);
      if (lost) l = NAN;
      const int row = cur.b * per_seq + cur.row;
      // this thread holds head g, columns t D/4 .. (t + 1) D/4
      if (at_row == 0 && ended) {
        const int64_t head = head_of(p, RowId{cur.b, cur.hk, cur.ch}, g);
        if (head >= 0) {
          const float inv = 1.0f / l;
          T f[D / 4];
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int d = 0; d < DN; ++d) f[j * DN + d] = from_f32<T>(o[d][j] * inv);
          uint4 raw[sizeof f / 16];
          memcpy(raw, f, sizeof f);
          uint4 *out = reinterpret_cast<uint4 *>((T *)p.out + head * D + t * (D / 4));
#pragma unroll
          for (int i = 0; i < (int)(sizeof f / 16); ++i) out[i] = raw[i];
        }
        if (t == 0) write_lse(p, row, g, head, m + log2f(l));
      } else {
        // a part: inside the range it goes to the workspace (the stage holds the next tile), at its end to the stage
        const int slot = more ? 0 : 1;
        float4 *rec = reinterpret_cast<float4 *>(
            (more ? p.warp_rec + ((int64_t)cta * NW + warp) * C::REC : reinterpret_cast<float *>(stage)) + g * D +
            t * (D / 4));
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int d = 0; d < DN; d += 4)
            rec[(j * DN + d) / 4] = make_float4(o[d][j], o[d + 1][j], o[d + 2][j], o[d + 3][j]);
        if (t == 0) {
          rec_ml[(warp * 2 + slot) * 16 + g] = m;
          rec_ml[(warp * 2 + slot) * 16 + 8 + g] = l;
        }
        if (lane == 0) rec_row[warp * 2 + slot] = make_int2(row, cur.b);
      }
    }
    go = more;
    first = false;
    cur = ahead;
    if (more) {
      bad = is_bad(ahead, page);
      advance(ahead);
    }
  }
  __syncthreads();

  // ---- join the parts of this CTA's rows: a warp takes a head, a lane one part's statistics and D / 32 columns ----
  // (a row has at most one part in the workspace, its last one here: it ended inside a warp's range)
  static_assert(NW * 2 <= 32 && NW >= kHeadsPerRow, "a part per lane, a head per warp");
  int2 open = make_int2(-1, 0);
  const int2 mine = lane < NW * 2 ? rec_row[lane] : make_int2(-1, 0);
  for (uint32_t left = __ballot_sync(~0u, mine.x >= 0); left;) {
    const int from = __ffs(left) - 1, h = warp;
    const int row = __shfl_sync(~0u, mine.x, from), b = __shfl_sync(~0u, mine.y, from);
    const bool in = mine.x == row;
    const uint32_t parts = __ballot_sync(~0u, in);
    left &= ~parts;
    const int in_seq = row - b * per_seq, nu = units_of(lens(b));
    const int x0 = before(b) + in_seq * (nu + kRowUnits) + kRowUnits, x1 = x0 + nu;
    // (the CTA that holds the row's last unit is the last one with a part)
    if (x0 >= lo && x1 > hi) {
      open = make_int2(row, deal.part_of(x1 - 1) - cta + 1);
      if (p.row_parts && tid == 0) p.row_parts[row] = make_int2(cta, open.y);
    }
    if (h >= kHeadsPerRow) continue;
    const float mp = in ? rec_ml[lane * 16 + h] : -INFINITY;
    float M = mp;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, d));
    const float a = in ? ex2(mp - finite_max(M)) : 0.0f;
    float L = in ? rec_ml[lane * 16 + 8 + h] * a : 0.0f, O[D / 32];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) L += __shfl_xor_sync(~0u, L, d);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) O[i] = 0.0f;
    // (read from every stage at once; what is no part of this row is left out)
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __shfl_sync(~0u, a, 2 * w + 1);
      const float *r = reinterpret_cast<const float *>(smem + C::stage_at(w)) + h * D + lane;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const float y = r[i * 32];
        O[i] = parts >> (2 * w + 1) & 1 ? fmaf(y, f, O[i]) : O[i];
      }
    }
    if (const uint32_t last = parts & 0x55555555u) {
      const int k = __ffs(last) - 1;
      const float f = __shfl_sync(~0u, a, k);
      const float *r = p.warp_rec + ((int64_t)cta * NW + (k >> 1)) * C::REC + h * D + lane;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) O[i] = fmaf(r[i * 32], f, O[i]);
    }
    if (x0 >= lo && x1 <= hi) {
      const int hk = p.chunks == 1 ? in_seq : in_seq / p.chunks;
      const int64_t head = head_of(p, RowId{b, hk, in_seq - hk * p.chunks}, h);
      if (head >= 0) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) ((T *)p.out)[head * D + i * 32 + lane] = from_f32<T>(O[i] / L);
      }
      if (lane == 0) write_lse(p, row, h, head, M + log2f(L));
    } else {
      float *out = p.cta_rec + (cta * 2 + (x0 >= lo)) * (C::REC + 16);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) out[h * D + i * 32 + lane] = O[i];
      if (lane == 0) {
        out[C::REC + h] = M;
        out[C::REC + 8 + h] = L;
      }
    }
  }
  if (tid == 0) p.cta_row[cta] = open;
}

}  // namespace

// Launches the instance for (fmt, D, dtype) on `grid` CTAs.
int launch_kv_attend8(const AttendParams &p, int dtype, int grid, cudaStream_t s);
int launch_kv_attend16(const AttendParams &p, int dtype, int grid, cudaStream_t s);

template <int FMT, int D, typename T>
int launch_kv_attend_one(const AttendParams &p, int grid, cudaStream_t s) {
  using C = AttendCfg<FMT, D, T>;
  static_assert(C::SMEM <= 232448, "shared memory per CTA");
  static std::atomic<bool> ready[128];       // per device: the opt-in to shared memory, and where it starts
  int device = 0, reserved = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 128)
    return set_error(kENoDev, "k_kv_attend: no device");
  if (!ready[device].load(std::memory_order_relaxed)) {
    if (cudaDeviceGetAttribute(&reserved, cudaDevAttrReservedSharedMemoryPerBlock, device) != cudaSuccess ||
        reserved != kSharedReserved)
      return set_error(kENoDev, "k_kv_attend: shared memory starts at %d, not %d", reserved, kSharedReserved);
    cudaError_t e = cudaFuncSetAttribute(k_kv_attend<FMT, D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return set_error(kECuda, "k_kv_attend: %s", cudaGetErrorString(e));
    ready[device].store(true, std::memory_order_relaxed);
  }
  return launch_early(k_kv_attend<FMT, D, T>, dim3(grid), C::NW * 32, C::SMEM, s, "k_kv_attend", p);
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
