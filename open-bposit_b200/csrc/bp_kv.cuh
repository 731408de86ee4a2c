// bp_kv.cuh -- the paged key-value cache as the kernels see it (bp_kv_cache in
// include/bposit_b200.h, one layer selected), shared by bp_kv_append.cu,
// bp_kv_attend.cu and bp_kv_evict.cu.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/bposit_b200.h"
#include "bp_internal.cuh"

namespace bp {

struct KvView {
  int fmt, layers, pages, page_shift, kv_heads, dim, batch, max_pages, cap;
  uint8_t *k, *v;            // this layer's codes
  int8_t *k_exp, *v_exp;     // this layer's exponents (fmt 8)
  const int32_t *table, *lengths;
  int32_t *positions;        // this layer's, optional
  float *scores;
  int64_t layer_rows;        // (token, kv head) rows of one layer's pools

  __device__ __forceinline__ int length(int b) const {
    const int n = lengths[b];
    return n < 0 ? 0 : (n > cap ? cap : n);
  }
  // Page that holds entry i of sequence b, -1 when the table names none of the pool's.
  __device__ __forceinline__ int page_of(int b, int i) const {
    const int p = table[(int64_t)b * max_pages + (i >> page_shift)];
    return (unsigned)p < (unsigned)pages ? p : -1;
  }
  // Row of (page, kv head, entry) in the pools: a 64-bit count, pools pass 2^31 elements.
  __device__ __forceinline__ int64_t row(int page, int hk, int i) const {
    return (((int64_t)page * kv_heads + hk) << page_shift) + (i & ((1 << page_shift) - 1));
  }
};

// Argument checks common to the cache's entry points; fills `view` for `layer`.
int kv_check(const bp_kv_cache *c, int layer, const char *what, KvView *view);

// Whether contiguous results out [rows, width] lie on inputs in [rows, stride], other than row for row in their place:
// on a row that may be read after they were written.
inline bool crosses(const void *in, int64_t stride, const void *out, int64_t rows, int64_t width, int element) {
  if (rows < 1 || (in == out && (stride == width || rows == 1))) return false;
  const int64_t d = (int64_t)((intptr_t)out - (intptr_t)in), s = stride * element, w = width * element, n = rows * w;
  if (d < 0) return d + n > 0;
  const int64_t r = d / s;               // the row that starts at `out` or before it
  return (r < rows && d - r * s < w) || (r + 1 < rows && (r + 1) * s < d + n);
}

// Launches a kernel that begins with, or comes to, griddepcontrol.wait before it
// touches memory that earlier work of the stream writes: its start overlaps the
// end of the kernel ahead.
template <typename K, typename... P>
int launch_early(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t s, const char *what, const P &...params) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, params...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(kECuda, "%s: %s", what, cudaGetErrorString(e));
  }
  return check_launch(what);
}

template <typename T>
__device__ __forceinline__ float to_f32(T x) { return (float)x; }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x) { return (T)x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }

// 2^e for any int8 e, exactly (-127 and -128 are subnormal).
__device__ __forceinline__ float exp2_int(int e) {
  return __uint_as_float(e >= -126 ? (uint32_t)(e + 127) << 23 : 0x00400000u >> (-127 - e));
}

}  // namespace bp
