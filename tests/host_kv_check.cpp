// host_kv_check.cpp -- the cache's bp8 row encoder (bp_format.cuh) as a host library.  Test-only.
#include <stddef.h>

#include "../open-bposit_b200/csrc/bp_format.cuh"

extern "C" void kv_encode_bp8(const uint32_t *u, size_t n, int e, uint8_t *out) {
  for (size_t i = 0; i < n; ++i) out[i] = (uint8_t)bp::bp8_encode_exp(u[i], e);
}
extern "C" void kv_floor_log2(const uint32_t *a, size_t n, int *out) {
  for (size_t i = 0; i < n; ++i) out[i] = bp::f32_floor_log2(a[i]);
}
// The closed forms where they hold, the general ones elsewhere.
extern "C" void kv_encode_near(const uint32_t *u, size_t n, int fmt, uint32_t *out) {
  for (size_t i = 0; i < n; ++i) {
    const uint32_t a = u[i] & 0x7FFFFFFFu;
    uint32_t m = fmt == 8 ? (bp::bp8_in_range(a) ? bp::bp8_encode_near(a) : bp::bp8_encode_exp(a, 0))
                          : (bp::bp16_in_range(a) ? bp::bp16_encode_near(a) : bp::bp16_encode_bits(a, true));
    out[i] = (u[i] >> 31 ? 0u - m : m) & (fmt == 8 ? 0xFFu : 0xFFFFu);
  }
}
