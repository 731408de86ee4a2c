// bp_kv_attend16.cu -- instances of the one-token attention kernel for bp16 caches.
#include "bp_kv_attend.cuh"

namespace bp {
int launch_kv_attend16(const AttendParams &p, int dtype, int grid, cudaStream_t s) {
  return launch_kv_attend_fmt<16>(p, dtype, grid, s);
}
}  // namespace bp
