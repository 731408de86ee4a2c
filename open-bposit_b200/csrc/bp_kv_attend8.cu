// bp_kv_attend8.cu -- instances of the one-token attention kernel for bp8 caches.
#include "bp_kv_attend.cuh"

namespace bp {
int launch_kv_attend8(const AttendParams &p, int dtype, int grid, cudaStream_t s) {
  return launch_kv_attend_fmt<8>(p, dtype, grid, s);
}
}  // namespace bp
