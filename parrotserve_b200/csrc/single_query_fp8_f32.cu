// Single-query attention over the 8-bit cache, queries in f32: all head and block sizes.
#include "single_query_fp8.cuh"

namespace pb {

cudaError_t launch_single_query_fp8_f32(const AttnDev& d, int head_size, int block_size, cudaStream_t s) {
  return launch_sq8_all<float>(d, head_size, block_size, s);
}

}  // namespace pb
