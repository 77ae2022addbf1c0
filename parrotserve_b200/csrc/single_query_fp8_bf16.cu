// Single-query attention over the 8-bit cache, queries in bf16: all head and block sizes.
#include "single_query_fp8.cuh"

namespace pb {

cudaError_t launch_single_query_fp8_bf16(const AttnDev& d, int head_size, int block_size, cudaStream_t s) {
  return launch_sq8_all<__nv_bfloat16>(d, head_size, block_size, s);
}

}  // namespace pb
