// The kernel for many query rows over each user's own keys.
#include "cache8_tile.cuh"

int cxs::cache8::launch_tile(const cxs_cache_attend_call& a, const Shape& z, cudaStream_t stream) {
  return launch_of<false>(a, z, SharedPlan{}, stream);
}
