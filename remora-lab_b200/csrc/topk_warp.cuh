// topk_warp.cuh — a warp's running list of the 32 largest keys, one per lane
// in descending order (0: empty), and the buffer new candidates wait in.
#pragma once

#include "score.cuh"

namespace har {

using key_t = unsigned long long;

__device__ __forceinline__ key_t key_max(key_t a, key_t b) { return a > b ? a : b; }

// Descending bitonic sort of one key a lane.
__device__ __forceinline__ key_t warp_sort_desc(key_t v, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int step = size >> 1; step > 0; step >>= 1) {
      const key_t o = __shfl_xor_sync(0xffffffffu, v, step);
      const bool keep_max = ((lane & step) == 0) == ((lane & size) == 0);
      v = (o > v) == keep_max ? o : v;
    }
  return v;
}
// The 32 largest of two descending lists, descending.
__device__ __forceinline__ key_t warp_merge_desc(key_t a, key_t b, int lane) {
  key_t v = key_max(a, __shfl_sync(0xffffffffu, b, 31 - lane));
#pragma unroll
  for (int step = 16; step > 0; step >>= 1) {
    const key_t o = __shfl_xor_sync(0xffffffffu, v, step);
    v = (o > v) == ((lane & step) == 0) ? o : v;
  }
  return v;
}

// n (a power of two, at most twice the block's warps) descending lists at
// lists[i][32] -> their 32 largest in warp 0.  The whole block calls it, after
// a barrier that follows the lists' writes.
__device__ __forceinline__ key_t block_merge_lists(key_t (*lists)[32], int n, int warp, int lane) {
  key_t v = warp < n ? lists[warp][lane] : 0;
  for (int half = n >> 1; half > 0; half >>= 1) {
    if (warp < half) {
      v = warp_merge_desc(v, lists[warp + half][lane], lane);
      if (half > 1) lists[warp][lane] = v;  // read by nobody else before the barrier
    }
    __syncthreads();
  }
  return v;
}

}  // namespace har
