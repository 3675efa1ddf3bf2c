// topk_warp.cuh — the 32 largest keys of many, one a lane of a warp in
// descending order (0: no entry).
#pragma once

#include "score.cuh"

namespace har {

using key_t = unsigned long long;

template <typename K>
__device__ __forceinline__ K key_max(K a, K b) { return a > b ? a : b; }

// Descending bitonic sort of one key a lane.  Rolled: where it runs once, its
// instructions come from L2.
template <typename K>
__device__ __forceinline__ K warp_sort_desc(K v, int lane) {
#pragma unroll 1
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll 1
    for (int step = size >> 1; step > 0; step >>= 1) {
      const K o = __shfl_xor_sync(0xffffffffu, v, step);
      const bool keep_max = ((lane & step) == 0) == ((lane & size) == 0);
      v = (o > v) == keep_max ? o : v;
    }
  return v;
}
// The largest of v over the warp, which one lane that has it then gives up.
__device__ __forceinline__ uint32_t warp_pop_max(uint32_t &v, int lane) {
  const uint32_t m = __reduce_max_sync(0xffffffffu, v);
  if (lane == __ffs(__ballot_sync(0xffffffffu, v == m)) - 1) v = 0;
  return m;
}
// The k-th largest (1 to 32) of one value a lane, from the nearer end.
__device__ __forceinline__ uint32_t warp_kth(uint32_t v, int k, int lane) {
  const uint32_t flip = k <= 16 ? 0u : ~0u;
  uint32_t m = 0;
  v ^= flip;
#pragma unroll 1
  for (int i = k <= 16 ? k : 33 - k; i > 0; --i) m = warp_pop_max(v, lane);
  return m ^ flip;
}
// The 32 largest of two descending lists, descending.
template <typename K>
__device__ __forceinline__ K warp_merge_desc(K a, K b, int lane) {
  K v = key_max(a, __shfl_sync(0xffffffffu, b, 31 - lane));
#pragma unroll
  for (int step = 16; step > 0; step >>= 1) {
    const K o = __shfl_xor_sync(0xffffffffu, v, step);
    v = (o > v) == ((lane & step) == 0) ? o : v;
  }
  return v;
}
// Takes the keys of the lanes in `mask` into a descending list: a few one by
// one, many with a sort and a merge.  The whole warp.
__device__ __forceinline__ key_t warp_take(key_t list, key_t key, uint32_t mask, int lane) {
  if (__popc(mask) > 6)
    return warp_merge_desc(list, warp_sort_desc((mask >> lane) & 1u ? key : (key_t)0, lane), lane);
  for (; mask; mask &= mask - 1) {
    const key_t k = __shfl_sync(0xffffffffu, key, __ffs(mask) - 1);
    const int pos = __popc(__ballot_sync(0xffffffffu, list > k));
    const key_t up = __shfl_up_sync(0xffffffffu, list, 1);
    list = lane < pos ? list : lane == pos ? k : up;
  }
  return list;
}

// The 32 largest of n different keys in shared memory, in descending order (0
// behind the last): every key counts those above it.  The whole block of
// `threads`, between barriers; `sorted` was zeroed before the first.
__device__ __forceinline__ void block_rank(const key_t *keys, int n, key_t *sorted, int tid, int threads) {
  for (int i = tid; i < n; i += threads) {
    const key_t mine = keys[i];
    int above = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) above += keys[j] > mine;
    if (above < 32) sorted[above] = mine;
  }
}

// n (a power of two, at most twice the block's warps) descending lists at
// lists[i][32] -> their 32 largest in warp 0.  The whole block calls it, after
// a barrier that follows the lists' writes; it ends with a barrier.
template <typename K>
__device__ __forceinline__ K block_merge_lists(K (*lists)[32], int n, int warp, int lane) {
  K v = warp < n ? lists[warp][lane] : (K)0;
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
