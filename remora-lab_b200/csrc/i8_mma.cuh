// i8_mma.cuh — the tensor-core pipeline that the 8-bit kernels share: TMA
// producers, the MMA issuer, and the barriers between them and an epilogue.
//
//   D[A rows][B rows] = A [rows][K] * B [rows][K]^T, 32-bit sums in TMEM.
//
// CG = 1: a block computes tiles of 128 A rows x bn B rows.  CG = 2: a cluster
// of two computes tiles of 256 x bn; each block loads its own 128 rows of A and
// half the rows of B, so at bn = 256 a k-step of 128 bytes brings 32 KB into a
// block's shared memory for the products that cost a lone block 48 KB.  Either
// takes max(2 bn, 315) cycles once the bytes are there; with 148 blocks loading
// from memory and L2 (256 x 18,944 x 8,192) it took 983 cycles alone and 838 in
// pairs.  A lone tile's advantage is its size: half the channels, so fewer
// blocks stand idle in the last round of a product of few tiles.
#pragma once

#include "score.cuh"
#include "tc_ptx.cuh"

namespace har {

constexpr int G_A = 128, G_KS = 128, G_MAX_BN = 256;
constexpr int G_STAGE_BYTES = 160 * 1024, G_MAX_STAGES = 12;
constexpr int G_WARP_A = 0, G_WARP_MMA = 1, G_WARP_B = 2, G_WARP_EPI = 3, G_EPI_WARPS = 8;
constexpr int G_EPI_THREADS = 32 * G_EPI_WARPS;
constexpr int G_THREADS = 32 * G_WARP_EPI + G_EPI_THREADS;
constexpr uint32_t G_WAIT_LIMIT = 1u << 22;

struct Ring {
  uint64_t full[G_MAX_STAGES], empty[G_MAX_STAGES], acc_full[2], acc_empty[2];
  uint32_t tmem;
  int abort_flag;
};

// What every role knows: K, the k-steps [k0, k1) of it that a tile takes, the
// tile's columns, ring slots.
struct RingShape {
  int64_t K;
  int k0, k1;
  int bn, stages;
};
inline int ksteps_of(int64_t K) { return (int)((K + G_KS - 1) / G_KS); }

// A whole warp, lane 0 between polls asleep for up to sleep_ns.
__device__ __forceinline__ bool g_wait_warp(uint64_t *bar, uint32_t parity, volatile int *abort_s, int lane,
                                            uint32_t sleep_ns) {
  if (__all_sync(0xffffffffu, tc::mbar_try_wait(bar, parity))) return true;
  bool ok = true;
  if (lane == 0) {
    ok = !*abort_s && tc::mbar_wait_lazy(bar, parity, G_WAIT_LIMIT, sleep_ns);
    if (!ok) *abort_s = 1;
  }
  return __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
}
// The same for the roles that feed the tensor core: every step of it decided by
// a vote, so that the loop around it stays uniform and its descriptors,
// addresses and counters in uniform registers (see elect_one).
__device__ __forceinline__ bool g_wait_uniform(uint64_t *bar, uint32_t parity, volatile int *abort_s) {
  for (uint32_t i = 0; i < G_WAIT_LIMIT; ++i) {
    if (__all_sync(0xffffffffu, tc::mbar_try_wait(bar, parity))) return true;
    if (__any_sync(0xffffffffu, *abort_s)) return false;
  }
  *abort_s = 1;
  return false;
}

template <int CG>
__device__ __forceinline__ void ring_open(Ring &r, const RingShape &sh, const void *map_a, const void *map_b) {
  const int tid = threadIdx.x;
  if (tid < 32) {
    if (CG == 2) {
      tc::tmem_alloc_pair(&r.tmem, 512);
      tc::tmem_relinquish_pair();
    } else {
      tc::tmem_alloc(&r.tmem, 512);
      tc::tmem_relinquish();
    }
  }
  if (tid == 32) {
    for (int s = 0; s < sh.stages; ++s) {
      tc::mbar_init(r.full + s, 2);  // both producers
      tc::mbar_init(r.empty + s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      tc::mbar_init(r.acc_full + a, 1);
      tc::mbar_init(r.acc_empty + a, CG * G_EPI_WARPS);
    }
    tc::fence_mbar_init();
    r.abort_flag = 0;
  }
  if (tid == 64) {
    tc::tma_prefetch_desc(map_a);
    tc::tma_prefetch_desc(map_b);
  }
  tc::tc_fence_before();
  __syncthreads();
  if (CG == 2) {  // the peer's barriers are initialised before anything arrives on them
    tc::cluster_arrive();
    tc::cluster_wait();
  }
  tc::tc_fence_after();
}

template <int CG>
__device__ __forceinline__ void ring_close(Ring &r, int *status) {
  // a producer's lane rejoins its warp before the warp-wide instructions below
  __syncwarp();
  __syncthreads();
  if (*(volatile int *)&r.abort_flag) {
    if (threadIdx.x == 0) atomicOr(status, DEV_ERR_TIMEOUT);
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);  // let copies and MMAs in flight land
  }
  tc::tc_fence_before();
  __syncthreads();
  if (CG == 2) {  // neither block leaves while the other's MMAs or arrivals may reach it
    tc::cluster_arrive();
    tc::cluster_wait();
  }
  tc::tc_fence_after();
  if (threadIdx.x < 32) {
    if (CG == 2) tc::tmem_dealloc_pair(r.tmem, 512);
    else tc::tmem_dealloc(r.tmem, 512);
  }
}

// The ring slot of the next k-step, and the parity of the phase that it is in.
// Counted along: two divisions a k-step made a loop of one lane's instructions
// 640 cycles long, more than the MMAs of the largest tile (512).
struct Slot {
  uint32_t s = 0, phase = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++s == (uint32_t)stages) s = 0, phase ^= 1u;
  }
};

// One warp loads the A boxes, another the B boxes, of the tiles that `tiles`
// names: tiles.next(a_row, b_row).
template <int CG, typename Tiles>
__device__ __forceinline__ void ring_produce(Ring &r, const RingShape &sh, uint8_t *sm, bool is_b, const void *map,
                                             Tiles tiles, uint32_t rank) {
  volatile int *abort_s = &r.abort_flag;
  const int b_rows = sh.bn / CG;
  const uint32_t lead = tc::elect_one(), even = CG == 2 ? tc::cluster_rank() & ~1u : 0u;
  const uint32_t a_bytes = G_A * G_KS, b_bytes = (uint32_t)b_rows * G_KS, bytes = is_b ? b_bytes : a_bytes;
  const uint32_t full = tc::smem_u32(r.full), full_even = CG == 2 ? tc::map_rank(full, even) : full;
  const uint32_t dst = tc::smem_u32(sm) + (is_b ? a_bytes : 0u);
  Slot at;
  int a_row, b_row;
  while (tiles.next(a_row, b_row)) {
    const int row = is_b ? b_row + (int)rank * b_rows : a_row + (int)rank * G_A;
    for (int k = sh.k0; k < sh.k1; ++k, at.next(sh.stages)) {
      if (!g_wait_uniform(r.empty + at.s, at.phase ^ 1u, abort_s)) return;
      const uint32_t to = dst + at.s * (a_bytes + b_bytes), bar = at.s * (uint32_t)sizeof(uint64_t);
      if (rank == 0) tc::mbar_expect_tx_w(lead, full + bar, CG * bytes);
      if (CG == 2) tc::tma_load_2d_pair_w(lead, to, map, k * G_KS, row, full_even + bar);
      else tc::tma_load_2d_w(lead, to, map, k * G_KS, row, full + bar);
    }
  }
}

// The MMA issuer: a whole warp (of the even block of a pair).
template <int CG, typename Tiles>
__device__ __forceinline__ void ring_issue(Ring &r, const RingShape &sh, uint8_t *sm, Tiles tiles) {
  volatile int *abort_s = &r.abort_flag;
  const uint32_t tmem = __reduce_max_sync(0xffffffffu, r.tmem);  // one value, in a uniform register
  const uint32_t lead = tc::elect_one(), even = CG == 2 ? tc::cluster_rank() : 0u;
  const uint32_t a_bytes = G_A * G_KS, slot = a_bytes + (uint32_t)(sh.bn / CG) * G_KS, ring = tc::smem_u32(sm);
  const uint32_t idesc = tc::idesc_i8(CG * G_A, sh.bn);
  const int tail = (int)((sh.K - (int64_t)(sh.k1 - 1) * G_KS + 31) / 32);  // MMAs of the last k-step
  Slot at;
  int a_row, b_row;
  for (uint32_t n = 0; tiles.next(a_row, b_row); ++n) {
    const uint32_t a = n & 1u, par = ((n >> 1) & 1u) ^ 1u;
    if (CG == 2) {  // arrivals of both blocks
      bool ok = false;
      for (uint32_t i = 0; i < G_WAIT_LIMIT && !ok && !__any_sync(0xffffffffu, *abort_s); ++i)
        ok = __all_sync(0xffffffffu, tc::mbar_try_wait_cluster(r.acc_empty + a, par));
      if (!ok) {
        *abort_s = 1;
        return;
      }
    } else if (!g_wait_uniform(r.acc_empty + a, par, abort_s)) {
      return;
    }
    tc::tc_fence_after();
    const uint32_t d = tmem + a * 256u;
    for (int k = sh.k0; k < sh.k1; ++k, at.next(sh.stages)) {
      if (!g_wait_uniform(r.full + at.s, at.phase, abort_s)) return;
      tc::tc_fence_after();
      const uint32_t base = ring + at.s * slot;
      const uint64_t ad = tc::desc_sw128(base), bd = tc::desc_sw128(base + a_bytes);
      const int slices = k == sh.k1 - 1 ? min(tail, 4) : 4;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < slices) {
          if (CG == 2) tc::mma_i8_pair_w(lead, d, ad + 2 * j, bd + 2 * j, idesc, k != sh.k0 || j ? 1u : 0u);
          else tc::mma_i8_ss_w(lead, d, ad + 2 * j, bd + 2 * j, idesc, k != sh.k0 || j ? 1u : 0u);
        }
      if (CG == 2) tc::mma_commit_pair_w(lead, r.empty + at.s, even);
      else tc::mma_commit_w(lead, r.empty + at.s);
    }
    if (CG == 2) tc::mma_commit_pair_w(lead, r.acc_full + a, even);
    else tc::mma_commit_w(lead, r.acc_full + a);
  }
}

// An epilogue warp is done reading accumulator a.
template <int CG>
__device__ __forceinline__ void ring_release(Ring &r, uint32_t a, int lane) {
  tc::tc_fence_before();
  __syncwarp();
  if (lane == 0) {
    if (CG == 2) tc::mbar_arrive_cluster(tc::map_rank(tc::smem_u32(r.acc_empty + a), tc::cluster_rank() & ~1u));
    else tc::mbar_arrive(r.acc_empty + a);
  }
}

// Ring slots for tiles of bn columns.
template <int CG>
inline int ring_stages(int bn) {
  const int slot = G_A * G_KS + bn / CG * G_KS, n = G_STAGE_BYTES / slot;
  return n < G_MAX_STAGES ? n : G_MAX_STAGES;
}

// Launch of a kernel whose blocks work in clusters of `cluster`.  `smem` is the
// same for every launch of a kernel: its limit, set here, is the process's, and
// threads with contexts of their own launch at the same time.
template <typename... KArgs, typename... Args>
cudaError_t launch_clusters(void (*kern)(KArgs...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream,
                            unsigned cluster, Args... args) {
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

}  // namespace har
