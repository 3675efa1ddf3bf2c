// k_i8_gemm.cu — y = (q_x q_w^T) * s_x * s_w over 8-bit integers on the tensor
// cores (tcgen05.mma kind::i8, 32-bit sums in tensor memory).
#include <algorithm>

#include "score.cuh"
#include "tc_ptx.cuh"

namespace har {

// The weights are the MMA's 128-row side (a tensor-memory lane is an output
// channel), a tile of up to 256 tokens its columns: a warp of the epilogue
// then writes 32 neighbouring channels of one token with one store, and any
// number of tokens from 1 up is one rule.  Each k-step is 128 bytes of K: one
// swizzled TMA box of weights (16 KB) and one of tokens.
constexpr int G_M = 128, G_KS = 128, G_MAX_BN = 256;
constexpr int G_STAGE_BYTES = 216 * 1024, G_MAX_STAGES = 12;
constexpr int G_WARP_W = 0, G_WARP_MMA = 1, G_WARP_X = 2, G_WARP_EPI = 3, G_EPI_WARPS = 8;
constexpr int G_THREADS = 32 * (G_WARP_EPI + G_EPI_WARPS);
constexpr int G_GROUP = 8;  // weight tiles swept together over all token tiles
constexpr uint32_t G_WAIT_LIMIT = 1u << 22;

struct GemmParams {
  int64_t M, N, K, ldy;
  const float *sx, *sw;
  void *y;
  int bn, stages;     // tokens of a tile; ring slots
  int mt, nt;         // token and weight tiles
  int *status;
};

__device__ __forceinline__ bool g_wait(uint64_t *bar, uint32_t parity, volatile int *abort_s, uint32_t sleep_ns = 0) {
  if (*abort_s) return false;
  if (sleep_ns ? tc::mbar_wait_lazy(bar, parity, G_WAIT_LIMIT, sleep_ns) : tc::mbar_wait(bar, parity, G_WAIT_LIMIT))
    return true;
  *abort_s = 1;
  return false;
}
__device__ __forceinline__ bool g_wait_warp(uint64_t *bar, uint32_t parity, volatile int *abort_s, int lane) {
  if (__all_sync(0xffffffffu, tc::mbar_try_wait(bar, parity))) return true;
  bool ok = true;
  if (lane == 0) ok = g_wait(bar, parity, abort_s);
  return __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
}

// Tile number -> (token tile, weight tile): groups of G_GROUP weight tiles,
// inside a group all token tiles in order, so the tiles in flight at a time
// share their weights and, where there are many tokens, those too.
__device__ __forceinline__ void g_tile(const GemmParams &p, int64_t tile, int &mt, int &nt) {
  const int64_t per = (int64_t)G_GROUP * p.mt;
  const int g = (int)(tile / per);
  const int64_t r = tile - g * per;
  const int n = min(G_GROUP, p.nt - g * G_GROUP);
  mt = (int)(r / n);
  nt = g * G_GROUP + (int)(r - (int64_t)mt * n);
}

template <typename T>
__global__ void __launch_bounds__(G_THREADS, 1)
    i8_gemm_kernel(const __grid_constant__ TmaDesc map_w, const __grid_constant__ TmaDesc map_x, const GemmParams p) {
  extern __shared__ uint8_t g_raw[];
  __shared__ uint64_t full[G_MAX_STAGES], empty[G_MAX_STAGES], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  volatile int *abort_s = &abort_flag;
  uint8_t *sm = g_raw + ((1024u - (tc::smem_u32(g_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int bn = p.bn, stages = p.stages;
  const uint32_t x_bytes = (uint32_t)bn * G_KS, slot_bytes = G_M * G_KS + x_bytes;

  if (warp == 0) {
    tc::tmem_alloc(&tmem_base, 512);
    tc::tmem_relinquish();
  }
  if (tid == 32) {
    for (int s = 0; s < stages; ++s) {
      tc::mbar_init(full + s, 2);
      tc::mbar_init(empty + s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      tc::mbar_init(acc_full + a, 1);
      tc::mbar_init(acc_empty + a, G_EPI_WARPS);
    }
    tc::fence_mbar_init();
    abort_flag = 0;
  }
  if (tid == 0) {
    tc::tma_prefetch_desc(&map_w);
    tc::tma_prefetch_desc(&map_x);
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = tmem_base;
  const int ksteps = (int)((p.K + G_KS - 1) / G_KS);
  const int64_t total = (int64_t)p.mt * p.nt;

  if (warp == G_WARP_W || warp == G_WARP_X) {
    // producers: one thread loads the weight boxes, another the token boxes
    if (lane == 0) {
      const bool is_x = warp == G_WARP_X;
      uint32_t it = 0;
      bool ok = true;
      for (int64_t tile = blockIdx.x; ok && tile < total; tile += gridDim.x) {
        int mt, nt;
        g_tile(p, tile, mt, nt);
        const int row = is_x ? mt * bn : nt * G_M;
        for (int k = 0; k < ksteps; ++k, ++it) {
          const int s = (int)(it % (uint32_t)stages);
          if (!(ok = g_wait(empty + s, ((it / (uint32_t)stages) & 1u) ^ 1u, abort_s, 64))) break;
          uint8_t *dst = sm + (size_t)s * slot_bytes;
          tc::mbar_expect_tx(full + s, is_x ? x_bytes : (uint32_t)(G_M * G_KS));
          tc::tma_load_2d(is_x ? dst + G_M * G_KS : dst, is_x ? &map_x : &map_w, k * G_KS, row, full + s);
        }
      }
    }
  } else if (warp == G_WARP_MMA) {
    const uint32_t lead = tc::elect_one();
    const uint32_t idesc = tc::idesc_i8(G_M, bn);
    const int last = (int)((p.K - (int64_t)(ksteps - 1) * G_KS + 31) / 32);  // MMAs of the last k-step
    uint32_t it = 0, n = 0;
    bool ok = true;
    for (int64_t tile = blockIdx.x; ok && tile < total; tile += gridDim.x, ++n) {
      const uint32_t a = n & 1u;
      if (!(ok = g_wait_warp(acc_empty + a, ((n >> 1) & 1u) ^ 1u, abort_s, lane))) break;
      tc::tc_fence_after();
      const uint32_t d = tmem + a * 256u;
      for (int k = 0; k < ksteps; ++k, ++it) {
        const int s = (int)(it % (uint32_t)stages);
        if (!(ok = g_wait_warp(full + s, (it / (uint32_t)stages) & 1u, abort_s, lane))) break;
        tc::tc_fence_after();
        const uint32_t base = tc::smem_u32(sm + (size_t)s * slot_bytes);
        const uint64_t ad = tc::desc_sw128(base), bd = tc::desc_sw128(base + G_M * G_KS);
        const int slices = k == ksteps - 1 ? last : 4;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < slices) tc::mma_i8_ss_w(lead, d, ad + 2 * j, bd + 2 * j, idesc, (k | j) ? 1u : 0u);
        tc::mma_commit_w(lead, empty + s);
      }
      if (!ok) break;
      tc::mma_commit_w(lead, acc_full + a);
    }
  } else {
    // epilogue: lanes of quadrant warp % 4 are 32 channels; the two warps of a
    // quadrant take the tile's 16-token chunks in turn
    const int g = warp & 3, h = (warp - G_WARP_EPI) >> 2;
    const uint32_t lane_addr = (uint32_t)(32 * g) << 16;
    uint32_t n = 0;
    for (int64_t tile = blockIdx.x; tile < total; tile += gridDim.x, ++n) {
      int mt, nt;
      g_tile(p, tile, mt, nt);
      const uint32_t a = n & 1u;
      const int64_t chan = (int64_t)nt * G_M + 32 * g + lane, m0 = (int64_t)mt * bn;
      const bool live = chan < p.N;
      const float sw = live ? __ldg(p.sw + chan) : 0.0f;
      T *y = (T *)p.y + m0 * p.ldy + chan;
      const int rows = (int)min((int64_t)bn, p.M - m0);
      if (!g_wait_warp(acc_full + a, (n >> 1) & 1u, abort_s, lane)) break;
      tc::tc_fence_after();
      for (int c = 16 * h; c < rows; c += 32) {
        uint32_t v[16];
        tc::tmem_ld16(tmem + lane_addr + a * 256u + (uint32_t)c, v);
        const float sl = c + (lane & 15) < rows ? __ldg(p.sx + m0 + c + (lane & 15)) : 0.0f;
        tc::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float s = __shfl_sync(0xffffffffu, sl, i);
          if (live && c + i < rows)
            y[(int64_t)(c + i) * p.ldy] = from_f32<T>(__fmul_rn(__int2float_rn((int)v[i]), __fmul_rn(s, sw)));
        }
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(acc_empty + a);
    }
  }

  __syncthreads();
  if (*abort_s) {
    if (tid == 0) atomicOr(p.status, DEV_ERR_TIMEOUT);
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);  // let copies and MMAs in flight land
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == 0) tc::tmem_dealloc(tmem, 512);
}

// Tokens of a tile: the split of M into equal tiles of 16 to 256 tokens that
// costs least, a tile's k-step costing its MMAs (2 cycles a token at 8,192
// products a cycle) or its bytes from L2 (about 64 a cycle), whichever is
// more, and a tile about 1,500 cycles to fill and drain.
static int pick_bn(int64_t M, int64_t N, int64_t K, int sms) {
  const int64_t nt = (N + G_M - 1) / G_M, ksteps = (K + G_KS - 1) / G_KS;
  const int64_t first = (M + G_MAX_BN - 1) / G_MAX_BN;
  double best = 0;
  int bn = 0;
  for (int64_t mt = first; mt <= first + 15; ++mt) {
    const int64_t b = ((M + mt - 1) / mt + 15) / 16 * 16;
    const int64_t tiles = nt * ((M + b - 1) / b), waves = (tiles + sms - 1) / sms;
    const double step = std::max(2.0 * b, (G_M * G_KS + b * G_KS) / 64.0);
    const double cost = waves * (ksteps * step + 1500.0);
    if (!bn || cost < best) best = cost, bn = (int)b;
  }
  return bn;
}

int32_t launch_i8_matmul(har_cuda_ctx *ctx, const har_cuda_i8_weights *w, const int8_t *q,
                         int64_t ldq, const float *scale, int64_t M, void *y, int32_t y_dtype,
                         int64_t ldy) {
  GemmParams p = {};
  p.M = M, p.N = w->N, p.K = w->K, p.ldy = ldy;
  p.sx = scale, p.sw = w->scale, p.y = y, p.status = ctx->d_status;
  p.bn = pick_bn(M, w->N, w->K, ctx->num_sms);
  const int slot = G_M * G_KS + p.bn * G_KS;
  p.stages = std::min(G_MAX_STAGES, G_STAGE_BYTES / slot);
  p.mt = (int)((M + p.bn - 1) / p.bn);
  p.nt = (int)((w->N + G_M - 1) / G_M);
  TmaDesc map_x;
  int32_t st = encode_tmap_2d(ctx, &map_x, q, 1, (uint64_t)M, (uint64_t)w->K, (uint64_t)ldq, (uint32_t)p.bn, G_KS, true);
  if (st != HAR_CUDA_OK) return st;
  const size_t smem = (size_t)p.stages * slot + 1024;
  const unsigned grid = (unsigned)std::min<int64_t>(ctx->num_sms, (int64_t)p.mt * p.nt);
  cudaError_t e = cudaSuccess;
  prof_begin(ctx);
  with_dtype(y_dtype, [&](auto t) {
    using T = decltype(t);
    e = cudaFuncSetAttribute(i8_gemm_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, G_STAGE_BYTES + 1024);
    if (e != cudaSuccess) return;
    i8_gemm_kernel<T><<<grid, G_THREADS, smem, ctx->stream>>>(w->map, map_x, p);
  });
  st = check_launch(ctx, "i8_gemm_kernel");
  if (e != cudaSuccess)
    return set_error(ctx, HAR_CUDA_ERR_CUDA, std::string("i8_gemm_kernel: ") + cudaGetErrorString(e));
  return st;
}

}  // namespace har
