// k_i8_gemm.cu — y = (q_x q_w^T) * s_x * s_w over 8-bit integers on the tensor
// cores (tcgen05.mma kind::i8, 32-bit sums in tensor memory).
#include <algorithm>

#include "i8_mma.cuh"

namespace har {

// The weights are the MMA's A side (a tensor-memory lane is an output
// channel), a tile of up to 256 tokens its columns: a warp of the epilogue
// then writes 32 neighbouring channels of one token with one store, and any
// number of tokens from 1 up is one rule.
constexpr int G_GROUP = 1024;  // channels swept together over all token tiles

struct GemmParams {
  RingShape sh;
  int64_t M, N, ldy;
  const float *sx, *sw;
  void *y;
  int mt, nt;         // token and weight tiles
  int *status;
};

// Tiles of one block (or pair): groups of G_GROUP channels, inside a group all
// token tiles in order, so the tiles in flight at a time share their weights
// and, where there are many tokens, those too.
template <int CG>
struct GemmTiles {
  const GemmParams &p;
  int64_t tile;
  int m, n;
  __device__ __forceinline__ explicit GemmTiles(const GemmParams &p_) : p(p_), tile(blockIdx.x / CG) {}
  __device__ __forceinline__ bool next(int &a_row, int &b_row) {
    constexpr int GROUP = G_GROUP / (CG * G_A);
    if (tile >= (int64_t)p.mt * p.nt) return false;
    const int64_t per = (int64_t)GROUP * p.mt;
    const int g = (int)(tile / per);
    const int64_t r = tile - g * per;
    const int width = min(GROUP, p.nt - g * GROUP);
    m = (int)(r / width);
    n = g * GROUP + (int)(r - (int64_t)m * width);
    a_row = n * (CG * G_A);
    b_row = m * p.sh.bn;
    tile += gridDim.x / CG;
    return true;
  }
};

template <typename T, int CG>
__global__ void __launch_bounds__(G_THREADS, 1)
    i8_gemm_kernel(const __grid_constant__ TmaDesc map_w, const __grid_constant__ TmaDesc map_x, const GemmParams p) {
  extern __shared__ uint8_t g_raw[];
  __shared__ Ring ring;
  __shared__ __align__(16) float scales[G_EPI_WARPS][G_MAX_BN / 2];
  uint8_t *sm = g_raw + ((1024u - (tc::smem_u32(g_raw) & 1023u)) & 1023u);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? tc::cluster_rank() : 0u;
  ring_open<CG>(ring, p.sh, &map_w, &map_x);

  if (warp == G_WARP_A) {
    if (lane == 0) ring_produce<CG>(ring, p.sh, sm, false, &map_w, GemmTiles<CG>(p), rank);
  } else if (warp == G_WARP_B) {
    if (lane == 0) ring_produce<CG>(ring, p.sh, sm, true, &map_x, GemmTiles<CG>(p), rank);
  } else if (warp == G_WARP_MMA) {
    if (rank == 0) ring_issue<CG>(ring, p.sh, sm, GemmTiles<CG>(p));
  } else {
    // epilogue: lanes of quadrant warp % 4 are 32 channels; the two warps of a
    // quadrant take the tile's 16-token chunks in turn.  The tokens' scales wait
    // in shared memory (a broadcast read each four), the next chunk's sums are
    // on their way from tensor memory while this one's are written.
    volatile int *abort_s = &ring.abort_flag;
    const int g = warp & 3, h = (warp - G_WARP_EPI) >> 2;
    const uint32_t col0 = ring.tmem + ((uint32_t)(32 * g) << 16);
    float *sx = scales[warp - G_WARP_EPI];
    GemmTiles<CG> tiles(p);
    int a_row, b_row;
    for (uint32_t n = 0; tiles.next(a_row, b_row); ++n) {
      const uint32_t a = n & 1u;
      const int64_t chan = (int64_t)a_row + rank * G_A + 32 * g + lane, m0 = b_row;
      const bool live = chan < p.N;
      const float sw = live ? __ldg(p.sw + chan) : 0.0f;
      T *y = (T *)p.y + m0 * p.ldy + chan;
      const int rows = (int)min((int64_t)p.sh.bn, p.M - m0);
#pragma unroll
      for (int i = 0; i < G_MAX_BN / 64; ++i) {  // slot 32 i + lane: token 16 h + 64 i + (lane, chunks of 16 in turn)
        const int c = 64 * i + 32 * (lane >> 4) + 16 * h + (lane & 15);
        sx[32 * i + lane] = c < rows ? __ldg(p.sx + m0 + c) : 0.0f;
      }
      __syncwarp();
      if (!g_wait_warp(ring.acc_full + a, (n >> 1) & 1u, abort_s, lane)) break;
      tc::tc_fence_after();
      const uint32_t col = col0 + a * 256u;
      uint32_t v[2][16];
      if (16 * h < rows) tc::tmem_ld16(col + (uint32_t)(16 * h), v[0]);
#pragma unroll
      for (int j = 0; j < G_MAX_BN / 32; ++j) {
        const int c = 16 * h + 32 * j;
        if (c >= rows) break;
        tc::tmem_wait_ld16(v[j & 1]);
        if (c + 32 < rows) tc::tmem_ld16(col + (uint32_t)(c + 32), v[(j + 1) & 1]);
        const float4 *s4 = reinterpret_cast<const float4 *>(sx + 16 * j);
        T *yc = y + (int64_t)c * p.ldy;
        const int here = live ? rows - c : 0;
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const float4 s = s4[i >> 2];
          const float f[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (i + u < here)
              yc[(i + u) * p.ldy] = from_f32<T>(__fmul_rn(__int2float_rn((int)v[j & 1][i + u]), __fmul_rn(f[u], sw)));
        }
      }
      ring_release<CG>(ring, a, lane);
    }
  }
  ring_close<CG>(ring, p.status);
}

// Blocks a tile and tokens of a tile: the split of M into equal tiles that
// costs least.  A k-step of a tile costs a lone block its MMAs (2 cycles a
// token at 8,192 products a cycle) or its bytes from L2 (about 64 a cycle) or
// its bytes through shared memory, in and out (128 a cycle), whichever is most;
// a pair moves half the token bytes.  A tile costs about 1,500 cycles to fill
// and drain, a pair 500 more to join.
static int pick_tile(int64_t M, int64_t N, int64_t K, int sms, int &cg) {
  const int64_t ksteps = (K + G_KS - 1) / G_KS;
  double best = 0;
  int bn = 0;
  for (int g = 1; g <= 2; ++g) {
    const int64_t nt = (N + g * G_A - 1) / (g * G_A), first = (M + G_MAX_BN - 1) / G_MAX_BN;
    for (int64_t mt = first; mt <= first + 15; ++mt) {
      const int64_t b = ((M + mt - 1) / mt + 16 * g - 1) / (16 * g) * (16 * g);
      const int64_t tiles = nt * ((M + b - 1) / b), waves = (tiles + sms / g - 1) / (sms / g);
      const double bytes = G_A * G_KS + b / g * G_KS;
      const double step = std::max({2.0 * b, bytes / 64.0});
      const double cost = waves * (ksteps * std::max(step, 2.0 * bytes / 128.0) + 1500.0 + 500.0 * (g - 1));
      if (!bn || cost < best) best = cost, bn = (int)b, cg = g;
    }
  }
  return bn;
}

int32_t launch_i8_matmul(har_cuda_ctx *ctx, const har_cuda_i8_weights *w, const int8_t *q,
                         int64_t ldq, const float *scale, int64_t M, void *y, int32_t y_dtype,
                         int64_t ldy) {
  GemmParams p = {};
  int cg = 1;
  p.M = M, p.N = w->N, p.ldy = ldy;
  p.sx = scale, p.sw = w->scale, p.y = y, p.status = ctx->d_status;
  p.sh.K = w->K;
  p.sh.bn = pick_tile(M, w->N, w->K, ctx->num_sms, cg);
  p.sh.stages = cg == 2 ? ring_stages<2>(p.sh.bn) : ring_stages<1>(p.sh.bn);
  p.mt = (int)((M + p.sh.bn - 1) / p.sh.bn);
  p.nt = (int)((w->N + cg * G_A - 1) / (cg * G_A));
  TmaDesc map_x;
  int32_t st = encode_tmap_2d(ctx, &map_x, q, 1, (uint64_t)M, (uint64_t)w->K, (uint64_t)ldq, (uint32_t)(p.sh.bn / cg), G_KS, true);
  if (st != HAR_CUDA_OK) return st;
  const unsigned grid = (unsigned)std::min<int64_t>(ctx->num_sms / cg, (int64_t)p.mt * p.nt) * cg;
  cudaError_t e = cudaSuccess;
  prof_begin(ctx);
  with_dtype(y_dtype, [&](auto t) {
    using T = decltype(t);
    const size_t smem = G_STAGE_BYTES + 1024;
    e = cg == 2 ? launch_clusters(i8_gemm_kernel<T, 2>, grid, G_THREADS, smem, ctx->stream, 2, w->map, map_x, p)
                : launch_clusters(i8_gemm_kernel<T, 1>, grid, G_THREADS, smem, ctx->stream, 1, w->map, map_x, p);
  });
  st = check_launch(ctx, "i8_gemm_kernel");
  if (e != cudaSuccess)
    return set_error(ctx, HAR_CUDA_ERR_CUDA, std::string("i8_gemm_kernel: ") + cudaGetErrorString(e));
  return st;
}

}  // namespace har
