// k_i8_gemm.cu — y = (q_x q_w^T) * s_x * s_w over 8-bit integers on the tensor
// cores (tcgen05.mma kind::i8, 32-bit sums in tensor memory).
// 8,192 x 8,192 x 4,096 in bf16: 172 us, 3.2 POP/s, the tensor pipe active for 92% of
// the cycles; 48 x 65,536 x 2,048 in f32: 29 us, 5.1 TB/s of weights and output.
#include <algorithm>

#include "i8_mma.cuh"

namespace har {

// The weights are the MMA's A side (a tensor-memory lane is an output
// channel), a tile of up to 256 tokens its columns: a warp of the epilogue
// then writes 32 neighbouring channels of one token with one store, and any
// number of tokens from 1 up is one rule.
constexpr int G_GROUP = 1024;  // channels swept together over all token tiles
constexpr int G_SLAB = 8192;   // bytes of finished output on their way to memory
constexpr int G_SLABS = 4;     // two for each half of the epilogue

struct GemmParams {
  RingShape sh;
  int64_t M, N, ldy;
  const float *sx, *sw;
  void *y;
  int store;          // y's rows take TMA stores
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

// Tokens quad, quad + 4, ... of a slab, from shared memory to rows of any
// alignment, by one warp: whole 4-byte words, a 2-byte type's odd first and
// last element apart; four rows on their way at a time.
template <typename T>
__device__ __forceinline__ void put_rows(T *y, int64_t ldy, const T *slab, int tokens, int chans, int quad, int lane) {
  if (chans <= 0) return;
#pragma unroll 4
  for (int t = quad; t < tokens; t += 4) {
    T *to = y + t * ldy;
    const T *row = slab + t * G_A;
    if (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < G_A; i += 32)
        if (i + lane < chans) to[i + lane] = row[i + lane];
    } else {
      const int odd = (int)((uintptr_t)to >> 1) & 1;
      if (odd && lane == 0) to[0] = row[0];
#pragma unroll
      for (int i = 0; i < G_A; i += 64) {
        const int e = odd + i + 2 * lane;
        if (e + 1 < chans) {
          const T two[2] = {row[e], row[e + 1]};
          *reinterpret_cast<uint32_t *>(to + e) = *reinterpret_cast<const uint32_t *>(two);
        } else if (e < chans) {
          to[e] = row[e];
        }
      }
    }
  }
}

// Output of `n` tokens (at most 128, from token m) of 128 channels, by the
// four warps of one half; v holds this thread's channel.  Finished values are
// laid out in shared memory, [token][128 channels], and written by TMA, or row
// by row where y's rows do not start at multiples of 16 bytes (777 x 5,003 x 1,999
// in f16: 24.5 us, with rows 5,008 apart and whole 20.3).  A 2-byte value a lane
// straight to memory took 12,600 cycles a tile of 256 tokens, more than its
// MMAs at K = 2048 (8,200); a bulk copy a row held up the loads more than the
// warps' own stores do (28 us for the 777 rows).
template <typename T>
__device__ __forceinline__ void put_slabs(const GemmParams &p, const void *map_y, uint8_t *slabs, const float *sx, float sw,
                                          uint32_t (&v)[4][32], int n, int64_t m, int chan0, int h, int quad, int lane,
                                          uint32_t &used) {
  constexpr int TOK = G_SLAB / (G_A * (int)sizeof(T));  // tokens of a slab: 32, or 16 of f32
  const int id = 1 + h;
#pragma unroll
  for (int i = 0; i < 128 / TOK; ++i, ++used) {
    if (i * TOK >= n) break;
    T *slab = reinterpret_cast<T *>(slabs + (2 * h + (used & 1u)) * G_SLAB);
    if (p.store && quad == 0 && lane == 0) tc::bulk_wait_read<1>();  // the slab two before has been read
    tc::bar_sync(id, 128);
#pragma unroll
    for (int t = 0; t < TOK; t += 4) {
      const int c = i * TOK + t;
      const float4 s = *reinterpret_cast<const float4 *>(sx + c);
      const float f[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int u = 0; u < 4; ++u)
        slab[(t + u) * G_A + 32 * quad + lane] =
            from_f32<T>(__fmul_rn(__int2float_rn((int)v[(c + u) >> 5][(c + u) & 31]), __fmul_rn(f[u], sw)));
    }
    if (p.store) tc::fence_proxy_async_smem();
    tc::bar_sync(id, 128);
    if (p.store) {
      if (quad == 0 && lane == 0) {
#pragma unroll
        for (int t = 0; t < TOK; t += 16)
          if (i * TOK + t < n && chan0 < p.N) tc::tma_store_2d(map_y, chan0, (int)m + i * TOK + t, slab + t * G_A);
        tc::bulk_commit();
      }
    } else {
      T *y = (T *)p.y + (m + i * TOK) * p.ldy + chan0;
      const int chans = (int)min((int64_t)G_A, p.N - chan0);
      put_rows(y, p.ldy, slab, min(TOK, n - i * TOK), chans, quad, lane);
    }
  }
}

template <typename T, int CG>
__global__ void __launch_bounds__(G_THREADS, 1)
    i8_gemm_kernel(const __grid_constant__ TmaDesc map_w, const __grid_constant__ TmaDesc map_x,
                   const __grid_constant__ TmaDesc map_y, const GemmParams p) {
  extern __shared__ uint8_t g_raw[];
  __shared__ Ring ring;
  __shared__ int go[2][2];
  __shared__ __align__(16) float scales[G_EPI_WARPS][G_MAX_BN / 2];
  uint8_t *sm = g_raw + ((1024u - (tc::smem_u32(g_raw) & 1023u)) & 1023u);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? tc::cluster_rank() : 0u;
  ring_open<CG>(ring, p.sh, &map_w, &map_x);

  if (warp == G_WARP_A) {
    ring_produce<CG>(ring, p.sh, sm, false, &map_w, GemmTiles<CG>(p), rank);
  } else if (warp == G_WARP_B) {
    ring_produce<CG>(ring, p.sh, sm, true, &map_x, GemmTiles<CG>(p), rank);
  } else if (warp == G_WARP_MMA) {
    if (rank == 0) ring_issue<CG>(ring, p.sh, sm, GemmTiles<CG>(p));
  } else {
    // epilogue: lanes of quadrant warp % 4 are 32 channels, half h of the warps
    // takes half of the tile's tokens: it reads its sums into registers in one
    // go, gives the accumulator back and only then converts and writes
    volatile int *abort_s = &ring.abort_flag;
    const int quad = warp & 3, h = (warp - G_WARP_EPI) >> 2;
    const uint32_t col0 = ring.tmem + ((uint32_t)(32 * quad) << 16);
    const int half = (p.sh.bn / 16 + 1) / 2 * 16;
    float *sx = scales[warp - G_WARP_EPI];
    uint8_t *slabs = sm + G_STAGE_BYTES;
    uint32_t used = 0;  // slabs written so far
    GemmTiles<CG> tiles(p);
    int a_row, b_row;
    for (uint32_t n = 0; tiles.next(a_row, b_row); ++n) {
      const uint32_t a = n & 1u;
      const int chan0 = a_row + (int)rank * G_A;
      const int64_t chan = (int64_t)chan0 + 32 * quad + lane, m = (int64_t)b_row + h * half;
      const bool live = chan < p.N;
      const float sw = live ? __ldg(p.sw + chan) : 0.0f;
      // this half's tokens: within the tile, and within M
      const int mine = (int)max((int64_t)0, min((int64_t)(h == 0 ? half : p.sh.bn - half), p.M - m));
#pragma unroll
      for (int i = 0; i < G_MAX_BN / 64; ++i) {
        const int c = 32 * i + lane;
        sx[c] = c < mine ? __ldg(p.sx + m + c) : 0.0f;
      }
      __syncwarp();
      // one warp waits for the half and says whether to go on, so that all four
      // leave together when a wait gave up
      if (quad == 0) {
        const bool ok = g_wait_warp(ring.acc_full + a, (n >> 1) & 1u, abort_s, lane, 256);
        if (lane == 0) go[h][a] = ok;
      }
      tc::bar_sync(1 + h, 128);
      if (!go[h][a]) break;
      tc::tc_fence_after();
      const uint32_t col = col0 + a * 256u + (uint32_t)(h * half);
      uint32_t v[4][32];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (32 * j < mine) tc::tmem_ld32(col + (uint32_t)(32 * j), v[j]);
#pragma unroll
      for (int j = 0; j < 4; ++j) tc::tmem_wait_ld32(v[j]);
      ring_release<CG>(ring, a, lane);
      put_slabs<T>(p, &map_y, slabs, sx, sw, v, mine, m, chan0, h, quad, lane, used);
    }
    if (p.store && quad == 0 && lane == 0) tc::bulk_wait<0>();
  }
  ring_close<CG>(ring, p.status);
}

// The same product where there are fewer tiles than pairs: a cluster of S pairs
// shares one tile, each pair a part of K, because a k-step takes its 315 cycles
// however narrow the tile (8 x 512 x 16,384: 24.6 us whole, 15.4 in four parts;
// 8 x 2,048 x 8,192: 16.2 and 10.8).  The pairs leave their 32-bit sums in their
// shared memory; pair s reads every pair's sums of token slice s, adds them up
// (whole numbers: any order) and writes its slice.  (Sent instead of fetched
// they took two barriers and 3.3 us for the smallest tile.)
template <typename T, int S>
__global__ void __launch_bounds__(G_THREADS, 1)
    i8_split_kernel(const __grid_constant__ TmaDesc map_w, const __grid_constant__ TmaDesc map_x, GemmParams p) {
  extern __shared__ uint8_t g_raw[];
  __shared__ Ring ring;
  uint8_t *sm = g_raw + ((1024u - (tc::smem_u32(g_raw) & 1023u)) & 1023u);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = tc::cluster_rank(), rank = crank & 1u, part = crank >> 1;
  const int all = p.sh.k1;  // at least 2 S, so no part is empty
  p.sh.k0 = all * (int)part / S;
  p.sh.k1 = all * ((int)part + 1) / S;
  // this cluster's tile, once
  struct One {
    int a_row, b_row;
    bool left;
    __device__ __forceinline__ bool next(int &a, int &b) {
      a = a_row, b = b_row;
      const bool was = left;
      left = false;
      return was;
    }
  };
  const int tile = (int)(blockIdx.x / (2 * S));
  const One one = {tile / p.mt * (2 * G_A), tile % p.mt * p.sh.bn, true};
  ring_open<2>(ring, p.sh, &map_w, &map_x);

  const int quad = warp & 3, h = (warp - G_WARP_EPI) >> 2;
  const int half = (p.sh.bn / 16 + 1) / 2 * 16, slice = p.sh.bn / S;
  const int cols = h == 0 ? half : p.sh.bn - half;  // this half's tokens
  uint32_t v[4][32];
  bool ok = false;
  if (warp == G_WARP_A) {
    ring_produce<2>(ring, p.sh, sm, false, &map_w, one, rank);
  } else if (warp == G_WARP_B) {
    ring_produce<2>(ring, p.sh, sm, true, &map_x, one, rank);
  } else if (warp == G_WARP_MMA) {
    if (rank == 0) ring_issue<2>(ring, p.sh, sm, one);
  } else {
    ok = g_wait_warp(ring.acc_full, 0, &ring.abort_flag, lane, 64);
    tc::tc_fence_after();
    const uint32_t col = ring.tmem + ((uint32_t)(32 * quad) << 16) + (uint32_t)(h * half);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (ok && 32 * j < cols) tc::tmem_ld32(col + (uint32_t)(32 * j), v[j]);
#pragma unroll
    for (int j = 0; j < 4; ++j) tc::tmem_wait_ld32(v[j]);
  }
  if (warp >= G_WARP_EPI && ok) {
    // the pair's MMAs are done with the ring: it takes the sums, [token][128 channels]
    uint32_t *mine = reinterpret_cast<uint32_t *>(sm) + (h * half) * G_A + 32 * quad + lane;
#pragma unroll
    for (int c = 0; c < 128; ++c)
      if (c < cols) mine[c * G_A] = v[c >> 5][c & 31];
  }
  __syncwarp();
  tc::cluster_arrive();
  tc::cluster_wait();
  if (warp >= G_WARP_EPI) {
    const int tid = (int)threadIdx.x - 32 * G_WARP_EPI, c = 4 * (tid & 31);
    const int64_t chan = (int64_t)one.a_row + rank * G_A + c, m0 = (int64_t)one.b_row + part * slice;
    const int tokens = (int)max((int64_t)0, min((int64_t)slice, p.M - m0));
    const int chans = (int)max((int64_t)0, min((int64_t)4, p.N - chan));
    float sw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) sw[i] = i < chans ? __ldg(p.sw + chan + i) : 0.0f;
    uint32_t from[S];
#pragma unroll
    for (int s = 0; s < S; ++s)
      from[s] = tc::map_rank(tc::smem_u32(sm) + ((uint32_t)(part * slice) * G_A + (uint32_t)c) * 4u, (uint32_t)(2 * s) + rank);
#pragma unroll 2
    for (int t = tid >> 5; t < tokens; t += G_EPI_WARPS) {
      int4 a[S];
#pragma unroll
      for (int s = 0; s < S; ++s) a[s] = tc::ld_cluster_v4(from[s] + (uint32_t)t * (G_A * 4u));
#pragma unroll
      for (int s = 1; s < S; ++s) a[0].x += a[s].x, a[0].y += a[s].y, a[0].z += a[s].z, a[0].w += a[s].w;
      const float sx = __ldg(p.sx + m0 + t);
      const int sum[4] = {a[0].x, a[0].y, a[0].z, a[0].w};
      T *y = (T *)p.y + (m0 + t) * p.ldy + chan;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < chans) y[i] = from_f32<T>(__fmul_rn(__int2float_rn(sum[i]), __fmul_rn(sx, sw[i])));
    }
  }
  ring_close<2>(ring, p.status);
}

// How a product is cut up.  Blocks a tile (cg), tokens of a tile (bn), pairs
// that share a tile (split): the first by this order of merit.  It ranks cuts of
// one product and does not predict times, which are more than twice its cycles
// (512 x 2,048 x 2,048 takes 8.2 us for 3.4 by it, 777 x 5,003 x 1,999 19.6 when
// aligned for 8.2, 48 x 65,536 x 2,048 29 for 12.7): it leaves out the launch, the
// memory's bytes and the waits for L2.
// A k-step counts for its MMAs, 2 cycles a token at 8,192 products a cycle, and 315
// at the least, which issuing them takes; or for its bytes, 72 a cycle, of which a
// pair's blocks share the tokens'.  A tile counts 1,000 cycles to fill and drain, a
// pair 2,000 more to join, and 4,000 if its sums have to meet.  Of 220 cuts of
// 31 products from 64 x 64 x 64 to 4096^3 the cut that it names is 1.5% slower
// than the best on average: 777 x 5,008 x 1,999 takes 19.6 us as 280 lone tiles of
// 112 tokens and 19.9 as 140 pairs' of 128, 203 x 50,024 x 1,999 44 us alone and 38
// in pairs, 4096^3 54 and 51.  Clusters of 4 and 8 blocks do not fill every
// group of SMs: 35 and 15 of them ran at a time.
struct GemmPlan {
  int cg, bn, split;
};
static GemmPlan pick_plan(int64_t M, int64_t N, int64_t K, int sms) {
  const int64_t ksteps = ksteps_of(K), first = (M + G_MAX_BN - 1) / G_MAX_BN;
  double best = 0;
  GemmPlan plan = {};
  for (int g = 1; g <= 2; ++g) {
    const int64_t nt = (N + g * G_A - 1) / (g * G_A);
    for (int64_t mt = first; mt <= first + 15; ++mt) {
      const int64_t b = ((M + mt - 1) / mt + 16 * g - 1) / (16 * g) * (16 * g);
      const int64_t tiles = nt * ((M + b - 1) / b);
      const double step = std::max({2.0 * b, (G_A + b / g) * (G_KS / 72.0), 315.0});
      for (int s = 1; s <= (g == 2 ? 4 : 1); s *= 2) {
        if (s > 1 && (tiles > (s == 2 ? 35 : 15) * sms / 148 || ksteps < 2 * s)) continue;
        const int64_t waves = (tiles * s + sms / g - 1) / (sms / g);
        const double cost = waves * ((ksteps + s - 1) / s * step + 1000.0 + 2000.0 * (g - 1)) + (s > 1 ? 4000.0 : 0.0);
        if (!plan.bn || cost < best) best = cost, plan = {g, (int)b, s};
      }
    }
  }
  return plan;
}

int32_t launch_i8_matmul(har_cuda_ctx *ctx, const har_cuda_i8_weights *w, const int8_t *q,
                         int64_t ldq, const float *scale, int64_t M, void *y, int32_t y_dtype,
                         int64_t ldy, bool padded) {
  const GemmPlan plan = pick_plan(M, w->N, w->K, ctx->num_sms);
  const int cg = plan.cg;
  GemmParams p = {};
  p.M = M, p.N = w->N, p.ldy = ldy;
  p.sx = scale, p.sw = w->scale, p.y = y, p.status = ctx->d_status;
  p.sh.K = w->K, p.sh.k0 = 0, p.sh.k1 = ksteps_of(w->K);
  p.sh.bn = plan.bn;
  p.sh.stages = cg == 2 ? ring_stages<2>(p.sh.bn) : ring_stages<1>(p.sh.bn);
  p.mt = (int)((M + p.sh.bn - 1) / p.sh.bn);
  p.nt = (int)((w->N + cg * G_A - 1) / (cg * G_A));
  TmaDesc map_x;
  int32_t st = encode_tmap_2d(ctx, &map_x, q, 1, (uint64_t)M, (uint64_t)w->K, (uint64_t)ldq, (uint32_t)(p.sh.bn / cg), G_KS, true);
  if (st != HAR_CUDA_OK) return st;
  // y by TMA where its rows start and end at multiples of 16 bytes (a TMA
  // store fills the last 16 bytes of a row with zeros)
  TmaDesc map_y = map_x;
  const size_t eb = dtype_bytes(y_dtype);
  p.store = plan.split == 1 && ((uintptr_t)y & 15u) == 0 && (padded || (w->N * (int64_t)eb) % 16 == 0) &&
            (M == 1 || (ldy * (int64_t)eb) % 16 == 0);
  if (p.store) {
    const uint64_t pitch = ((uint64_t)(M == 1 ? w->N : ldy) * eb + 15) / 16 * 16;
    st = encode_tmap_2d(ctx, &map_y, y, (int)eb, (uint64_t)M, (uint64_t)w->N, pitch, 16, G_A, false);
    if (st != HAR_CUDA_OK) return st;
  }
  const unsigned grid = (unsigned)std::min<int64_t>(ctx->num_sms / cg, (int64_t)p.mt * p.nt) * cg;
  const unsigned split_grid = (unsigned)(p.mt * p.nt * 2 * plan.split);
  cudaError_t e = cudaSuccess;
  const char *name = plan.split > 1 ? "i8_split_kernel" : "i8_gemm_kernel";
  prof_begin(ctx);
  with_dtype(y_dtype, [&](auto t) {
    using T = decltype(t);
    const size_t smem = G_STAGE_BYTES + G_SLABS * G_SLAB + 1024, split_smem = G_STAGE_BYTES + 1024;
    e = plan.split == 4 ? launch_clusters(i8_split_kernel<T, 4>, split_grid, G_THREADS, split_smem, ctx->stream, 8, w->map, map_x, p)
        : plan.split == 2 ? launch_clusters(i8_split_kernel<T, 2>, split_grid, G_THREADS, split_smem, ctx->stream, 4, w->map, map_x, p)
        : cg == 2 ? launch_clusters(i8_gemm_kernel<T, 2>, grid, G_THREADS, smem, ctx->stream, 2, w->map, map_x, map_y, p)
                  : launch_clusters(i8_gemm_kernel<T, 1>, grid, G_THREADS, smem, ctx->stream, 1, w->map, map_x, map_y, p);
  });
  st = check_launch(ctx, name);
  if (e != cudaSuccess)
    return set_error(ctx, HAR_CUDA_ERR_CUDA, std::string(name) + ": " + cudaGetErrorString(e));
  return st;
}

}  // namespace har
