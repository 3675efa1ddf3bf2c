// k_i8_gemv.cu — y = (q_x q_w^T) * s_x * s_w for a few rows, on the CUDA cores
// (dp4a): one launch that quantises the rows itself, no workspace.
#include <algorithm>

#include "score.cuh"

namespace har {

constexpr int V_T = 512, V_WARPS = V_T / 32, V_R = 2, V_UN = 4;
constexpr int V_MAX_SMEM = 96 * 1024;

struct GemvParams {
  const int8_t *w;
  const float *sw;
  int64_t N, K, ldw;
  const void *x;      // float rows of x_dtype, or 8-bit rows with their scales
  const float *sx;    // null: quantise x
  int64_t ldx;        // elements (bytes of 8-bit rows) between rows
  int x_dtype, M;
  void *y;
  int64_t ldy;
};

__device__ __forceinline__ float load_float(const void *x, int dtype, int64_t i) {
  if (dtype == HAR_CUDA_DTYPE_F32) return ((const float *)x)[i];
  if (dtype == HAR_CUDA_DTYPE_F16) return __half2float(((const __half *)x)[i]);
  return __bfloat162float(((const __nv_bfloat16 *)x)[i]);
}

// MT rows (the last ones repeated as zeros) share every weight read.  A warp
// takes V_R neighbouring channels at a time, lanes over 16-byte pieces of K,
// and adds its lanes' integer sums with one reduction instruction each.  The
// first pieces are asked for before the rows are quantised: at the smallest
// sizes the two latencies are all there is.
template <typename T, int MT>
__global__ void __launch_bounds__(V_T, 2) i8_gemv_kernel(const GemvParams p) {
  extern __shared__ __align__(16) uint8_t v_raw[];  // q [MT][pieces][16]
  __shared__ float scale[MT];
  __shared__ uint32_t part[V_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int pieces = (int)((p.K + 15) / 16);
  const int64_t step = (int64_t)gridDim.x * V_WARPS * V_R;
  int64_t n0 = ((int64_t)blockIdx.x * V_WARPS + warp) * V_R;

  uint4 ahead[V_UN][V_R];
  auto load = [&](uint4(&w)[V_UN][V_R], int64_t n, int i0) {
#pragma unroll
    for (int u = 0; u < V_UN; ++u) {
      const int c = i0 + u * 32 + lane;
#pragma unroll
      for (int r = 0; r < V_R; ++r)
        w[u][r] = c < pieces && n + r < p.N ? ldg_nc_v4(p.w + (n + r) * p.ldw + 16 * (int64_t)c) : make_uint4(0, 0, 0, 0);
    }
  };
  load(ahead, n0, 0);

  // the rows, quantised, zeros behind K: the bytes there in the weights count nothing
  if (p.sx) {
    for (int m = 0; m < MT; ++m)
      for (int c = tid; c < pieces; c += V_T) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (m < p.M) {
          const int8_t *at = (const int8_t *)p.x + m * p.ldx + 16 * (int64_t)c;
          if (16 * (int64_t)c + 16 <= p.K) {
            v = *reinterpret_cast<const uint4 *>(at);
          } else {
            uint32_t b[4] = {0, 0, 0, 0};
            for (int i = 0; 16 * (int64_t)c + i < p.K; ++i) b[i >> 2] |= (uint32_t)(uint8_t)at[i] << (8 * (i & 3));
            v = make_uint4(b[0], b[1], b[2], b[3]);
          }
        }
        reinterpret_cast<uint4 *>(v_raw)[(int64_t)m * pieces + c] = v;
      }
    if (tid < MT) scale[tid] = tid < p.M ? p.sx[tid] : 0.0f;
  } else {
    constexpr int WPR = V_WARPS / MT;  // warps a row
    const int m = warp / WPR, t = (warp % WPR) * 32 + lane;
    const bool live = m < p.M;
    uint32_t top = 0;
    for (int64_t k = t; live && k < p.K; k += WPR * 32)
      top = max(top, __float_as_uint(load_float(p.x, p.x_dtype, m * p.ldx + k)) & 0x7fffffffu);
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) part[warp] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WPR; ++i) top = max(top, part[m * WPR + i]);
    const RowScale rs(top);
    if (t == 0) scale[m] = rs.s;
    int8_t *q = (int8_t *)v_raw + (int64_t)m * pieces * 16;
    for (int64_t k = t; k < (int64_t)pieces * 16; k += WPR * 32)
      q[k] = live && k < p.K ? (int8_t)rs.round(load_float(p.x, p.x_dtype, m * p.ldx + k)) : (int8_t)0;
  }
  __syncthreads();

  const uint4 *xq = reinterpret_cast<const uint4 *>(v_raw);
  for (bool first = true; n0 < p.N; n0 += step, first = false) {
    int acc[V_R][MT] = {};
    for (int i0 = 0; i0 < pieces; i0 += 32 * V_UN) {
      uint4 w[V_UN][V_R];
      if (first && i0 == 0) {
#pragma unroll
        for (int u = 0; u < V_UN; ++u)
#pragma unroll
          for (int r = 0; r < V_R; ++r) w[u][r] = ahead[u][r];
      } else {
        load(w, n0, i0);
      }
#pragma unroll
      for (int u = 0; u < V_UN; ++u) {
        const int c = i0 + u * 32 + lane;
        if (c < pieces) {
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const uint4 x = xq[m * pieces + c];
#pragma unroll
            for (int r = 0; r < V_R; ++r) {
              acc[r][m] = __dp4a((int)w[u][r].x, (int)x.x, acc[r][m]);
              acc[r][m] = __dp4a((int)w[u][r].y, (int)x.y, acc[r][m]);
              acc[r][m] = __dp4a((int)w[u][r].z, (int)x.z, acc[r][m]);
              acc[r][m] = __dp4a((int)w[u][r].w, (int)x.w, acc[r][m]);
            }
          }
        }
      }
    }
    int mine = 0;  // lane r * MT + m keeps the sum of (channel r, row m)
#pragma unroll
    for (int r = 0; r < V_R; ++r)
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int s = __reduce_add_sync(0xffffffffu, acc[r][m]);
        if (lane == r * MT + m) mine = s;
      }
    const int r = lane / MT, m = lane % MT;
    if (lane < V_R * MT && m < p.M && n0 + r < p.N)
      ((T *)p.y)[m * p.ldy + n0 + r] =
          from_f32<T>(__fmul_rn(__int2float_rn(mine), __fmul_rn(scale[m], __ldg(p.sw + n0 + r))));
  }
}

bool i8_gemv_takes(int64_t M, int64_t N, int64_t K) {
  (void)N;
  const int64_t mt = M <= 1 ? 1 : M <= 2 ? 2 : M <= 4 ? 4 : 8;
  return M <= 8 && mt * ((K + 15) / 16 * 16) <= V_MAX_SMEM;
}

int32_t launch_i8_gemv(har_cuda_ctx *ctx, const har_cuda_i8_weights *w, const void *x, int32_t x_dtype,
                       int64_t ldx, const float *sx, int64_t M, void *y, int32_t y_dtype, int64_t ldy) {
  GemvParams p = {};
  p.w = w->q, p.sw = w->scale, p.N = w->N, p.K = w->K, p.ldw = w->ldq;
  p.x = x, p.sx = sx, p.ldx = ldx, p.x_dtype = x_dtype, p.M = (int)M, p.y = y, p.ldy = ldy;
  const int mt = M <= 1 ? 1 : M <= 2 ? 2 : M <= 4 ? 4 : 8;
  const size_t smem = (size_t)mt * (size_t)((w->K + 15) / 16 * 16);
  const int64_t blocks = (w->N + V_WARPS * V_R - 1) / (V_WARPS * V_R);
  const unsigned grid = (unsigned)std::min<int64_t>(blocks, 2 * ctx->num_sms);
  cudaError_t e = cudaSuccess;
  auto go = [&](auto kernel) {
    if (smem > 48 * 1024) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, V_MAX_SMEM);
    if (e == cudaSuccess) kernel<<<grid, V_T, smem, ctx->stream>>>(p);
  };
  prof_begin(ctx);
  with_dtype(y_dtype, [&](auto t) {
    using T = decltype(t);
    if (mt == 1) go(i8_gemv_kernel<T, 1>);
    else if (mt == 2) go(i8_gemv_kernel<T, 2>);
    else if (mt == 4) go(i8_gemv_kernel<T, 4>);
    else go(i8_gemv_kernel<T, 8>);
  });
  const int32_t st = check_launch(ctx, "i8_gemv_kernel");
  if (e != cudaSuccess)
    return set_error(ctx, HAR_CUDA_ERR_CUDA, std::string("i8_gemv_kernel: ") + cudaGetErrorString(e));
  return st;
}

}  // namespace har
