// k_i8_gemm.cu — y = (q_x q_w^T) * s_x * s_w over 8-bit integers.
#include "score.cuh"

namespace har {

// Four bytes at column k of a row of K bytes; past the end, zeros (the bytes
// behind a row's K are not read: the last row may end the allocation).
__device__ __forceinline__ uint32_t i8_word(const int8_t *row, int64_t k, int64_t K) {
  if (k + 4 <= K) return *reinterpret_cast<const uint32_t *>(row + k);
  uint32_t w = 0;
  for (int i = 0; i < 4; ++i)
    if (k + i < K) w |= (uint32_t)(uint8_t)row[k + i] << (8 * i);
  return w;
}

template <typename T>
__global__ void __launch_bounds__(256)
    i8_matmul_kernel(const int8_t *__restrict__ x, int64_t ldx, const float *__restrict__ sx, int64_t M,
                     const int8_t *__restrict__ w, int64_t ldw, const float *__restrict__ sw, int64_t N,
                     int64_t K, T *__restrict__ y, int64_t ldy) {
  __shared__ uint32_t a[64][17], b[64][17];
  const int64_t n0 = (int64_t)blockIdx.x * 64, m0 = (int64_t)blockIdx.y * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int acc[4][4] = {};
  for (int64_t k0 = 0; k0 < K; k0 += 64) {
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
      const int r = i >> 4, c = i & 15;
      a[r][c] = m0 + r < M ? i8_word(x + (m0 + r) * ldx, k0 + 4 * c, K) : 0u;
      b[r][c] = n0 + r < N ? i8_word(w + (n0 + r) * ldw, k0 + 4 * c, K) : 0u;
    }
    __syncthreads();
    for (int c = 0; c < 16; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a((int)a[ty + 16 * i][c], (int)b[tx + 16 * j][c], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m < M && n < N)
        y[m * ldy + n] = from_f32<T>(__fmul_rn(__int2float_rn(acc[i][j]), __fmul_rn(sx[m], sw[n])));
    }
}

int32_t launch_i8_matmul(har_cuda_ctx *ctx, const har_cuda_i8_weights *w, const int8_t *q,
                         int64_t ldq, const float *scale, int64_t M, void *y, int32_t y_dtype,
                         int64_t ldy) {
  // the token axis of a grid holds 65,535 tiles
  constexpr int64_t ROWS = (int64_t)64 * 65535;
  for (int64_t m0 = 0; m0 < M; m0 += ROWS) {
    const int64_t m = M - m0 < ROWS ? M - m0 : ROWS;
    const dim3 grid((unsigned)((w->N + 63) / 64), (unsigned)((m + 63) / 64));
    prof_begin(ctx);
    with_dtype(y_dtype, [&](auto t) {
      using T = decltype(t);
      i8_matmul_kernel<T><<<grid, 256, 0, ctx->stream>>>(q + m0 * ldq, ldq, scale + m0, m, w->q, w->ldq, w->scale,
                                                         w->N, w->K, (T *)y + m0 * ldy, ldy);
    });
    const int32_t st = check_launch(ctx, "i8_matmul_kernel");
    if (st != HAR_CUDA_OK) return st;
  }
  return HAR_CUDA_OK;
}

}  // namespace har
