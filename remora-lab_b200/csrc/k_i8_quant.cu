// k_i8_quant.cu — rows of floats to 8-bit integers with one scale per row:
//   s = max|x| / 127,  q = rint(x / s)   (both quotients rounded to f32).
#include "score.cuh"

namespace har {

// Eight elements of a row: 16-byte loads where the row allows, else one
// element at a time (rows that are slices of wider ones); past `n`, zeros.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T *p, int n, float (&v)[8]) {
  if (VEC && n >= 8) {
    if (sizeof(T) == 4) {
      const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4 *>(p);
      const T *e = reinterpret_cast<const T *>(&a);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32(p[i]) : 0.0f;
  }
}

// TPR threads share a row, each holding eight-element pieces tid, tid + TPR,
// ...: up to four of them stay in registers between the maximum and the
// rounding; longer rows are read again.
template <typename T, int TPR, bool VEC>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR)
    i8_quantize_kernel(const T *__restrict__ x, int64_t M, int K, int64_t ldx, int8_t *__restrict__ q, int64_t ldq,
                       float *__restrict__ scale, int q8) {
  constexpr int THREADS = TPR < 256 ? 256 : TPR;
  constexpr int ROWS = THREADS / TPR, HELD = 4;
  __shared__ uint32_t part[THREADS / 32];
  const int tid = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
  const bool live = row < M;
  const T *xr = x + (live ? row : 0) * ldx;
  float v[HELD][8];
  float most = 0.0f;
#pragma unroll
  for (int c = 0; c < HELD; ++c) {
    const int k0 = (c * TPR + tid) * 8;
    const int n = live ? min(8, K - k0) : 0;
    if (n > 0) {
      load8<T, VEC>(xr + k0, n, v[c]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c][i] = 0.0f;
    }
  }
#pragma unroll
  for (int c = 0; c < HELD; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max_nan(most, fabsf(v[c][i]));
  for (int64_t k0 = (int64_t)(HELD * TPR + tid) * 8; live && k0 < K; k0 += TPR * 8) {
    float u[8];
    load8<T, VEC>(xr + k0, min(8, K - (int)k0), u);
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max_nan(most, fabsf(u[i]));
  }
  uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
  if (TPR > 32) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x / 32] = top;
    __syncthreads();
    constexpr int WARPS = TPR / 32;
    top = part[threadIdx.x / TPR * WARPS];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) top = max(top, part[threadIdx.x / TPR * WARPS + w]);
  }
  if (!live) return;
  const RowScale rs(top);
  if (tid == 0) scale[row] = rs.s;
  int8_t *qr = q + row * ldq;
  auto put = [&](int64_t k0, const float (&u)[8]) {
    const uint2 w = make_uint2(rs.round4(u), rs.round4(u + 4));
    if (q8 && k0 + 8 <= K) {
      *reinterpret_cast<uint2 *>(qr + k0) = w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k0 + i < K) qr[k0 + i] = (int8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
    }
  };
#pragma unroll
  for (int c = 0; c < HELD; ++c) {
    const int k0 = (c * TPR + tid) * 8;
    if (k0 < K) put(k0, v[c]);
  }
  for (int64_t k0 = (int64_t)(HELD * TPR + tid) * 8; k0 < K; k0 += TPR * 8) {
    float u[8];
    load8<T, VEC>(xr + k0, min(8, K - (int)k0), u);
    put(k0, u);
  }
}

template <typename T, int TPR>
static void quantize_rows(har_cuda_ctx *ctx, const void *x, bool vec, int64_t M, int64_t K, int64_t ldx,
                          int8_t *q, int64_t ldq, float *scale, int q8) {
  constexpr int THREADS = TPR < 256 ? 256 : TPR;
  const unsigned grid = (unsigned)((M + THREADS / TPR - 1) / (THREADS / TPR));
  if (vec)
    i8_quantize_kernel<T, TPR, true><<<grid, THREADS, 0, ctx->stream>>>((const T *)x, M, (int)K, ldx, q, ldq, scale, q8);
  else
    i8_quantize_kernel<T, TPR, false><<<grid, THREADS, 0, ctx->stream>>>((const T *)x, M, (int)K, ldx, q, ldq, scale, q8);
}

int32_t launch_i8_quantize(har_cuda_ctx *ctx, const void *x, int32_t dtype, int64_t M, int64_t K,
                           int64_t ldx, int8_t *q, int64_t ldq, float *scale) {
  const size_t eb = dtype_bytes(dtype);
  const bool vec = ((uintptr_t)x & 15u) == 0 && (M == 1 || (ldx * eb & 15u) == 0);
  const int q8 = ((uintptr_t)q & 7u) == 0 && (M == 1 || (ldq & 7) == 0);
  prof_begin(ctx);
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    // as many threads as hold a row in registers at 32 values each
    if (K <= 1024)
      quantize_rows<T, 32>(ctx, x, vec, M, K, ldx, q, ldq, scale, q8);
    else if (K <= 4096)
      quantize_rows<T, 128>(ctx, x, vec, M, K, ldx, q, ldq, scale, q8);
    else
      quantize_rows<T, 512>(ctx, x, vec, M, K, ldx, q, ldq, scale, q8);
  });
  return check_launch(ctx, "i8_quantize_kernel");
}

}  // namespace har
