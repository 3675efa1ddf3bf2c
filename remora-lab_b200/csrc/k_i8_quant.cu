// k_i8_quant.cu — rows of floats to 8-bit integers with one scale per row:
//   s = max|x| / 127,  q = rint(x / s)   (both quotients rounded to f32).
#include "score.cuh"

namespace har {

// How a row's elements are read: one at a time (rows that are slices of wider
// ones), or 16 bytes at a time with or without a shorter piece at the end.
enum { SINGLY, WIDE, WHOLE };

// Eight elements of a row, kept as they are stored; past `n`, zeros.
template <typename T>
struct Eight {
  static constexpr int W = sizeof(T) / 2;
  uint4 raw[W];
  template <int HOW>
  __device__ __forceinline__ void load(const T *p, int n) {
    if (HOW == WHOLE) {
#pragma unroll
      for (int i = 0; i < W; ++i)
        raw[i] = n > 0 ? ldg_nc_v4(reinterpret_cast<const uint4 *>(p) + i) : make_uint4(0u, 0u, 0u, 0u);
    } else if (HOW == WIDE && n >= 8) {
#pragma unroll
      for (int i = 0; i < W; ++i) raw[i] = ldg_nc_v4(reinterpret_cast<const uint4 *>(p) + i);
    } else {
      T e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = i < n ? p[i] : from_f32<T>(0.0f);
#pragma unroll
      for (int i = 0; i < W; ++i) raw[i] = reinterpret_cast<const uint4 *>(e)[i];
    }
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(reinterpret_cast<const T *>(raw)[i]);
  }
  // largest |x|, NaN kept
  __device__ __forceinline__ float most(float m) const {
    float v[8];
    get(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max_nan(m, fabsf(v[i]));
    return m;
  }
};

// TPR threads share a row, each holding eight-element pieces tid, tid + TPR,
// ...: up to four of them stay in registers, as loaded, between the maximum
// and the rounding; longer rows are read again.  What bounds it is the bytes
// on their way: 16-bit rows kept as f32 took 57 registers, half the loads in
// flight and 36 us for 8,192 x 4,096; as loaded it takes 21 us, 4.8 TB/s, two thirds
// of the issue slots in use.
template <typename T, int TPR, int HOW>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR, (sizeof(T) == 2 ? 5 : 4) * 256 / (TPR < 256 ? 256 : TPR))
    i8_quantize_kernel(const T *__restrict__ x, int64_t M, int K, int64_t ldx, int8_t *__restrict__ q, int64_t ldq,
                       float *__restrict__ scale, int q8) {
  constexpr int THREADS = TPR < 256 ? 256 : TPR;
  constexpr int ROWS = THREADS / TPR, HELD = 4;
  __shared__ uint32_t part[THREADS / 32];
  const int tid = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
  const bool live = row < M;
  const T *xr = x + (live ? row : 0) * ldx;
  Eight<T> held[HELD];
#pragma unroll
  for (int c = 0; c < HELD; ++c) {
    const int k0 = (c * TPR + tid) * 8;
    held[c].template load<HOW>(xr + k0, live ? min(8, K - k0) : 0);
  }
  float most = 0.0f;
#pragma unroll
  for (int c = 0; c < HELD; ++c) most = held[c].most(most);
  for (int64_t k0 = (int64_t)(HELD * TPR + tid) * 8; live && k0 < K; k0 += TPR * 8) {
    Eight<T> u;
    u.template load<HOW>(xr + k0, min(8, K - (int)k0));
    most = u.most(most);
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
  if (rs.odd()) {
    for (int k = tid; k < K; k += TPR) qr[k] = rs.round_odd(to_f32(xr[k]));
    return;
  }
  auto put = [&](int64_t k0, const Eight<T> &u) {
    float v[8];
    u.get(v);
    const uint2 w = make_uint2(rs.round4(v), rs.round4(v + 4));
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
    if (k0 < K) put(k0, held[c]);
  }
  for (int64_t k0 = (int64_t)(HELD * TPR + tid) * 8; k0 < K; k0 += TPR * 8) {
    Eight<T> u;
    u.template load<HOW>(xr + k0, min(8, K - (int)k0));
    put(k0, u);
  }
}

template <typename T, int TPR>
static void quantize_rows(har_cuda_ctx *ctx, const void *x, int how, int64_t M, int64_t K, int64_t ldx,
                          int8_t *q, int64_t ldq, float *scale, int q8) {
  constexpr int THREADS = TPR < 256 ? 256 : TPR;
  const unsigned grid = (unsigned)((M + THREADS / TPR - 1) / (THREADS / TPR));
  auto go = [&](auto kernel) {
    kernel<<<grid, THREADS, 0, ctx->stream>>>((const T *)x, M, (int)K, ldx, q, ldq, scale, q8);
  };
  if (how == WHOLE) go(i8_quantize_kernel<T, TPR, WHOLE>);
  else if (how == WIDE) go(i8_quantize_kernel<T, TPR, WIDE>);
  else go(i8_quantize_kernel<T, TPR, SINGLY>);
}

int32_t launch_i8_quantize(har_cuda_ctx *ctx, const void *x, int32_t dtype, int64_t M, int64_t K,
                           int64_t ldx, int8_t *q, int64_t ldq, float *scale) {
  const size_t eb = dtype_bytes(dtype);
  const bool wide = ((uintptr_t)x & 15u) == 0 && (M == 1 || (ldx * eb & 15u) == 0);
  const int how = !wide ? SINGLY : K % 8 == 0 ? WHOLE : WIDE;
  const int q8 = ((uintptr_t)q & 7u) == 0 && (M == 1 || (ldq & 7) == 0);
  prof_begin(ctx);
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    // as many threads as hold a row in registers at 32 values each
    if (K <= 1024)
      quantize_rows<T, 32>(ctx, x, how, M, K, ldx, q, ldq, scale, q8);
    else if (K <= 2048)
      quantize_rows<T, 64>(ctx, x, how, M, K, ldx, q, ldq, scale, q8);
    else if (K <= 4096)
      quantize_rows<T, 128>(ctx, x, how, M, K, ldx, q, ldq, scale, q8);
    else if (K <= 8192)
      quantize_rows<T, 256>(ctx, x, how, M, K, ldx, q, ldq, scale, q8);
    else
      quantize_rows<T, 512>(ctx, x, how, M, K, ldx, q, ldq, scale, q8);
  });
  return check_launch(ctx, "i8_quantize_kernel");
}

}  // namespace har
