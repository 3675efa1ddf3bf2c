// score.cuh — shared by the 8-bit integer products and the log-probability
// kernels: the weight handle, element types, the order of alternatives, and
// the kernel launchers that score.cu's entry points call.
#pragma once

#include <cuda_bf16.h>

#include "har_internal.cuh"

// A weight matrix [N][K] in 8-bit integers, one f32 scale per row.
struct har_cuda_i8_weights {
  const int8_t *q = nullptr;
  const float *scale = nullptr;
  int64_t N = 0, K = 0, ldq = 0;
  int device = 0, sms = 148;
  bool owned = false;  // q and scale share one allocation, at q
  // TMA map of q for the tensor-core kernels: boxes of 128 rows x 128 bytes
  TmaDesc map;
};

namespace har {

// Longest row whose integer sum fits in 32 bits with every product at its
// largest, 128 * 128: 131,071, rounded down to whole 16-byte pieces.
constexpr int64_t I8_MAX_K = 131056;
constexpr int64_t I8_MAX_ROWS = (int64_t)1 << 30;  // row numbers, tiles included, fit in 32 bits
constexpr int I8_MAX_TOP = HAR_CUDA_LOGPROBS_MAX_TOP;

inline size_t dtype_bytes(int32_t dtype) { return dtype == HAR_CUDA_DTYPE_F32 ? 4 : 2; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Order of alternatives as one unsigned 64-bit key: larger value first, then
// lower index.  The high word orders floats (-0 and +0 alike, NaN below -inf);
// the low word is the complement of the index.  0 is below every entry.
__device__ __forceinline__ uint32_t order_bits(float v) {
  const uint32_t b = __float_as_uint(__fadd_rn(v, 0.0f));
  if (v != v) return 0u;
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t o) {
  if (o == 0u) return __int_as_float(0x7fffffff);
  return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ unsigned long long order_key(float v, uint32_t id) {
  return ((unsigned long long)order_bits(v) << 32) | (0xffffffffu - id);
}

// max that keeps a NaN of either side
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The quantiser's rule for one row, from the largest |x| as bits (infinities
// and NaN order above every number): s = max|x| / 127, q = rint(x / s), both
// quotients rounded to f32.  The quotient by the row's one divisor: from
// y = 1/s rounded, two corrections q <- q + (x - q s) y.  The first brings q to
// within an ulp of x / s, the second is then correctly rounded (P. Markstein,
// IBM J. Res. Dev. 34, 1990), as long as the remainders are exact: s above
// 2^-100; rows below divide.  Adding 1.5 * 2^23 leaves the nearest integer,
// halves to even, in the low bits.  16-bit inputs land on halves often (x =
// max / 2 is 63.5), so a shortcut with a branch near halves took the branch in
// most warps (8192 x 4096 bf16: 36 us).
struct RowScale {
  static constexpr float MAGIC = 12582912.0f;
  float s, y;
  bool zero, tiny;
  __device__ __forceinline__ explicit RowScale(uint32_t top) {
    const bool finite = top < 0x7f800000u;
    s = finite ? __fdiv_rn(__uint_as_float(top), 127.0f) : __int_as_float(0x7fffffff);
    zero = !finite || s == 0.0f;
    tiny = s < 0x1p-100f;
    y = tiny || zero ? 0.0f : __fdiv_rn(1.0f, s);
  }
  __device__ __forceinline__ bool odd() const { return zero || tiny; }
  __device__ __noinline__ int8_t round_odd(float v) const {
    return zero ? (int8_t)0 : (int8_t)max(-127, min(127, (int)rintf(__fdiv_rn(v, s))));
  }
  __device__ __forceinline__ float2 nearest(float2 x) const {
    const float2 y2 = make_float2(y, y), ns = make_float2(-s, -s);
    float2 q = __fmul2_rn(x, y2);
    q = __ffma2_rn(__ffma2_rn(q, ns, x), y2, q);
    q = __ffma2_rn(__ffma2_rn(q, ns, x), y2, q);
    return __fadd2_rn(q, make_float2(MAGIC, MAGIC));
  }
  // four values as the bytes of a word; not where `odd`
  __device__ __forceinline__ uint32_t round4(const float *v) const {
    const float2 a = nearest(make_float2(v[0], v[1])), c = nearest(make_float2(v[2], v[3]));
    const uint32_t lo = __byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(c.x), __float_as_uint(c.y), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
  }
};

// Calls f with a value of the element type that `dtype` names.
template <typename F>
auto with_dtype(int32_t dtype, F &&f) {
  if (dtype == HAR_CUDA_DTYPE_F32) return f(float());
  if (dtype == HAR_CUDA_DTYPE_F16) return f(__half());
  return f(__nv_bfloat16());
}

// The outputs of one log-probability call; any of them may be null.
struct LogprobOut {
  const int32_t *tokens;
  int G, k;
  float *logprobs, *entropy, *top_logprobs;
  int32_t *top_ids;
  int *status;  // the context's device error word
};

int32_t launch_i8_quantize(har_cuda_ctx *ctx, const void *x, int32_t dtype, int64_t M, int64_t K,
                           int64_t ldx, int8_t *q, int64_t ldq, float *scale);
// padded: y's rows are padded to multiples of 16 bytes, and the padding may be
// written.
int32_t launch_i8_matmul(har_cuda_ctx *ctx, const har_cuda_i8_weights *w, const int8_t *q,
                         int64_t ldq, const float *scale, int64_t M, void *y, int32_t y_dtype,
                         int64_t ldy, bool padded = false);
// The product for a few rows: whether it takes these sizes, and the launch, from
// float rows (sx null: quantised on the way) or from 8-bit rows with scales sx.
bool i8_gemv_takes(int64_t M, int64_t N, int64_t K);
int32_t launch_i8_gemv(har_cuda_ctx *ctx, const har_cuda_i8_weights *w, const void *x, int32_t x_dtype,
                       int64_t ldx, const float *sx, int64_t M, void *y, int32_t y_dtype, int64_t ldy);
// The whole head call on a workspace of head_workspace_bytes.
size_t head_workspace_bytes(const har_cuda_i8_weights *w, int64_t T, int k);
int32_t launch_i8_head(har_cuda_ctx *ctx, const har_cuda_i8_weights *w, const void *x, int32_t x_dtype, int64_t ldx,
                       int64_t T, const LogprobOut &out, uint8_t *workspace);
int32_t launch_token_logprobs(har_cuda_ctx *ctx, const void *logits, int32_t dtype, int64_t T,
                              int64_t V, int64_t ldl, const LogprobOut &out);

}  // namespace har
