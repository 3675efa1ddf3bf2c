// k_i8_gemv.cu — y = (q_x q_w^T) * s_x * s_w for a few rows, on the CUDA cores
// (dp4a): one launch that quantises the rows itself, no workspace.  Bound by
// the weights' bytes: one row of 131,072 x 4,096 takes 80 us, 6.7 TB/s.
#include <algorithm>

#include "score.cuh"

namespace har {

constexpr int V_T = 512, V_WARPS = V_T / 32, V_R = 2, V_UN = 2;
constexpr int V_MAX_SMEM = 24 * 1024;

struct GemvParams {
  const int8_t *w;
  const float *sw;
  int64_t N, K, ldw;
  const void *x;      // float rows of x_dtype, or 8-bit rows with their scales
  const float *sx;    // null: quantise x
  int64_t ldx;        // elements (bytes of 8-bit rows) between rows
  int x_dtype, M, wide;
  void *y;
  int64_t ldy;
};

// Elements i .. i + 3 of a row of n; `wide`: one load for the four.
__device__ __forceinline__ void load4(const void *x, int dtype, int64_t at, int left, bool wide, float (&v)[4]) {
  if (wide && left >= 4) {
    if (dtype == HAR_CUDA_DTYPE_F32) {
      const float4 a = *reinterpret_cast<const float4 *>((const float *)x + at);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    } else {
      const uint2 a = *reinterpret_cast<const uint2 *>((const uint16_t *)x + at);
      const uint32_t w[2] = {a.x, a.y};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned short b = (unsigned short)(w[i >> 1] >> (16 * (i & 1)));
        v[i] = dtype == HAR_CUDA_DTYPE_F16 ? __half2float(__ushort_as_half(b)) : __uint_as_float((uint32_t)b << 16);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = 0.0f;
    if (i < left)
      v[i] = dtype == HAR_CUDA_DTYPE_F32   ? ((const float *)x)[at + i]
             : dtype == HAR_CUDA_DTYPE_F16 ? __half2float(((const __half *)x)[at + i])
                                           : __bfloat162float(((const __nv_bfloat16 *)x)[at + i]);
  }
}

// MT rows (the last ones repeated as zeros) share every weight read.  A warp
// takes V_R neighbouring channels at a time, lanes over 16-byte pieces of K,
// and adds its lanes' integer sums with one reduction instruction each.  A
// step's pieces are asked for one step ahead, the first before the rows are
// quantised: at the smallest sizes the two latencies are all there is.
template <typename T, int MT>
__global__ void __launch_bounds__(V_T, 2) i8_gemv_kernel(const GemvParams p) {
  extern __shared__ __align__(16) uint8_t v_raw[];  // q [MT][pieces][16]
  __shared__ float scale[MT];
  __shared__ uint32_t part[V_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int pieces = (int)((p.K + 15) / 16);
  const int64_t step = (int64_t)gridDim.x * V_WARPS * V_R;
  int64_t n0 = ((int64_t)blockIdx.x * V_WARPS + warp) * V_R;

  auto load = [&](uint4(&w)[V_UN][V_R], int64_t n, int i0) {
#pragma unroll
    for (int u = 0; u < V_UN; ++u) {
      const int c = i0 + u * 32 + lane;
#pragma unroll
      for (int r = 0; r < V_R; ++r)
        w[u][r] = c < pieces && n + r < p.N ? ldg_nc_v4(p.w + (n + r) * p.ldw + 16 * (int64_t)c) : make_uint4(0, 0, 0, 0);
    }
  };
  uint4 next[V_UN][V_R];
  load(next, n0, 0);

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
    const int64_t x0 = m * p.ldx;
    float most = 0.0f;
    for (int k = 4 * t; live && k < (int)p.K; k += WPR * 128) {
      float v[4];
      load4(p.x, p.x_dtype, x0 + k, (int)p.K - k, p.wide, v);
      most = max_nan(max_nan(most, max_nan(fabsf(v[0]), fabsf(v[1]))), max_nan(fabsf(v[2]), fabsf(v[3])));
    }
    uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
    if (lane == 0) part[warp] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WPR; ++i) top = max(top, part[m * WPR + i]);
    const RowScale rs(top);
    if (t == 0) scale[m] = rs.s;
    uint32_t *q = (uint32_t *)v_raw + (int64_t)m * pieces * 4;
    for (int k = 4 * t; k < pieces * 16; k += WPR * 128) {
      float v[4];
      load4(p.x, p.x_dtype, x0 + k, live ? (int)p.K - k : 0, p.wide, v);
      if (rs.odd()) {
        uint32_t w = 0;
        for (int i = 0; i < 4; ++i) w |= (uint32_t)(uint8_t)rs.round_odd(v[i]) << (8 * i);
        q[k >> 2] = w;
      } else {
        q[k >> 2] = rs.round4(v);
      }
    }
  }
  __syncthreads();

  const uint4 *xq = reinterpret_cast<const uint4 *>(v_raw);
  int acc[V_R][MT] = {};
  for (int i0 = 0; n0 < p.N;) {
    uint4 w[V_UN][V_R];
#pragma unroll
    for (int u = 0; u < V_UN; ++u)
#pragma unroll
      for (int r = 0; r < V_R; ++r) w[u][r] = next[u][r];
    const int i1 = i0 + 32 * V_UN;
    const bool end = i1 >= pieces;
    load(next, end ? n0 + step : n0, end ? 0 : i1);  // past the last channel: no loads
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
    i0 = i1;
    if (!end) continue;
    i0 = 0;
    int mine = 0;  // lane r * MT + m keeps the sum of (channel r, row m)
#pragma unroll
    for (int r = 0; r < V_R; ++r)
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int s = __reduce_add_sync(0xffffffffu, acc[r][m]);
        if (lane == r * MT + m) mine = s;
        acc[r][m] = 0;
      }
    const int r = lane / MT, m = lane % MT;
    if (lane < V_R * MT && m < p.M && n0 + r < p.N)
      ((T *)p.y)[m * p.ldy + n0 + r] =
          from_f32<T>(__fmul_rn(__int2float_rn(mine), __fmul_rn(scale[m], __ldg(p.sw + n0 + r))));
    n0 += step;
  }
}

static int gemv_rows(int64_t M) { return M <= 1 ? 1 : M <= 2 ? 2 : M <= 4 ? 4 : 8; }

// Up to 4 rows, and 8 of a small matrix, that take 24 KB: above, the tensor cores'
// launch and its quantising pass cost less than quantising the rows in every
// block and a dp4a a row and four bytes.  Here and there, us: 131,072 x 4,096 with
// 2 rows 80 and 91, 4 rows 96 and 91; 4,096 x 2,048 with 4 rows 8.2 and 12.3, 8
// rows 10.3 and 12.3; 8 rows of 65,536 x 2,048 47 and 31; 512 x 4,096 with 4 rows
// 10.3 and 12.3, 8 rows 16.4 and 12.3; 1,024 x 16,384 with one row 18.5 and 19.5, 2
// rows 22.6 and 19.5.  Up to 4 rows the rule does not look at N: the 4 rows of
// 131,072 x 4,096 lose their 5 us by it.
bool i8_gemv_takes(int64_t M, int64_t N, int64_t K) {
  return (M <= 4 || (M <= 8 && N * K <= 8 << 20)) && gemv_rows(M) * ((K + 15) / 16 * 16) <= V_MAX_SMEM;
}

int32_t launch_i8_gemv(har_cuda_ctx *ctx, const har_cuda_i8_weights *w, const void *x, int32_t x_dtype,
                       int64_t ldx, const float *sx, int64_t M, void *y, int32_t y_dtype, int64_t ldy) {
  GemvParams p = {};
  p.w = w->q, p.sw = w->scale, p.N = w->N, p.K = w->K, p.ldw = w->ldq;
  p.x = x, p.sx = sx, p.ldx = ldx, p.x_dtype = x_dtype, p.M = (int)M, p.y = y, p.ldy = ldy;
  const size_t eb = dtype_bytes(x_dtype);
  p.wide = sx == nullptr && ((uintptr_t)x & (4 * eb - 1)) == 0 && (M == 1 || ldx % 4 == 0);
  const int mt = gemv_rows(M);
  const size_t smem = (size_t)mt * (size_t)((w->K + 15) / 16 * 16);
  const int64_t blocks = (w->N + V_WARPS * V_R - 1) / (V_WARPS * V_R);
  const unsigned grid = (unsigned)std::min<int64_t>(blocks, 2 * ctx->num_sms);
  auto go = [&](auto kernel) { kernel<<<grid, V_T, smem, ctx->stream>>>(p); };
  prof_begin(ctx);
  with_dtype(y_dtype, [&](auto t) {
    using T = decltype(t);
    if (mt == 1) go(i8_gemv_kernel<T, 1>);
    else if (mt == 2) go(i8_gemv_kernel<T, 2>);
    else if (mt == 4) go(i8_gemv_kernel<T, 4>);
    else go(i8_gemv_kernel<T, 8>);
  });
  return check_launch(ctx, "i8_gemv_kernel");
}

}  // namespace har
