// k_logprobs.cu — log probabilities of given tokens, entropy and the largest
// alternatives of each row of logits.
#include "score.cuh"

namespace har {

// Running sums of a softmax: m the largest logit, s = sum exp(x - m),
// t = sum exp(x - m) (x - m).  A logit of -inf adds nothing.
struct Stat {
  float m, s, t;
};
__device__ __forceinline__ Stat stat_merge(Stat a, Stat b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return {m, a.s + b.s, a.t + b.t};  // both empty, or NaN kept in the sums
  auto part = [m](Stat c, float &s, float &t) {
    if (c.m == -INFINITY) {
      s = c.s, t = c.t;
      return;
    }
    const float d = c.m - m, e = expf(d);
    s = c.s * e;
    t = e == 0.0f ? 0.0f * c.t : e * (c.t + d * c.s);
  };
  float s1, t1, s2, t2;
  part(a, s1, t1);
  part(b, s2, t2);
  return {m, s1 + s2, t1 + t2};
}

template <typename T>
__global__ void __launch_bounds__(256)
    token_logprobs_kernel(const T *__restrict__ x, int64_t V, int64_t ldl, LogprobOut out) {
  __shared__ Stat stats[8];
  __shared__ unsigned long long keys[8];
  const int64_t row = blockIdx.x;
  const T *xr = x + row * ldl;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Stat st = {-INFINITY, 0.0f, 0.0f};
  for (int64_t i = threadIdx.x; i < V; i += 256) {
    const float v = to_f32(xr[i]);
    if (v != -INFINITY) st = stat_merge(st, {v, v != v ? v : 1.0f, 0.0f});
  }
  for (int o = 16; o; o >>= 1) {
    Stat b = {__shfl_xor_sync(~0u, st.m, o), __shfl_xor_sync(~0u, st.s, o), __shfl_xor_sync(~0u, st.t, o)};
    st = stat_merge(st, b);
  }
  if (lane == 0) stats[warp] = st;
  __syncthreads();
  st = stats[0];
  for (int w = 1; w < 8; ++w) st = stat_merge(st, stats[w]);
  const bool empty = st.m == -INFINITY && !(st.s != st.s);
  const float logz = empty ? 0.0f : logf(st.s);
  auto logp = [&](float v) { return empty ? -INFINITY : (v - st.m) - logz; };
  if (threadIdx.x == 0 && out.entropy) out.entropy[row] = empty ? 0.0f : logz - st.t / st.s;
  if (out.logprobs)
    for (int g = threadIdx.x; g < out.G; g += 256) {
      const int32_t tok = out.tokens[row * out.G + g];
      float r = 0.0f;
      if (tok >= 0 && tok < V) {
        r = logp(to_f32(xr[tok]));
      } else if (tok != -1) {
        r = __int_as_float(0x7fffffff);
        atomicOr(out.status, DEV_ERR_BOUNDS);
      }
      out.logprobs[row * out.G + g] = r;
    }
  if (!out.top_ids && !out.top_logprobs) return;
  unsigned long long last = ~0ull;
  for (int j = 0; j < out.k; ++j) {
    unsigned long long best = 0;
    for (int64_t i = threadIdx.x; i < V; i += 256) {
      const unsigned long long key = order_key(to_f32(xr[i]), (uint32_t)i);
      if (key < last && key > best) best = key;
    }
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(~0u, best, o));
    __syncthreads();
    if (lane == 0) keys[warp] = best;
    __syncthreads();
    for (int w = 0; w < 8; ++w) best = max(best, keys[w]);
    last = best;
    if (threadIdx.x == 0) {
      if (out.top_ids) out.top_ids[row * out.k + j] = best ? (int32_t)(0xffffffffu - (uint32_t)best) : -1;
      if (out.top_logprobs)
        out.top_logprobs[row * out.k + j] =
            st.s != st.s ? st.s : best ? logp(order_value((uint32_t)(best >> 32))) : -INFINITY;
    }
  }
}

int32_t launch_token_logprobs(har_cuda_ctx *ctx, const void *logits, int32_t dtype, int64_t T,
                              int64_t V, int64_t ldl, const LogprobOut &out) {
  prof_begin(ctx);
  with_dtype(dtype, [&](auto t) {
    using E = decltype(t);
    token_logprobs_kernel<E><<<(unsigned)T, 256, 0, ctx->stream>>>((const E *)logits, V, ldl, out);
  });
  return check_launch(ctx, "token_logprobs_kernel");
}

}  // namespace har
