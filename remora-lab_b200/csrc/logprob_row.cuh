// logprob_row.cuh — the sums of one row's distribution, shared by the kernels
// that walk logits in memory and logits on the tensor cores:
//   s = sum exp(x - r),  t = sum exp(x - r) (x - r)  for a reference r near the
// row's maximum, so log p = (x - r) - log s and H = log s - t / s whatever r is.
#pragma once

#include "topk_warp.cuh"

namespace har {

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Sums about a reference: r starts at -inf (nothing seen but -inf and NaN).
struct Stat {
  float r, s, t;
};
// Moves the sums to reference r (>= a.r).  From -inf the sums are 0, or NaN.
__device__ __forceinline__ void stat_move(Stat &a, float r) {
  if (a.r == r) return;
  const float d = a.r - r, f = ex2(d * LOG2E);
  const float shift = a.r == -INFINITY ? 0.0f : f == 0.0f ? 0.0f : d;
  a.t = f * fmaf(shift, a.s, a.t);
  a.s = f * a.s;
  a.r = r;
}
__device__ __forceinline__ Stat warp_stat(Stat a) {
  stat_move(a, order_value(__reduce_max_sync(0xffffffffu, order_bits(a.r))));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
  }
  return a;
}

// What a row's sums say.  A row of -inf alone has no reference; a NaN or +inf
// makes s NaN.
struct RowEnd {
  float r, logz, s, entropy;
  bool empty;
  __device__ __forceinline__ explicit RowEnd(const Stat &st) : r(st.r), s(st.s) {
    empty = st.r == -INFINITY && st.s == 0.0f;
    logz = empty ? 0.0f : logf(st.s);
    entropy = empty ? 0.0f : logz - st.t / st.s;
  }
  __device__ __forceinline__ float logp(float v) const { return empty ? -INFINITY : (v - r) - logz; }
};

// Adds N values, the largest of them `top` (NaN left out), to the sums.  The
// reference follows the maximum only once it is left behind by more than 6
// (e^6 = 403 a term at most): a move costs an exponential, and close behind
// the maximum it would run at almost every call.  at(i) gives value i.
template <int N, typename At>
__device__ __forceinline__ void stat_add(Stat &a, float top, At &&at) {
  if (top > a.r + 6.0f) stat_move(a, top);
  const float r = a.r == -INFINITY ? 0.0f : a.r;
  const float2 nr = make_float2(-r, -r), l2e = make_float2(LOG2E, LOG2E);
  float2 s = make_float2(0.0f, 0.0f), t = s;  // added to the row's sums once: fewer roundings at their size
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    float2 d = __fadd2_rn(make_float2(at(i), at(i + 1)), nr);
    d.x = max_nan(d.x, -1e4f);  // -inf (0 times it would be NaN) and all that underflows
    d.y = max_nan(d.y, -1e4f);
    const float2 g = __fmul2_rn(d, l2e);
    const float2 e = make_float2(ex2(g.x), ex2(g.y));
    s = __fadd2_rn(s, e);
    t = __ffma2_rn(e, d, t);
  }
  a.s += s.x + s.y;
  a.t += t.x + t.y;
}

}  // namespace har
