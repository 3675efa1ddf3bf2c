// k_logprobs.cu — log probabilities of given tokens, entropy and the largest
// alternatives of each row of logits, in one pass over the row.
// 4,096 x 131,072: f32 303 us without alternatives (7.1 TB/s) and 337 with 5; bf16
// 182 and 202 (5.3 TB/s), where the exponentials' unit (56% busy) and the issue
// slots (67%) share the time with the loads.
#include <algorithm>
#include <cooperative_groups.h>

#include "logprob_row.cuh"

namespace har {

namespace cg = cooperative_groups;

constexpr int LP_U = 4, LP_MAX_CLUSTER = 16;
constexpr int LP_QUEUE = 256, LP_CAND = 512;
// One 16-byte piece of a row.
template <typename T>
struct Piece {
  static constexpr int N = 16 / sizeof(T);
  uint4 raw;
  // elements e0 .. e0 + N - 1 of the row at x, whole pieces with one load; an
  // element outside [0, V) reads as -inf, which adds nothing to the sums
  __device__ __forceinline__ void load(const T *x, int64_t e0, int64_t V) {
    if (e0 >= 0 && e0 + N <= V) {
      raw = ldg_nc_v4(x + e0);
    } else {
      T v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = e0 + i >= 0 && e0 + i < V ? x[e0 + i] : from_f32<T>(-INFINITY);
      raw = *reinterpret_cast<const uint4 *>(v);
    }
  }
  __device__ __forceinline__ void none() {
    T v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = from_f32<T>(-INFINITY);
    raw = *reinterpret_cast<const uint4 *>(v);
  }
  __device__ __forceinline__ float at(int i) const { return to_f32(reinterpret_cast<const T *>(&raw)[i]); }
  // largest element, NaN left out
  __device__ __forceinline__ float top() const;
};
template <>
__device__ __forceinline__ float Piece<float>::top() const {
  return fmaxf(fmaxf(at(0), at(1)), fmaxf(at(2), at(3)));
}
template <>
__device__ __forceinline__ float Piece<__half>::top() const {
  const __half2 *v = reinterpret_cast<const __half2 *>(&raw);
  const __half2 m = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
  return __half2float(__hmax(__low2half(m), __high2half(m)));
}
template <>
__device__ __forceinline__ float Piece<__nv_bfloat16>::top() const {
  const __nv_bfloat162 *v = reinterpret_cast<const __nv_bfloat162 *>(&raw);
  const __nv_bfloat162 m = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
  return __bfloat162float(__hmax(__low2bfloat16(m), __high2bfloat16(m)));
}

// A cluster of C blocks shares a row (C = 1: no cluster), each a contiguous
// part of its pieces, walked in trips of LP_T (its threads) x LP_U pieces.  The alternatives
// cost the walk one store: a thread notes the largest element of each trip (a
// group of LP_U pieces).  After some trips (LP_SEG) the k-th largest of 32 of
// the threads' largest elements bounds the k-th largest of all from below, so
// only groups that reach it (k or a few more of thousands) can hold an
// alternative: they are queued, read again from L2, one element a lane, and the
// elements that reach the bound are ranked by counting.
// Where ties are so many that the queue overflows, each warp goes through its
// own groups in order instead.
template <typename T, int LP_T>
__global__ void __launch_bounds__(LP_T, 1024 / LP_T)
    token_logprobs_kernel(const T *__restrict__ logits, int64_t V, int64_t ldl, LogprobOut out, int C) {
  constexpr int N = Piece<T>::N, LP_WARPS = LP_T / 32;
  constexpr int LP_SEG = LP_T == 256 ? 32 : 40;  // trips between two searches
  __shared__ float group_top[LP_SEG][LP_T];
  __shared__ uint32_t tops[32], least_s;
  __shared__ int queued, found;
  __shared__ int queue[LP_QUEUE];
  __shared__ key_t cand[LP_CAND];
  __shared__ key_t sorted[32];                 // the block's largest so far
  __shared__ key_t lists[LP_MAX_CLUSTER][32];  // the cluster's
  __shared__ key_t part_list[LP_WARPS][32];
  __shared__ Stat stats[LP_WARPS], part_stats[LP_MAX_CLUSTER];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x / C;
  const int rank = (int)(blockIdx.x - row * C);
  const T *x = logits + row * ldl;
  const bool want_top = out.k > 0 && (out.top_ids || out.top_logprobs);
  if (C > 1) cg::this_cluster().barrier_arrive();

  // the first given tokens' logits are asked for before anything else
  int32_t tok = -1;
  float given = 0.0f;
  if (rank == 0 && out.logprobs && tid < out.G) {
    tok = out.tokens[row * out.G + tid];
    if (tok >= 0 && tok < V) given = to_f32(x[tok]);
  }

  // pieces are 16-byte aligned: the first may start before the row
  const int off = (int)(((uintptr_t)x & 15u) / sizeof(T));
  const int64_t pieces = (V + off + N - 1) / N, share = (pieces + C - 1) / C;
  const int64_t j0 = rank * share, j1 = min(pieces, j0 + share);
  const int64_t whole0 = off ? 1 : 0, whole1 = min(j1, (V + off) / N);  // pieces inside the row
  auto load_trip = [&](Piece<T>(&p)[LP_U], int64_t jt) {
    if (jt >= whole0 && jt + LP_T * LP_U <= whole1) {
      const T *at = x + (jt + tid) * N - off;
#pragma unroll
      for (int u = 0; u < LP_U; ++u) p[u].raw = ldg_nc_v4(at + u * LP_T * N);
    } else {
#pragma unroll
      for (int u = 0; u < LP_U; ++u) {
        const int64_t j = jt + tid + u * LP_T;
        if (j < j1) p[u].load(x, j * N - off, V);
        else p[u].none();
      }
    }
  };
  Stat st = {-INFINITY, 0.0f, 0.0f};
  if (tid == 0) queued = found = 0, least_s = order_bits(-INFINITY) + 1u;  // -inf never enters: see the end
  if (tid < 32) sorted[tid] = 0;
  Piece<T> next[LP_U];
  if (j0 < j1) load_trip(next, j0);
  for (int64_t seg = j0; seg < j1; seg += (int64_t)LP_SEG * LP_T * LP_U) {
    float most = -INFINITY;
    const int trips = (int)min((int64_t)LP_SEG, (j1 - seg + LP_T * LP_U - 1) / (LP_T * LP_U));
    for (int s = 0; s < trips; ++s) {
      Piece<T> p[LP_U];
#pragma unroll
      for (int u = 0; u < LP_U; ++u) p[u] = next[u];
      const int64_t jn = seg + (int64_t)(s + 1) * (LP_T * LP_U);
      if (jn < j1) load_trip(next, jn);
      float top = p[0].top();
#pragma unroll
      for (int u = 1; u < LP_U; ++u) top = fmaxf(top, p[u].top());
      group_top[s][tid] = top;
      most = fmaxf(most, top);
      stat_add<LP_U * N>(st, top, [&](int i) { return p[i / N].at(i % N); });
    }
    if (!want_top) continue;
    // The k-th largest of 32 of the threads' largest, the best of each warp.
    // (The exact k-th of all, by counting, cost 2,600 cycles.)
    constexpr int EACH = 32 / LP_WARPS;
    const uint32_t mine = order_bits(most);
    uint32_t rest = mine;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const uint32_t m = warp_pop_max(rest, lane);
      if (lane == 0) tops[EACH * warp + i] = m;
    }
    __syncthreads();
    const uint32_t bound = max(warp_kth(tops[lane], out.k, lane), least_s);
    if (mine >= bound) {
#pragma unroll 4
      for (int s = 0; s < trips; ++s)
        if (order_bits(group_top[s][tid]) >= bound) {
          const int at = atomicAdd(&queued, 1);
          if (at < LP_QUEUE) queue[at] = s * LP_T + tid;
        }
    }
    // what the parts before had joins the new candidates
    if (tid < 32 && sorted[tid]) cand[atomicAdd(&found, 1)] = sorted[tid];
    __syncthreads();
    const int nq = queued;
    // element `lane` of a group, -inf outside the row
    auto element = [&](int g, int64_t &e) {
      const int64_t j = seg + (int64_t)(g / LP_T) * (LP_T * LP_U) + g % LP_T + (lane / N) * LP_T;
      e = j * N - off + lane % N;
      return lane < LP_U * N && j < j1 && e >= 0 && e < V ? to_f32(x[e]) : -INFINITY;
    };
    if (nq <= LP_QUEUE) {
      for (int i = warp; i < nq; i += 4 * LP_WARPS) {
        int64_t e[4];
        float v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          v[u] = -INFINITY;
          if (i + u * LP_WARPS < nq) v[u] = element(queue[i + u * LP_WARPS], e[u]);
        }
        uint32_t in[4];
        int total = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          in[u] = __ballot_sync(0xffffffffu, order_bits(v[u]) >= bound);
          total += __popc(in[u]);
        }
        int at = 0;
        if (lane == 0) at = atomicAdd(&found, total);
        at = __shfl_sync(0xffffffffu, at, 0) + __popc(in[0] & ((1u << lane) - 1u));
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (((in[u] >> lane) & 1u) && at < LP_CAND) cand[at] = order_key(v[u], (uint32_t)e[u]);
          if (u < 3) at += __popc(in[u] >> lane) + __popc(in[u + 1] & ((1u << lane) - 1u));
        }
      }
    }
    __syncthreads();
    const int n = found;
    if (nq <= LP_QUEUE && n <= LP_CAND) {
      if (seg > j0) {
        if (tid < 32) sorted[tid] = 0;
        __syncthreads();
      }
      if (n <= 64) {
        block_rank(cand, n, sorted, tid, LP_T);
      } else {
        key_t list = 0;
        for (int i = 32 * warp; i < n; i += LP_T)
          list = warp_merge_desc(list, warp_sort_desc(i + lane < n ? cand[i + lane] : (key_t)0, lane), lane);
        part_list[warp][lane] = list;
        __syncthreads();
        list = block_merge_lists(part_list, LP_WARPS, warp, lane);
        if (warp == 0) sorted[lane] = list;
      }
    } else {
      key_t list = 0;
      float bar = -INFINITY;  // the k-th entry's value, once there are k
      for (int s = 0; s < trips; ++s) {
        const float top = group_top[s][tid];
        // trips come in ascending order: a value equal to the k-th entry of
        // the trips before loses to it
        uint32_t groups = __ballot_sync(0xffffffffu, order_bits(top) >= bound && top > bar);
        if (!groups) continue;
        for (; groups; groups &= groups - 1) {
          int64_t e = 0;
          const float v = element(s * LP_T + 32 * warp + __ffs(groups) - 1, e);
          const key_t key = order_key(v, (uint32_t)e);
          const key_t last = __shfl_sync(0xffffffffu, list, out.k - 1);
          list = warp_take(list, key, __ballot_sync(0xffffffffu, v > -INFINITY && key > last), lane);
        }
        const key_t last = __shfl_sync(0xffffffffu, list, out.k - 1);
        if (last) bar = order_value((uint32_t)(last >> 32));
      }
      part_list[warp][lane] = list;
      __syncthreads();
      list = block_merge_lists(part_list, LP_WARPS, warp, lane);
      if (warp == 0) sorted[lane] = warp_merge_desc(list, sorted[lane], lane);
    }
    __syncthreads();
    if (tid == 0) {
      // what comes later and only equals the k-th entry loses to it
      const key_t last = sorted[out.k - 1];
      if (last) least_s = max(least_s, (uint32_t)(last >> 32) + 1u);
      queued = found = 0;
    }
    __syncthreads();
  }
  st = warp_stat(st);
  if (lane == 0) stats[warp] = st;
  __syncthreads();
  if (warp == 0) st = warp_stat(lane < LP_WARPS ? stats[lane] : Stat{-INFINITY, 0.0f, 0.0f});
  if (C > 1) {
    cg::cluster_group cl = cg::this_cluster();
    cl.barrier_wait();  // every block of the cluster has started: its shared memory is there
    if (warp == 0) {
      if (want_top) *cl.map_shared_rank(&lists[rank][lane], 0) = sorted[lane];
      if (lane == 0) *cl.map_shared_rank(&part_stats[rank], 0) = st;
    }
    cl.sync();
    if (rank != 0) return;
    st = warp_stat(lane < C ? part_stats[lane] : Stat{-INFINITY, 0.0f, 0.0f});
    if (want_top) {
      const key_t list = block_merge_lists(lists, C, warp, lane);
      if (warp == 0) sorted[lane] = list;
      __syncwarp();
    }
  } else {
    if (tid == 0) part_stats[0] = st;
    __syncthreads();
    st = part_stats[0];
  }

  const RowEnd row_end(st);
  if (tid == 0 && out.entropy) out.entropy[row] = row_end.entropy;
  if (out.logprobs)
    for (int g = tid; g < out.G; g += LP_T) {
      if (g >= LP_T) {
        tok = out.tokens[row * out.G + g];
        if (tok >= 0 && tok < V) given = to_f32(x[tok]);
      }
      float r = 0.0f;
      if (tok >= 0 && tok < V) {
        r = row_end.logp(given);
      } else if (tok != -1) {
        r = __int_as_float(0x7fffffff);
        atomicOr(out.status, DEV_ERR_BOUNDS);
      }
      out.logprobs[row * out.G + g] = r;
    }
  if (want_top && warp == 0) {
    const key_t best = sorted[lane];
    int id = best ? (int)(0xffffffffu - (uint32_t)best) : -1;
    float lp = best ? row_end.logp(order_value((uint32_t)(best >> 32))) : -INFINITY;
    // places left: the first masked elements, then the first NaN
    int have = __popc(__ballot_sync(0xffffffffu, best != 0));
    for (int pass = 0; pass < 2 && have < out.k; ++pass)
      for (int64_t e = lane; have < out.k && e - lane < V; e += 32) {
        const float v = e < V ? to_f32(x[e]) : 0.0f;
        uint32_t m = __ballot_sync(0xffffffffu, e < V && (pass == 0 ? v == -INFINITY : v != v));
        for (; m && have < out.k; m &= m - 1, ++have)
          if (lane == have) id = (int)(e - lane) + __ffs(m) - 1;
      }
    if (lane < out.k) {
      const int64_t o = row * out.k + lane;
      if (out.top_ids) out.top_ids[o] = id;
      if (out.top_logprobs) out.top_logprobs[o] = st.s != st.s ? st.s : lp;
    }
  }
}

// Blocks a row: the most, 1 to 16 and a power of two, that leave a block 12 KB
// while there is a block an SM at most, or 32 KB while there are two.  A cluster
// costs its blocks about 3 us to join: 148 rows of 131,072 f32 took 35, 24, 30
// and 34 us with 1, 2, 4 and 8 blocks a row, 37 rows 26, 19, 15 and 15, 301 rows
// 40, 44, 48 and 62; one row of 50,021 f16 took 13.5, 13.7, 12.0 and 11.2.
static int pick_cluster(int64_t T, int64_t bytes, int sms) {
  int c = 1;
  while (c < LP_MAX_CLUSTER) {
    const int64_t blocks = T * 2 * c, share = bytes / (2 * c);
    if (!(blocks <= sms && share >= 12 * 1024) && !(blocks <= 2 * sms && share >= 32 * 1024)) break;
    c *= 2;
  }
  return c;
}

int32_t launch_token_logprobs(har_cuda_ctx *ctx, const void *logits, int32_t dtype, int64_t T,
                              int64_t V, int64_t ldl, const LogprobOut &out) {
  const int C = pick_cluster(T, V * (int64_t)dtype_bytes(dtype), ctx->num_sms);
  cudaError_t e = cudaSuccess;
  // a grid holds 2^31 - 1 blocks
  const int64_t most = ((int64_t)1 << 30) / C;
  for (int64_t t0 = 0; t0 < T; t0 += most) {
    const int64_t rows = std::min(most, T - t0);
    LogprobOut o = out;
    if (o.tokens) o.tokens += t0 * o.G;
    if (o.logprobs) o.logprobs += t0 * o.G;
    if (o.entropy) o.entropy += t0;
    if (o.top_ids) o.top_ids += t0 * o.k;
    if (o.top_logprobs) o.top_logprobs += t0 * o.k;
    prof_begin(ctx);
    with_dtype(dtype, [&](auto t) {
      using E = decltype(t);
      // many rows, not the longest: blocks of 128 threads, so that more rows are
      // in different phases and the ends of some overlap the walks of others
      // (4,000 rows of 5,000 f32: 63 -> 47 us; 2,400 of 131,072 bf16: 138 -> 144)
      const bool narrow = C == 1 && T >= 4 * ctx->num_sms && V * (int64_t)sizeof(E) <= 128 * 1024;
      if (C > 8) e = cudaFuncSetAttribute(token_logprobs_kernel<E, 256>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e != cudaSuccess) return;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)(rows * C));
      cfg.blockDim = dim3(narrow ? 128 : 256);
      cfg.stream = ctx->stream;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = (unsigned)C;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = C > 1 ? 1 : 0;
      e = cudaLaunchKernelEx(&cfg, narrow ? token_logprobs_kernel<E, 128> : token_logprobs_kernel<E, 256>,
                             (const E *)logits + t0 * ldl, V, ldl, o, C);
    });
    const int32_t st = check_launch(ctx, "token_logprobs_kernel");
    if (e != cudaSuccess)
      return set_error(ctx, HAR_CUDA_ERR_CUDA, std::string("token_logprobs_kernel: ") + cudaGetErrorString(e));
    if (st != HAR_CUDA_OK) return st;
  }
  return HAR_CUDA_OK;
}

}  // namespace har
