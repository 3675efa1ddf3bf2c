// k_i8_head.cu — log probabilities straight from hidden states and an 8-bit LM
// head: the product's epilogue folds every logit into its row's sums and keeps
// the largest, so many rows' logits are never stored (f32 logits of 2,048
// tokens x 131,072 would be 1 GB written and 1 GB read back).  2,048 x 131,072 x
// 2,048 takes 350 us without alternatives, 3.1 POP/s, and 376 with 5 of them, what
// the lists add to the epilogue.
#include <algorithm>

#include "i8_mma.cuh"
#include "logprob_row.cuh"

namespace har {

// A pair of blocks works on tiles of 256 tokens (tensor-memory lanes) x 256
// vocabulary rows (columns): a thread of the epilogue owns one token and half
// the columns, and keeps the token's sums and list to itself.
constexpr int H_TILE = 2 * G_A, H_COLS = 128;
constexpr int H_ROW = 8 * G_EPI_THREADS;  // bytes between two entries of a thread's list
constexpr int H_SLOT = 2 * G_A * G_KS;    // bytes of a k-step
// Ring slots and entries of a thread's list, which share a block's memory: a
// list of 40 leaves four slots, and up to 32 entries one sort cuts it.  Above 22
// alternatives that leaves too few new entries between two cuts (2,048 x 131,072 x
// 2,048 with 5: 384 us with 40 entries and 405 with 60; with 20: 445 and 449, 24:
// 500 and 466, 32: 3,148 and 604): a list of 60 beside three slots.
constexpr int H_SLOTS = 4, H_CAP = 40, H_SLOTS_LONG = 3, H_CAP_LONG = 60, H_LONG = 22;
// Bytes of either division.  Every launch asks for the larger: the function's
// limit belongs to the process, and another thread's smaller one would refuse it.
constexpr size_t H_SMEM = (size_t)std::max(H_SLOTS * H_SLOT + H_CAP * H_ROW, H_SLOTS_LONG * H_SLOT + H_CAP_LONG * H_ROW) + 1024;
constexpr int H_PEERS = 16;  // parts that a part asks
constexpr int H_JOIN = 64, H_JOIN_MOST = 320;  // threads of a joining block: one a part
constexpr int64_t H_TOKENS = 4096;  // tokens of one launch
constexpr int64_t H_WALK_TOKENS = 64, H_WALK_BYTES = 12 << 20;

struct HeadPlan {
  int tt, vt, g, C;                 // token tiles, vocabulary tiles, token tiles at a time, vocabulary streams
  int64_t Tp;                       // tokens rounded up to tiles
  int parts() const { return 2 * C; }
  int blocks() const { return 2 * g * C; }
};

struct HeadParams {
  RingShape sh;
  int64_t T, V, Tp;
  const float *sx, *sw;
  int tt, vt, g, C, k;
  int full;                        // entries at which a list is cut back: 8 below its room
  // part 2 c + h (stream c, half h of a tile's columns) of token t at [part][t]
  float *part_r, *part_s, *part_t;
  key_t *part_best;                // its largest key, 0: no entry
  int32_t *part_n;                 // its entries
  float *part_v;                   // [part][k][Tp]
  int32_t *part_i;
  uint64_t *best2;                 // [part][Tp]: order_bits of two of its logits, 0 at first
  int *status;
};

// Pair b works on token tile pass * g + b / C and vocabulary tiles b % C,
// b % C + C, ...: the g pairs of a stream read the same weights at about the
// same time, so they come from memory once.
struct HeadTiles {
  const HeadParams &p;
  int slot, c, pass, v;
  __device__ __forceinline__ explicit HeadTiles(const HeadParams &p_) : p(p_), pass(0) {
    const int b = blockIdx.x / 2;
    slot = b / p.C;
    c = v = b - slot * p.C;
  }
  __device__ __forceinline__ bool next(int &a_row, int &b_row) {
    if (v >= p.vt) {
      ++pass;
      v = c;
    }
    const int t = pass * p.g + slot;
    if (t >= p.tt) return false;
    a_row = t * H_TILE;
    b_row = v * H_TILE;
    v += p.C;
    return true;
  }
};

// N values (a power of two) a thread in descending order (bitonic, in registers).
template <int N>
__device__ __forceinline__ void sort_desc(float (&v)[N]) {
#pragma unroll
  for (int size = 2; size <= N; size <<= 1)
#pragma unroll
    for (int step = size >> 1; step > 0; step >>= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int j = i ^ step;
        if (j > i) {
          const float hi = fmaxf(v[i], v[j]), lo = fminf(v[i], v[j]);
          const bool desc = (i & size) == 0;
          v[i] = desc ? hi : lo;
          v[j] = desc ? lo : hi;
        }
      }
}
// a <- the 32 largest of two descending runs.
__device__ __forceinline__ void merge32_desc(float (&a)[32], const float (&b)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) a[i] = fmaxf(a[i], b[31 - i]);
#pragma unroll
  for (int step = 16; step > 0; step >>= 1)
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const int j = i ^ step;
      if (j > i) {
        const float hi = fmaxf(a[i], a[j]), lo = fminf(a[i], a[j]);
        a[i] = hi;
        a[j] = lo;
      }
    }
}
template <int N>
__device__ __forceinline__ float pick(const float (&v)[N], int i) {
  float r = v[0];
#pragma unroll
  for (int j = 1; j < N; ++j) r = j == i ? v[j] : r;
  return r;
}

// The parts of a token tell each other their two largest logits so far.  The
// k-th largest of what H_PEERS of them tell bounds the k-th largest of all from below, and far closer than a
// part's own k-th: 1 or 2 of the logits that a part has seen reach it, not k.
// Both in one word: the first of one telling and the second of a later one may
// be the same logit.
__device__ __forceinline__ void tell_best2(uint64_t *at, float a, float b) {
  const uint64_t two = ((uint64_t)order_bits(b) << 32) | order_bits(a);
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(at), "l"(two) : "memory");
}
// A float just below that bound: what equals it may have the lower id.
__device__ __noinline__ float peers_bar(const uint64_t *best2, int64_t Tp, int part, int parts, int k) {
  float v[2 * H_PEERS];
#pragma unroll
  for (int i = 0; i < H_PEERS; ++i) {
    uint64_t two = 0;
    const int p = part + i < parts ? part + i : part + i - parts;
    if (i < parts)
      asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(two) : "l"(best2 + p * Tp) : "memory");
    const uint32_t a = (uint32_t)two, b = (uint32_t)(two >> 32);
    v[2 * i] = a ? order_value(a) : -INFINITY;
    v[2 * i + 1] = b ? order_value(b) : -INFINITY;
  }
  sort_desc(v);
  // two steps down: the one below +0 is -0, its equal; of -inf a NaN, no bar
  return order_value(order_bits(pick(v, k - 1)) - 2u);
}

// A thread's list in shared memory: entries (value, id), H_ROW bytes apart,
// from `at`; `end` is behind the last, values above `bar` may enter.
struct List {
  uint32_t at, end;
  float bar;
  __device__ __forceinline__ int n() const { return (int)(end - at) / H_ROW; }
};
__device__ __forceinline__ float list_value(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ int32_t list_id(uint32_t at) {
  int32_t v;
  asm volatile("ld.shared.s32 %0, [%1+4];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
// Appends (v, id) if v is above the bar: four instructions and no branch.
__device__ __forceinline__ void list_push(List &l, float v, int32_t id) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.gt.f32 p, %1, %2;\n\t"
      "@p st.shared.v2.b32 [%0], {%3, %4};\n\t"
      "@p add.u32 %0, %0, %5;\n\t}"
      : "+r"(l.end)
      : "f"(v), "f"(l.bar), "r"(__float_as_uint(v)), "r"(id), "n"(H_ROW)
      : "memory");
}
// Cuts a list back to its k largest entries: the k-th value from a sort of the
// values alone, then one sweep that keeps what is above it and, of its equals,
// the first (entries stand in the order of their ids).  The whole warp; a
// thread with fewer than k entries keeps them and its bar.  A list holds 32
// entries and `MORE`.
template <int MORE>
__device__ __noinline__ List list_cut(List s, int k) {
  float top[32];
  const int n = s.n();
#pragma unroll
  for (int i = 0; i < 32; ++i) top[i] = i < n ? list_value(s.at + i * H_ROW) : -INFINITY;
  sort_desc(top);
  if (__any_sync(0xffffffffu, n > 32)) {
    float more[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) more[i] = i < MORE && 32 + i < n ? list_value(s.at + (32 + i) * H_ROW) : -INFINITY;
    sort_desc(more);
    merge32_desc(top, more);
  }
  if (n < k) return s;
  const float bar = pick(top, k - 1);
  int equals = k;
#pragma unroll
  for (int i = 0; i < 32; ++i) equals -= i < k && top[i] > bar;
  uint32_t end = s.at;
  for (uint32_t e = s.at; e < s.end; e += H_ROW) {
    const float x = list_value(e);
    const int32_t id = list_id(e);
    if (x > bar || (x == bar && equals-- > 0)) {
      asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(end), "r"(__float_as_uint(x)), "r"(id) : "memory");
      end += H_ROW;
    }
  }
  return {s.at, end, bar};
}

__global__ void __launch_bounds__(G_THREADS, 1)
    i8_head_kernel(const __grid_constant__ TmaDesc map_x, const __grid_constant__ TmaDesc map_w, const HeadParams p) {
  extern __shared__ uint8_t g_raw[];
  __shared__ Ring ring;
  __shared__ int go[2][2];
  __shared__ __align__(16) float scales[2][2][H_COLS];
  uint8_t *sm = g_raw + ((1024u - (tc::smem_u32(g_raw) & 1023u)) & 1023u);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = tc::cluster_rank();
  ring_open<2>(ring, p.sh, &map_x, &map_w);

  if (warp == G_WARP_A) {
    ring_produce<2>(ring, p.sh, sm, false, &map_x, HeadTiles(p), rank);
  } else if (warp == G_WARP_B) {
    ring_produce<2>(ring, p.sh, sm, true, &map_w, HeadTiles(p), rank);
  } else if (warp == G_WARP_MMA) {
    if (rank == 0) ring_issue<2>(ring, p.sh, sm, HeadTiles(p));
  } else {
    volatile int *abort_s = &ring.abort_flag;
    const int quad = warp & 3, h = (warp - G_WARP_EPI) >> 2;
    const int row = 32 * quad + lane;
    const uint32_t col0 = ring.tmem + ((uint32_t)(32 * quad) << 16) + (uint32_t)(h * H_COLS);
    HeadTiles tiles(p);
    Stat st = {-INFINITY, 0.0f, 0.0f};
    List ls;
    ls.at = ls.end = tc::smem_u32(sm + p.sh.stages * H_SLOT) + 8u * (uint32_t)(128 * h + row);
    ls.bar = INFINITY;
    int64_t token = -1;
    float sx = 0.0f;
    int cur = -1;

    const int mine = 2 * tiles.c + h;  // this thread's part
    int walked = 0;                    // tiles of the token tile so far
    auto cut = [&](const List &l) {
      List c = p.k > H_LONG ? list_cut<H_CAP_LONG - 32>(l, p.k) : list_cut<H_CAP - 32>(l, p.k);
      c.bar = fmaxf(c.bar, l.bar);  // the peers' may be higher
      return c;
    };
    // after 1, 2, 4, ... tiles: tells the list's two largest, and learns (2,048 x
    // 131,072 x 2,048 with 5, 20 and 32: 418, 575 and 704 us without, 376, 460 and
    // 610 with it; 768 tokens with 8 and 20: 218 and 293, 188 and 234)
    auto confer = [&]() {
      float a = -INFINITY, b = -INFINITY;
      for (uint32_t e = ls.at; e < ls.end; e += H_ROW) {
        const float x = list_value(e);
        b = fmaxf(b, fminf(a, x));
        a = fmaxf(a, x);
      }
      if (token >= p.T) return;
      if (b > -INFINITY) tell_best2(p.best2 + mine * p.Tp + token, a, b);
      ls.bar = fmaxf(ls.bar, peers_bar(p.best2 + token, p.Tp, mine, 2 * p.C, p.k));
    };
    // the token tile's part is done
    auto flush = [&]() {
      if (p.k > 0) ls = cut(ls);
      if (token >= p.T) return;
      const int64_t part = 2 * tiles.c + h, at = part * p.Tp + token;
      p.part_r[at] = st.r;
      p.part_s[at] = st.s;
      p.part_t[at] = st.t;
      if (p.k == 0) return;
      key_t best = 0;
      const int n = ls.n();
      for (int e = 0; e < n; ++e) {
        const float x = list_value(ls.at + e * H_ROW);
        const int32_t id = list_id(ls.at + e * H_ROW);
        const int64_t to = (part * p.k + e) * p.Tp + token;
        p.part_v[to] = x;
        p.part_i[to] = id;
        best = key_max(best, order_key(x, (uint32_t)id));
      }
      p.part_n[at] = n;
      p.part_best[at] = best;
    };

    int a_row, b_row;
    for (uint32_t n = 0; tiles.next(a_row, b_row); ++n) {
      const uint32_t a = n & 1u;
      bool first = false;
      if (a_row != cur) {
        if (cur >= 0) flush();
        cur = a_row;
        first = p.k > 0;
        token = (int64_t)a_row + rank * G_A + row;
        sx = token < p.T ? __ldg(p.sx + token) : 0.0f;
        st = {-INFINITY, 0.0f, 0.0f};
        ls.end = ls.at;
        ls.bar = token < p.T ? -INFINITY : INFINITY;
        walked = 0;
      }
      const int64_t v0 = (int64_t)b_row + h * H_COLS;  // this half's first vocabulary row
      scales[a][h][row] = v0 + row < p.V ? __ldg(p.sw + v0 + row) : 0.0f;
      // one warp waits for the half and says whether to go on, so that all four
      // leave together when a wait gave up
      if (quad == 0) {
        const bool ok = g_wait_warp(ring.acc_full + a, (n >> 1) & 1u, abort_s, lane, 256);
        if (lane == 0) go[h][a] = ok;
      }
      tc::bar_sync(1 + h, 128);
      if (!go[h][a]) {
        cur = -1;  // nothing to flush
        break;
      }
      tc::tc_fence_after();
      const uint32_t col = col0 + a * 256u;
      const int width = (int)min((int64_t)H_COLS, p.V - v0);  // columns within V
      uint32_t v[32];
      // 32 logits from column c on, as i8_linear writes them; -inf past V
      auto logits = [&](int c, float (&l)[32]) {
        __syncwarp();  // lists grow and are cut lane by lane
        tc::tmem_wait_ld32(v);
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 s = *reinterpret_cast<const float4 *>(&scales[a][h][c + i]);
          l[i] = __fmul_rn(__int2float_rn((int)v[i]), __fmul_rn(sx, s.x));
          l[i + 1] = __fmul_rn(__int2float_rn((int)v[i + 1]), __fmul_rn(sx, s.y));
          l[i + 2] = __fmul_rn(__int2float_rn((int)v[i + 2]), __fmul_rn(sx, s.z));
          l[i + 3] = __fmul_rn(__int2float_rn((int)v[i + 3]), __fmul_rn(sx, s.w));
        }
        if (c + 32 > width) {
#pragma unroll
          for (int i = 0; i < 32; ++i) l[i] = c + i < width ? l[i] : -INFINITY;
        }
      };
      if (first) {
        // the k-th largest of 32 groups' largest logits: k logits are at least
        // as large, so the list starts behind a float below them
        float top[32];
#pragma unroll
        for (int c = 0; c < H_COLS; c += 32) {
          float l[32];
          tc::tmem_ld32(col + (uint32_t)c, v);
          logits(c, l);
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            top[(c + i) / 4] = fmaxf(fmaxf(fmaxf(l[i], l[i + 1]), fmaxf(l[i + 2], l[i + 3])), -INFINITY);
        }
        sort_desc(top);
        const uint32_t o = order_bits(pick(top, p.k - 1));
        if (token < p.T && top[1] > -INFINITY) tell_best2(p.best2 + mine * p.Tp + token, top[0], top[1]);
        if (token < p.T) ls.bar = order_value(max(o - 2u, order_bits(-INFINITY)));
      }
      if (p.k > 0) {
        if (walked > 0 && (walked & (walked - 1)) == 0) confer();
        ++walked;
      }
      // lanes past T told and asked nothing: the warp is whole again before
      // tcgen05.ld, which all its lanes execute together
      __syncwarp();
      tc::tmem_ld32(col, v);
#pragma unroll 1
      for (int c = 0; c < H_COLS; c += 32) {
        float l[32];
        logits(c, l);
        if (c + 32 < H_COLS) tc::tmem_ld32(col + (uint32_t)(c + 32), v);
        else ring_release<2>(ring, a, lane);
        float top[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          top[q] = l[8 * q];
#pragma unroll
          for (int i = 1; i < 8; ++i) top[q] = fmaxf(top[q], l[8 * q + i]);
        }
        if (p.k > 0) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (__any_sync(0xffffffffu, top[q] > ls.bar)) {
#pragma unroll
              for (int i = 8 * q; i < 8 * q + 8; ++i) list_push(ls, l[i], (int32_t)v0 + c + i);
              if (__any_sync(0xffffffffu, ls.n() > p.full)) ls = cut(ls);
            }
        }
        stat_add<32>(st, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), [&](int i) { return l[i]; });
      }
    }
    if (cur >= 0) flush();
  }
  ring_close<2>(ring, p.status);
}

// ---- joining the parts --------------------------------------------------------------

struct HeadJoin {
  HeadParams p;
  LogprobOut out;
  const int8_t *x, *w;   // quantised rows, for the given tokens' logits
  int64_t ldx, ldw, K;
  int parts;
};

// Exact dot product of two 8-bit rows by one warp.
__device__ __forceinline__ int warp_dot(const int8_t *a, const int8_t *b, int64_t K, int lane) {
  int acc = 0;
  for (int64_t k = 16 * lane; k < K; k += 512) {
    if (k + 16 <= K) {
      const uint4 u = ldg_nc_v4(a + k), v = ldg_nc_v4(b + k);
      acc = __dp4a((int)u.x, (int)v.x, acc);
      acc = __dp4a((int)u.y, (int)v.y, acc);
      acc = __dp4a((int)u.z, (int)v.z, acc);
      acc = __dp4a((int)u.w, (int)v.w, acc);
    } else {
      for (int i = 0; k + i < K; ++i) acc += (int)a[k + i] * (int)b[k + i];
    }
  }
  return __reduce_add_sync(0xffffffffu, acc);
}

// One block a token.  The alternatives are found as in the walk over logits: a
// part whose largest key is below the k-th largest of the parts' has none, so
// at most k parts, of at most k entries each, are read.
template <int TH>
__global__ void __launch_bounds__(TH) head_join_kernel(const HeadJoin j) {
  constexpr int W = TH / 32, LISTS = W <= 2 ? 2 : 16;
  __shared__ Stat stats[W];
  __shared__ key_t lists[LISTS][32];
  __shared__ key_t cand[I8_MAX_TOP * I8_MAX_TOP];
  __shared__ key_t bound_s;
  __shared__ int count;
  const HeadParams &p = j.p;
  const LogprobOut &out = j.out;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t t = blockIdx.x;
  const float sx = p.sx[t];
  Stat st = {-INFINITY, 0.0f, 0.0f};
  if (tid < j.parts) {
    const int64_t at = (int64_t)tid * p.Tp + t;
    st = {p.part_r[at], p.part_s[at], p.part_t[at]};
  }
  st = warp_stat(st);
  if (lane == 0) stats[warp] = st;
  key_t best = p.k > 0 && tid < j.parts ? p.part_best[(int64_t)tid * p.Tp + t] : 0;
  for (int i = tid; i < LISTS * 32; i += TH) (&lists[0][0])[i] = 0;
  if (tid == 0) count = 0;
  __syncthreads();
  st = warp_stat(lane < W ? stats[lane] : Stat{-INFINITY, 0.0f, 0.0f});
  const RowEnd end(st);
  if (tid == 0 && out.entropy) out.entropy[t] = end.entropy;
  if (out.logprobs)
    for (int g = warp; g < out.G; g += W) {
      const int32_t tok = out.tokens[t * out.G + g];
      float r = 0.0f;
      if (tok >= 0 && tok < p.V) {
        const int acc = warp_dot(j.x + t * j.ldx, j.w + tok * j.ldw, j.K, lane);
        r = end.logp(__fmul_rn(__int2float_rn(acc), __fmul_rn(sx, p.sw[tok])));
      } else if (tok != -1) {
        r = __int_as_float(0x7fffffff);
        if (lane == 0) atomicOr(out.status, DEV_ERR_BOUNDS);
      }
      if (lane == 0) out.logprobs[t * out.G + g] = r;
    }
  if (p.k == 0) return;

  lists[warp][lane] = warp_sort_desc(best, lane);
  __syncthreads();
  const key_t merged = block_merge_lists(lists, LISTS, warp, lane);
  if (warp == 0 && lane == p.k - 1) bound_s = key_max(merged, (key_t)1);
  __syncthreads();
  const key_t bound = bound_s;
  if (best >= bound) {
    // (k at the most; a launch that gave up on a wait leaves whatever was there)
    const int n = min(p.part_n[(int64_t)tid * p.Tp + t], p.k);
    for (int e = 0; e < n; ++e) {
      const int64_t at = ((int64_t)tid * p.k + e) * p.Tp + t;
      const key_t key = order_key(p.part_v[at], (uint32_t)p.part_i[at]);
      if (key >= bound) {
        const int to = atomicAdd(&count, 1);
        if (to < I8_MAX_TOP * I8_MAX_TOP) cand[to] = key;
      }
    }
  }
  __syncthreads();
  const int n = min(count, I8_MAX_TOP * I8_MAX_TOP);
  key_t list = 0;
  for (int i = 32 * warp; i < n; i += TH)
    list = warp_merge_desc(list, warp_sort_desc(i + lane < n ? cand[i + lane] : (key_t)0, lane), lane);
  for (int i = W * 32 + tid; i < LISTS * 32; i += TH) (&lists[0][0])[i] = 0;
  lists[warp][lane] = list;
  __syncthreads();
  best = block_merge_lists(lists, LISTS, warp, lane);
  if (warp != 0) return;
  int id = best ? (int)(0xffffffffu - (uint32_t)best) : -1;
  const float lp = best ? end.logp(order_value((uint32_t)(best >> 32))) : -INFINITY;
  // Places left go to -inf logits, then to NaN, each by id.  A logit is neither
  // unless its scale is NaN, or so large that the product may overflow.
  int have = __popc(__ballot_sync(0xffffffffu, best != 0));
  for (int pass = sx == sx ? 0 : 1; pass < 2 && have < p.k; ++pass)
    for (int64_t v = lane; have < p.k && v - lane < p.V; v += 32) {
      const float s = v < p.V ? __fmul_rn(sx, p.sw[v]) : 0.0f;
      uint32_t odd = __ballot_sync(0xffffffffu, !(fabsf(s) < 1e28f));
      for (; odd && have < p.k; odd &= odd - 1) {
        const int b = __ffs(odd) - 1;
        const float sb = __shfl_sync(0xffffffffu, s, b);
        const int64_t vb = v - lane + b;
        float x = sb;
        if (sb == sb) x = __fmul_rn(__int2float_rn(warp_dot(j.x + t * j.ldx, j.w + vb * j.ldw, j.K, lane)), sb);
        if (pass == 0 ? x == -INFINITY : x != x) {
          if (lane == have) id = (int)vb;
          ++have;
        }
      }
    }
  if (lane < p.k) {
    const int64_t o = t * p.k + lane;
    if (out.top_ids) out.top_ids[o] = id;
    if (out.top_logprobs) out.top_logprobs[o] = end.s != end.s ? end.s : lp;
  }
}

// ---- host ---------------------------------------------------------------------------

// Token tiles at a time: the number that takes the fewest steps of a tile,
// more of them (fewer parts) for equal steps.
static HeadPlan head_plan(int64_t T, int64_t V, int sms) {
  HeadPlan h = {};
  const int slots = sms / 2;
  h.tt = (int)((T + H_TILE - 1) / H_TILE);
  h.vt = (int)((V + H_TILE - 1) / H_TILE);
  h.Tp = (int64_t)h.tt * H_TILE;
  double best = 0;
  for (int g = std::min(h.tt, slots); g >= 1; --g) {
    const int C = std::min({h.vt, slots / g, H_JOIN_MOST / 2}), passes = (h.tt + g - 1) / g;
    const double cost = passes * ((h.vt + C - 1) / C + 0.5);
    if (!h.g || cost < best) best = cost, h.g = g, h.C = C;
  }
  return h;
}

static size_t up(size_t n) { return (n + 255) & ~(size_t)255; }

// Places of the launch's arrays in a workspace; `base` null: its size.
static size_t head_layout(const HeadPlan &h, int64_t T, int64_t K, int k, uint8_t *base, HeadParams &p, int8_t *&q,
                          float *&sx) {
  size_t n = 0;
  auto take = [&](size_t bytes) {
    uint8_t *at = base + n;
    n += up(bytes);
    return at;
  };
  const size_t cells = (size_t)h.parts() * (size_t)h.Tp;
  sx = (float *)take(sizeof(float) * (size_t)T);
  q = (int8_t *)take((size_t)T * (size_t)((K + 15) / 16 * 16));
  p.part_r = (float *)take(sizeof(float) * cells);
  p.part_s = (float *)take(sizeof(float) * cells);
  p.part_t = (float *)take(sizeof(float) * cells);
  if (k > 0) {
    p.part_best = (key_t *)take(sizeof(key_t) * cells);
    p.part_n = (int32_t *)take(sizeof(int32_t) * cells);
    p.part_v = (float *)take(sizeof(float) * cells * (size_t)k);
    p.part_i = (int32_t *)take(sizeof(int32_t) * cells * (size_t)k);
    p.best2 = (uint64_t *)take(sizeof(uint64_t) * cells);
  }
  return n;
}

// All tokens, in launches of equal size of at most H_TOKENS.
static int64_t head_chunk(int64_t T) {
  const int64_t n = (T + H_TOKENS - 1) / H_TOKENS, c = (T + n - 1) / n;
  return n == 1 ? T : (c + H_TILE - 1) / H_TILE * H_TILE;
}

// Whether the logits go through memory.  A product and a walk do for up to 64
// tokens, of which a tile of 256 makes little (64 x 131,072 x 4,096: 110 us against
// 118), and where the lists that every part of a row keeps cost more than the
// logits' way: that grows with the alternatives.  For 256 x 131,072 x 2,048 the
// walk takes 110 to 115 us, this kernel 72, 100, 101, 106 and 135 with 0, 1, 5, 8 and
// 20 of them; for 203 x 50,021 x 1,999 58 to 61, and 50, 67, 72 (5) and 99 (20);
// for 768 x 131,072 x 2,048 252 (8), 254 (20) and 262 (32), and 188, 234 and 322.
// The threshold rests on these shapes: the product, which both ways share, grows
// with K and the lists do not, so it is off where K is much larger or smaller.
static bool head_walks(int64_t T, int64_t V, int k) {
  return T <= H_WALK_TOKENS || T * V * (int64_t)sizeof(float) <= (k ? std::max(k, 8) : 1) * H_WALK_BYTES;
}

// Their places then: scales, q, logits.
static size_t walk_layout(int64_t T, int64_t V, int64_t K, uint8_t *base, int8_t *&q, float *&sx, float *&logits) {
  sx = (float *)base;
  q = (int8_t *)(base + up(sizeof(float) * (size_t)T));
  const size_t before = up(sizeof(float) * (size_t)T) + up((size_t)T * (size_t)((K + 15) / 16 * 16));
  logits = (float *)(base + before);
  return before + sizeof(float) * (size_t)T * (size_t)((V + 3) / 4 * 4);
}

size_t head_workspace_bytes(const har_cuda_i8_weights *w, int64_t T, int k) {
  HeadParams p = {};
  int8_t *q;
  float *sx, *logits;
  if (head_walks(T, w->N, k)) return walk_layout(T, w->N, w->K, nullptr, q, sx, logits);
  const int64_t c = head_chunk(T), rest = T % c;
  const size_t most = head_layout(head_plan(c, w->N, w->sms), c, w->K, k, nullptr, p, q, sx);
  // the last launch is shorter, but its plan may have more parts
  return rest ? std::max(most, head_layout(head_plan(rest, w->N, w->sms), rest, w->K, k, nullptr, p, q, sx)) : most;
}

static int32_t head_walk(har_cuda_ctx *ctx, const har_cuda_i8_weights *w, const void *x, int32_t x_dtype, int64_t ldx,
                         int64_t T, const LogprobOut &out, uint8_t *workspace) {
  int8_t *q;
  float *sx, *logits;
  walk_layout(T, w->N, w->K, workspace, q, sx, logits);
  const int64_t ldq = (w->K + 15) / 16 * 16, ldl = (w->N + 3) / 4 * 4;
  int32_t st;
  if (i8_gemv_takes(T, w->N, w->K)) {
    st = launch_i8_gemv(ctx, w, x, x_dtype, ldx, nullptr, T, logits, HAR_CUDA_DTYPE_F32, ldl);
  } else {
    st = launch_i8_quantize(ctx, x, x_dtype, T, w->K, ldx, q, ldq, sx);
    if (st == HAR_CUDA_OK) st = launch_i8_matmul(ctx, w, q, ldq, sx, T, logits, HAR_CUDA_DTYPE_F32, ldl, true);
  }
  return st != HAR_CUDA_OK ? st : launch_token_logprobs(ctx, logits, HAR_CUDA_DTYPE_F32, T, w->N, ldl, out);
}

int32_t launch_i8_head(har_cuda_ctx *ctx, const har_cuda_i8_weights *w, const void *x, int32_t x_dtype, int64_t ldx,
                       int64_t T, const LogprobOut &out, uint8_t *workspace) {
  if (head_walks(T, w->N, out.k)) return head_walk(ctx, w, x, x_dtype, ldx, T, out, workspace);
  const int k = out.top_ids || out.top_logprobs ? out.k : 0;
  const int64_t chunk = head_chunk(T), ldq = (w->K + 15) / 16 * 16;
  for (int64_t t0 = 0; t0 < T; t0 += chunk) {
    const int64_t n = std::min(chunk, T - t0);
    const HeadPlan h = head_plan(n, w->N, w->sms);
    HeadJoin j = {};
    HeadParams &p = j.p;
    int8_t *q;
    float *sx;
    head_layout(h, n, w->K, k, workspace, p, q, sx);
    const uint8_t *xs = (const uint8_t *)x + (size_t)(t0 * ldx) * dtype_bytes(x_dtype);
    int32_t st = launch_i8_quantize(ctx, xs, x_dtype, n, w->K, ldx, q, ldq, sx);
    if (st != HAR_CUDA_OK) return st;
    p.sh.K = w->K, p.sh.k0 = 0, p.sh.k1 = ksteps_of(w->K);
    p.sh.bn = H_TILE;
    const int cap = k > H_LONG ? H_CAP_LONG : H_CAP;
    p.sh.stages = k > H_LONG ? H_SLOTS_LONG : H_SLOTS;
    // early cuts pay: a list is cut at twice its length, and not before 8 new
    p.full = std::min(cap - 8, std::max(2 * k, k + 8));
    p.T = n, p.V = w->N, p.Tp = h.Tp, p.sx = sx, p.sw = w->scale;
    p.tt = h.tt, p.vt = h.vt, p.g = h.g, p.C = h.C, p.k = k, p.status = ctx->d_status;
    TmaDesc map_x;
    st = encode_tmap_2d(ctx, &map_x, q, 1, (uint64_t)n, (uint64_t)w->K, (uint64_t)ldq, G_A, G_KS, true);
    if (st != HAR_CUDA_OK) return st;
    if (k > 0 && cudaMemsetAsync(p.best2, 0, sizeof(uint64_t) * (size_t)h.parts() * (size_t)h.Tp, ctx->stream) != cudaSuccess)
      return set_error(ctx, HAR_CUDA_ERR_CUDA, std::string("i8_head_logprobs: ") + cudaGetErrorString(cudaGetLastError()));
    prof_begin(ctx);
    const cudaError_t e = launch_clusters(i8_head_kernel, (unsigned)h.blocks(), G_THREADS, H_SMEM, ctx->stream, 2, map_x, w->map, p);
    st = check_launch(ctx, "i8_head_kernel");
    if (e != cudaSuccess)
      return set_error(ctx, HAR_CUDA_ERR_CUDA, std::string("i8_head_kernel: ") + cudaGetErrorString(e));
    if (st != HAR_CUDA_OK) return st;
    j.out = out;
    if (j.out.tokens) j.out.tokens += t0 * out.G;
    if (j.out.logprobs) j.out.logprobs += t0 * out.G;
    if (j.out.entropy) j.out.entropy += t0;
    if (j.out.top_ids) j.out.top_ids += t0 * out.k;
    if (j.out.top_logprobs) j.out.top_logprobs += t0 * out.k;
    j.x = q, j.w = w->q, j.ldx = ldq, j.ldw = w->ldq, j.K = w->K, j.parts = h.parts();
    prof_begin(ctx);
    if (j.parts <= H_JOIN) head_join_kernel<H_JOIN><<<(unsigned)n, H_JOIN, 0, ctx->stream>>>(j);
    else head_join_kernel<H_JOIN_MOST><<<(unsigned)n, H_JOIN_MOST, 0, ctx->stream>>>(j);
    st = check_launch(ctx, "head_join_kernel");
    if (st != HAR_CUDA_OK) return st;
  }
  return HAR_CUDA_OK;
}

}  // namespace har
