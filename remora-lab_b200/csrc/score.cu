// score.cu — C ABI entry points of the 8-bit integer products and the
// log-probability operators (declared in include/har_cuda.h): argument checks,
// weight handles, workspaces.  Kernels: k_i8_*.cu, k_logprobs.cu.
#include <new>

#include "score.cuh"

namespace har {

// The context's device for the length of a call; the caller's current device
// is restored.
struct OnDevice {
  int before = -1;
  cudaError_t err;
  explicit OnDevice(const har_cuda_ctx *ctx) {
    err = cudaGetDevice(&before);
    if (err == cudaSuccess && before != ctx->device) err = cudaSetDevice(ctx->device);
    else if (err == cudaSuccess) before = -1;
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
  int32_t status(har_cuda_ctx *ctx) const {
    return err == cudaSuccess ? HAR_CUDA_OK
                              : set_error(ctx, HAR_CUDA_ERR_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(err));
  }
};

static size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }

static int32_t check_dtype(har_cuda_ctx *ctx, int32_t dtype, const char *who) {
  if (dtype == HAR_CUDA_DTYPE_F32 || dtype == HAR_CUDA_DTYPE_F16 || dtype == HAR_CUDA_DTYPE_BF16) return HAR_CUDA_OK;
  return set_error(ctx, HAR_CUDA_ERR_ARG, std::string(who) + ": unknown element type " + std::to_string(dtype));
}

// A matrix of `rows` rows of `cols` elements: not null, aligned to its
// elements, rows ld apart.  Inputs may overlap (ld 0 repeats a row), outputs not.
static int32_t check_rows(har_cuda_ctx *ctx, const void *p, size_t elem, int64_t rows, int64_t cols, int64_t ld,
                          bool output, const std::string &who) {
  if (!p) return set_error(ctx, HAR_CUDA_ERR_ARG, who + " is null");
  if ((uintptr_t)p & (elem - 1)) return set_error(ctx, HAR_CUDA_ERR_ARG, who + " is not aligned to its elements");
  if (rows > 1 && (ld < 0 || (output && ld < cols)))
    return set_error(ctx, HAR_CUDA_ERR_GEOMETRY, who + ": rows of " + std::to_string(cols) + " elements cannot lie " +
                                                     std::to_string(ld) + " apart");
  return HAR_CUDA_OK;
}

static int32_t check_i8_rows(har_cuda_ctx *ctx, const int8_t *q, int64_t rows, int64_t K, int64_t ldq,
                             const std::string &who) {
  if (!q) return set_error(ctx, HAR_CUDA_ERR_ARG, who + " is null");
  if (((uintptr_t)q & 15u) || (rows > 1 && (ldq & 15)))
    return set_error(ctx, HAR_CUDA_ERR_ARG, who + ": rows must start at multiples of 16 bytes");
  if (rows > 1 && ldq < K)
    return set_error(ctx, HAR_CUDA_ERR_GEOMETRY, who + ": rows overlap");
  return HAR_CUDA_OK;
}

static int32_t check_nk(har_cuda_ctx *ctx, int64_t N, int64_t K, const char *who) {
  if (N < 1 || N > I8_MAX_ROWS || K < 1 || K > I8_MAX_K)
    return set_error(ctx, HAR_CUDA_ERR_GEOMETRY, std::string(who) + ": need 1 <= N <= 2^30 and 1 <= K <= " +
                                                     std::to_string(I8_MAX_K));
  return HAR_CUDA_OK;
}

static int32_t check_i8_weights(har_cuda_ctx *ctx, const har_cuda_i8_weights *w, const char *who) {
  if (!w) return set_error(ctx, HAR_CUDA_ERR_ARG, std::string(who) + ": weights are null");
  if (w->device != ctx->device)
    return set_error(ctx, HAR_CUDA_ERR_ARG, std::string(who) + ": weights live on another device");
  return HAR_CUDA_OK;
}

// Whether the context's stream is being captured.
static int32_t capturing(har_cuda_ctx *ctx, const char *who, bool *yes) {
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  const cudaError_t e = cudaStreamIsCapturing(ctx->stream, &cap);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(ctx, HAR_CUDA_ERR_CUDA, std::string(who) + ": " + cudaGetErrorString(e));
  }
  *yes = cap != cudaStreamCaptureStatusNone;
  return HAR_CUDA_OK;
}

// A stream that lasts as long as the context.  Any other may be destroyed
// before the context is bound to the next, so its handle is not used then.
static bool lasting(const har_cuda_ctx *ctx, cudaStream_t s) { return s == ctx->own_stream || s == cudaStreamLegacy; }

void free_workspace(har_cuda_ctx *ctx) {
  har_cuda_ctx::Workspace &a = ctx->ws;
  if (a.p) {
    if (lasting(ctx, a.stream)) cudaStreamSynchronize(a.stream);
    else cudaEventSynchronize(a.used);
    cudaFree(a.p);
  }
  if (a.used) cudaEventDestroy(a.used);
  a = {};
}

// The workspace of one call: the caller's, or outside a capture the context's.
// The context's is used in order by the streams that the context is bound to one
// after the other: a call on another stream than the last use's waits for that
// use on the device.  What it waits for is an event: recorded behind the use
// where the stream may be gone later, and otherwise only once another stream
// comes, so that calls on one lasting stream (torch's default one) pay nothing.
class CallWorkspace {
 public:
  uint8_t *p = nullptr;

  explicit CallWorkspace(har_cuda_ctx *ctx) : ctx_(ctx) {}
  ~CallWorkspace() {
    if (!shared_) return;
    har_cuda_ctx::Workspace &a = ctx_->ws;
    a.stream = ctx_->stream;
    a.stream_id = id_;
    if (!lasting(ctx_, a.stream)) cudaEventRecord(a.used, a.stream);
  }
  CallWorkspace(const CallWorkspace &) = delete;
  CallWorkspace &operator=(const CallWorkspace &) = delete;

  int32_t take(void *given, size_t bytes, size_t need, const char *who) {
    if (need == 0) return HAR_CUDA_OK;
    if (given) {
      if (((uintptr_t)given & 15u) || bytes < need)
        return set_error(ctx_, HAR_CUDA_ERR_ARG, std::string(who) + ": the workspace must be 16-byte aligned and hold " +
                                                     std::to_string(need) + " bytes, got " + std::to_string(bytes));
      p = (uint8_t *)given;
      return HAR_CUDA_OK;
    }
    bool captured = false;
    const int32_t st = capturing(ctx_, who, &captured);
    if (st != HAR_CUDA_OK) return st;
    if (captured)
      return set_error(ctx_, HAR_CUDA_ERR_ARG, std::string(who) + ": a captured call needs a workspace of " +
                                                   std::to_string(need) + " bytes from the caller");
    har_cuda_ctx::Workspace &a = ctx_->ws;
    cudaError_t e = cudaStreamGetId(ctx_->stream, &id_);
    if (e == cudaSuccess && need > a.bytes) {
      free_workspace(ctx_);
      const size_t sz = (need + (1u << 20) - 1) & ~((size_t)(1u << 20) - 1);
      if (cudaMalloc(&a.p, sz) != cudaSuccess) {
        cudaGetLastError();
        a.p = nullptr;
        return set_error(ctx_, HAR_CUDA_ERR_OOM, std::string(who) + ": a workspace of " + std::to_string(sz) + " bytes failed");
      }
      a.bytes = sz;
      a.stream = ctx_->own_stream;  // nobody uses it yet
      a.stream_id = id_;
      e = cudaEventCreateWithFlags(&a.used, cudaEventDisableTiming);
      if (e != cudaSuccess) free_workspace(ctx_);
    } else if (e == cudaSuccess && id_ != a.stream_id) {
      if (lasting(ctx_, a.stream)) e = cudaEventRecord(a.used, a.stream);
      if (e == cudaSuccess) e = cudaStreamWaitEvent(ctx_->stream, a.used, 0);
    }
    if (e != cudaSuccess) {
      cudaGetLastError();
      return set_error(ctx_, HAR_CUDA_ERR_CUDA, std::string(who) + ": " + cudaGetErrorString(e));
    }
    p = (uint8_t *)a.p;
    shared_ = true;
    return HAR_CUDA_OK;
  }

 private:
  har_cuda_ctx *ctx_;
  unsigned long long id_ = 0;
  bool shared_ = false;
};

}  // namespace har

using namespace har;

#define HAR_TRY(expr)                       \
  do {                                      \
    int32_t _st = (expr);                   \
    if (_st != HAR_CUDA_OK) return _st;     \
  } while (0)

extern "C" {

int32_t har_cuda_i8_quantize(har_cuda_ctx *ctx, const void *x_dev, int32_t dtype, int64_t M,
                             int64_t K, int64_t ldx, int8_t *q_dev, int64_t ldq,
                             float *scale_dev) {
  if (!ctx) return HAR_CUDA_ERR_ARG;
  HAR_TRY(check_dtype(ctx, dtype, "i8_quantize"));
  if (M < 0 || M > I8_MAX_ROWS || K < 1 || K > I8_MAX_ROWS)
    return set_error(ctx, HAR_CUDA_ERR_GEOMETRY, "i8_quantize: need 0 <= M <= 2^30 and 1 <= K <= 2^30");
  if (M == 0) return HAR_CUDA_OK;
  HAR_TRY(check_rows(ctx, x_dev, dtype_bytes(dtype), M, K, ldx, false, "i8_quantize: x"));
  HAR_TRY(check_rows(ctx, q_dev, 1, M, K, ldq, true, "i8_quantize: q"));
  HAR_TRY(check_rows(ctx, scale_dev, 4, 1, M, M, true, "i8_quantize: scale"));
  OnDevice on(ctx);
  HAR_TRY(on.status(ctx));
  return launch_i8_quantize(ctx, x_dev, dtype, M, K, ldx, q_dev, ldq, scale_dev);
}

static int32_t finish_i8_weights(har_cuda_ctx *ctx, har_cuda_i8_weights *w, har_cuda_i8_weights **out) {
  const int32_t st = encode_tmap_2d(ctx, &w->map, w->q, 1, (uint64_t)w->N, (uint64_t)w->K, (uint64_t)w->ldq, 128, 128, true);
  if (st != HAR_CUDA_OK) {
    har_cuda_i8_weights_free(w);
    return st;
  }
  *out = w;
  return HAR_CUDA_OK;
}

int32_t har_cuda_i8_weights_quantize(har_cuda_ctx *ctx, const void *w_dev, int32_t dtype,
                                     int64_t N, int64_t K, int64_t ldw,
                                     har_cuda_i8_weights **out) {
  if (!ctx || !out) return HAR_CUDA_ERR_ARG;
  *out = nullptr;
  HAR_TRY(check_dtype(ctx, dtype, "i8_weights_quantize"));
  HAR_TRY(check_nk(ctx, N, K, "i8_weights_quantize"));
  HAR_TRY(check_rows(ctx, w_dev, dtype_bytes(dtype), N, K, ldw, false, "i8_weights_quantize: weights"));
  OnDevice on(ctx);
  HAR_TRY(on.status(ctx));
  bool captured = false;
  HAR_TRY(capturing(ctx, "i8_weights_quantize", &captured));
  if (captured)  // the handle's memory would be written by the graph, and not before its first launch
    return set_error(ctx, HAR_CUDA_ERR_ARG, "i8_weights_quantize: not while the stream is being captured");
  const int64_t ldq = (int64_t)round16((size_t)K);
  const size_t qb = (size_t)N * (size_t)ldq, bytes = qb + sizeof(float) * (size_t)N;
  void *d = nullptr;
  if (cudaMalloc(&d, bytes) != cudaSuccess) {
    cudaGetLastError();
    return set_error(ctx, HAR_CUDA_ERR_OOM, "i8_weights_quantize: cudaMalloc of " + std::to_string(bytes) + " bytes failed");
  }
  int32_t st = launch_i8_quantize(ctx, w_dev, dtype, N, K, ldw, (int8_t *)d, ldq, (float *)((uint8_t *)d + qb));
  // any context of the device may use the handle, on any stream: it is filled
  // before it is given out, as uploaded weights are
  if (st == HAR_CUDA_OK) {
    const cudaError_t e = cudaStreamSynchronize(ctx->stream);
    if (e != cudaSuccess) {
      cudaGetLastError();
      st = set_error(ctx, HAR_CUDA_ERR_CUDA, std::string("i8_weights_quantize: ") + cudaGetErrorString(e));
    }
  }
  if (st != HAR_CUDA_OK) {
    cudaFree(d);
    return st;
  }
  har_cuda_i8_weights *w = new (std::nothrow) har_cuda_i8_weights();
  if (!w) {
    cudaFree(d);
    return set_error(ctx, HAR_CUDA_ERR_OOM, "i8_weights_quantize: out of host memory");
  }
  w->q = (const int8_t *)d;
  w->scale = (const float *)((uint8_t *)d + qb);
  w->N = N, w->K = K, w->ldq = ldq, w->device = ctx->device, w->sms = ctx->num_sms, w->owned = true;
  return finish_i8_weights(ctx, w, out);
}

int32_t har_cuda_i8_weights_wrap(har_cuda_ctx *ctx, const int8_t *q_dev, int64_t ldq,
                                 const float *scale_dev, int64_t N, int64_t K,
                                 har_cuda_i8_weights **out) {
  if (!ctx || !out) return HAR_CUDA_ERR_ARG;
  *out = nullptr;
  HAR_TRY(check_nk(ctx, N, K, "i8_weights_wrap"));
  HAR_TRY(check_i8_rows(ctx, q_dev, N, K, ldq, "i8_weights_wrap: q"));
  HAR_TRY(check_rows(ctx, scale_dev, 4, 1, N, N, false, "i8_weights_wrap: scale"));
  har_cuda_i8_weights *w = new (std::nothrow) har_cuda_i8_weights();
  if (!w) return set_error(ctx, HAR_CUDA_ERR_OOM, "i8_weights_wrap: out of host memory");
  w->q = q_dev;
  w->scale = scale_dev;
  w->N = N, w->K = K, w->ldq = N == 1 ? (int64_t)round16((size_t)K) : ldq, w->device = ctx->device, w->sms = ctx->num_sms;
  return finish_i8_weights(ctx, w, out);
}

int32_t har_cuda_i8_weights_free(har_cuda_i8_weights *w) {
  if (!w) return HAR_CUDA_ERR_ARG;
  if (w->owned) {
    int before = -1;
    cudaGetDevice(&before);
    cudaSetDevice(w->device);
    cudaFree((void *)w->q);
    if (before >= 0) cudaSetDevice(before);
  }
  delete w;
  return HAR_CUDA_OK;
}

int32_t har_cuda_i8_matmul(har_cuda_ctx *ctx, const har_cuda_i8_weights *w, const int8_t *q_dev,
                           int64_t ldq, const float *scale_dev, int64_t M, void *y_dev,
                           int32_t y_dtype, int64_t ldy) {
  if (!ctx) return HAR_CUDA_ERR_ARG;
  HAR_TRY(check_i8_weights(ctx, w, "i8_matmul"));
  HAR_TRY(check_dtype(ctx, y_dtype, "i8_matmul"));
  if (M < 0 || M > I8_MAX_ROWS) return set_error(ctx, HAR_CUDA_ERR_GEOMETRY, "i8_matmul: need 0 <= M <= 2^30");
  if (M == 0) return HAR_CUDA_OK;
  HAR_TRY(check_i8_rows(ctx, q_dev, M, w->K, ldq, "i8_matmul: q"));
  HAR_TRY(check_rows(ctx, scale_dev, 4, 1, M, M, false, "i8_matmul: scale"));
  HAR_TRY(check_rows(ctx, y_dev, dtype_bytes(y_dtype), M, w->N, ldy, true, "i8_matmul: y"));
  OnDevice on(ctx);
  HAR_TRY(on.status(ctx));
  if (M == 1) ldq = (int64_t)round16((size_t)w->K), ldy = w->N;
  if (i8_gemv_takes(M, w->N, w->K)) return launch_i8_gemv(ctx, w, q_dev, 0, ldq, scale_dev, M, y_dev, y_dtype, ldy);
  return launch_i8_matmul(ctx, w, q_dev, ldq, scale_dev, M, y_dev, y_dtype, ldy);
}

// workspace of the quantised rows: scales, then q with 16-byte rows
static size_t quantized_bytes(const har_cuda_i8_weights *w, int64_t M) {
  return round16(sizeof(float) * (size_t)M) + (size_t)M * round16((size_t)w->K);
}

int64_t har_cuda_i8_linear_workspace(const har_cuda_i8_weights *w, int64_t M) {
  if (!w || M < 0 || M > I8_MAX_ROWS) return -1;
  return M == 0 || i8_gemv_takes(M, w->N, w->K) ? 0 : (int64_t)quantized_bytes(w, M);
}

int32_t har_cuda_i8_linear(har_cuda_ctx *ctx, const har_cuda_i8_weights *w, const void *x_dev,
                           int32_t x_dtype, int64_t ldx, int64_t M, void *y_dev, int32_t y_dtype,
                           int64_t ldy, void *workspace_dev, size_t workspace_bytes) {
  if (!ctx) return HAR_CUDA_ERR_ARG;
  HAR_TRY(check_i8_weights(ctx, w, "i8_linear"));
  HAR_TRY(check_dtype(ctx, x_dtype, "i8_linear"));
  HAR_TRY(check_dtype(ctx, y_dtype, "i8_linear"));
  if (M < 0 || M > I8_MAX_ROWS) return set_error(ctx, HAR_CUDA_ERR_GEOMETRY, "i8_linear: need 0 <= M <= 2^30");
  if (M == 0) return HAR_CUDA_OK;
  HAR_TRY(check_rows(ctx, x_dev, dtype_bytes(x_dtype), M, w->K, ldx, false, "i8_linear: x"));
  HAR_TRY(check_rows(ctx, y_dev, dtype_bytes(y_dtype), M, w->N, ldy, true, "i8_linear: y"));
  OnDevice on(ctx);
  HAR_TRY(on.status(ctx));
  if (M == 1) ldx = w->K, ldy = w->N;
  if (i8_gemv_takes(M, w->N, w->K)) return launch_i8_gemv(ctx, w, x_dev, x_dtype, ldx, nullptr, M, y_dev, y_dtype, ldy);
  CallWorkspace ws(ctx);
  HAR_TRY(ws.take(workspace_dev, workspace_bytes, quantized_bytes(w, M), "i8_linear"));
  float *scale = (float *)ws.p;
  int8_t *q = (int8_t *)ws.p + round16(sizeof(float) * (size_t)M);
  const int64_t ldq = (int64_t)round16((size_t)w->K);
  HAR_TRY(launch_i8_quantize(ctx, x_dev, x_dtype, M, w->K, ldx, q, ldq, scale));
  return launch_i8_matmul(ctx, w, q, ldq, scale, M, y_dev, y_dtype, ldy);
}

static int32_t check_logprobs(har_cuda_ctx *ctx, int64_t T, int64_t V, const LogprobOut &o, const char *name) {
  const std::string who(name);
  if (T < 0 || T > I8_MAX_ROWS || V < 1 || V > I8_MAX_ROWS)
    return set_error(ctx, HAR_CUDA_ERR_GEOMETRY, who + ": need 0 <= T <= 2^30 and 1 <= V <= 2^30");
  if (o.G < 0 || o.k < 0 || o.k > I8_MAX_TOP)
    return set_error(ctx, HAR_CUDA_ERR_GEOMETRY, who + ": need G >= 0 and 0 <= k <= " + std::to_string(I8_MAX_TOP));
  if (T == 0) return HAR_CUDA_OK;
  if (o.logprobs && o.G > 0) HAR_TRY(check_rows(ctx, o.tokens, 4, 1, 1, 1, false, who + ": tokens"));
  const void *outs[] = {o.logprobs, o.entropy, o.top_ids, o.top_logprobs};
  for (const void *p : outs)
    if ((uintptr_t)p & 3u) return set_error(ctx, HAR_CUDA_ERR_ARG, who + ": an output is not aligned to its elements");
  return HAR_CUDA_OK;
}

int32_t har_cuda_token_logprobs(har_cuda_ctx *ctx, const void *logits_dev, int32_t dtype, int64_t T,
                                int64_t V, int64_t ldl, const int32_t *tokens_dev, int32_t G,
                                int32_t k, float *logprobs_dev, float *entropy_dev,
                                int32_t *top_ids_dev, float *top_logprobs_dev) {
  if (!ctx) return HAR_CUDA_ERR_ARG;
  const LogprobOut o = {tokens_dev, G, k, logprobs_dev, entropy_dev, top_logprobs_dev, top_ids_dev, ctx->d_status};
  HAR_TRY(check_dtype(ctx, dtype, "token_logprobs"));
  HAR_TRY(check_logprobs(ctx, T, V, o, "token_logprobs"));
  if (T == 0) return HAR_CUDA_OK;
  HAR_TRY(check_rows(ctx, logits_dev, dtype_bytes(dtype), T, V, ldl, false, "token_logprobs: logits"));
  OnDevice on(ctx);
  HAR_TRY(on.status(ctx));
  return launch_token_logprobs(ctx, logits_dev, dtype, T, V, T == 1 ? V : ldl, o);
}

int64_t har_cuda_i8_head_workspace(const har_cuda_i8_weights *w, int64_t T, int32_t G, int32_t k) {
  if (!w || T < 0 || T > I8_MAX_ROWS || G < 0 || k < 0 || k > I8_MAX_TOP) return -1;
  return T == 0 ? 0 : (int64_t)head_workspace_bytes(w, T, k);
}

int32_t har_cuda_i8_head_logprobs(har_cuda_ctx *ctx, const har_cuda_i8_weights *w,
                                  const void *x_dev, int32_t x_dtype, int64_t ldx, int64_t T,
                                  const int32_t *tokens_dev, int32_t G, int32_t k,
                                  float *logprobs_dev, float *entropy_dev, int32_t *top_ids_dev,
                                  float *top_logprobs_dev, void *workspace_dev,
                                  size_t workspace_bytes) {
  if (!ctx) return HAR_CUDA_ERR_ARG;
  HAR_TRY(check_i8_weights(ctx, w, "i8_head_logprobs"));
  HAR_TRY(check_dtype(ctx, x_dtype, "i8_head_logprobs"));
  const LogprobOut o = {tokens_dev, G, k, logprobs_dev, entropy_dev, top_logprobs_dev, top_ids_dev, ctx->d_status};
  HAR_TRY(check_logprobs(ctx, T, w->N, o, "i8_head_logprobs"));
  if (T == 0) return HAR_CUDA_OK;
  HAR_TRY(check_rows(ctx, x_dev, dtype_bytes(x_dtype), T, w->K, ldx, false, "i8_head_logprobs: x"));
  OnDevice on(ctx);
  HAR_TRY(on.status(ctx));
  if (T == 1) ldx = w->K;
  CallWorkspace ws(ctx);
  HAR_TRY(ws.take(workspace_dev, workspace_bytes, head_workspace_bytes(w, T, k), "i8_head_logprobs"));
  return launch_i8_head(ctx, w, x_dev, x_dtype, ldx, T, o, ws.p);
}

}  // extern "C"
