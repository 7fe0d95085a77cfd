// Entry points of the fp8 operators (include/moestream.h): argument checks
// and launches. Nothing here allocates or synchronises, but for ms_fp8_status,
// which waits for a stream and keeps a few pinned words, and nothing throws.
#include <cstdarg>
#include <cstdio>
#include <mutex>

#include "../../include/moestream.h"
#include "fp8.cuh"
#include "host_wait.h"

namespace ms {
void set_error_message(const char* msg);
}
using namespace ms;

namespace {

int __attribute__((format(printf, 2, 3))) bad(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  set_error_message(buf);
  return code;
}

// Makes `device` current for a call and the caller's device current again.
struct OnDevice {
  int before = -1, dev;
  cudaError_t err;
  explicit OnDevice(int d) : dev(d) {
    err = cudaGetDevice(&before);
    if (err == cudaSuccess && before != dev) err = cudaSetDevice(dev);
  }
  ~OnDevice() {
    if (before >= 0 && before != dev) cudaSetDevice(before);
  }
};

int sm_count(int device) {
  static int known[64] = {};
  if (device < 0 || device >= 64) return 148;
  if (!known[device] &&
      cudaDeviceGetAttribute(&known[device], cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
    return 148;
  return known[device];
}

bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }
int blocks(int n) { return (n + FP8_BLOCK - 1) / FP8_BLOCK; }

int launched(const char* what, cudaError_t e) {
  if (e == cudaSuccess) return MS_OK;
  return bad(MS_E_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
}

}  // namespace

extern "C" int ms_rms_norm_fp8(const ms_fp8_norm* p, void* stream) {
  const char* me = "ms_rms_norm_fp8";
  if (!p) return bad(MS_E_INVALID, "%s: the argument block is NULL", me);
  if (p->T < 0 || p->T > MS_FP8_MAX_ROWS) return bad(MS_E_INVALID, "%s: T must be in [0, %d]", me, MS_FP8_MAX_ROWS);
  if (p->T == 0) return MS_OK;
  if (!p->x || !p->q || !p->scales) return bad(MS_E_INVALID, "%s: x, q or scales is NULL", me);
  if (p->d < 1 || p->d > MS_FP8_MAX_FEATURES)
    return bad(MS_E_INVALID, "%s: d must be in [1, %d]", me, MS_FP8_MAX_FEATURES);
  if (p->dtype < MS_DT_BF16 || p->dtype > MS_DT_F32) return bad(MS_E_INVALID, "%s: unknown dtype %d", me, p->dtype);
  if (!p->weight && (p->residual || p->h || p->y))
    return bad(MS_E_INVALID, "%s: residual, h and y need a weight", me);
  if (p->residual && !p->h) return bad(MS_E_INVALID, "%s: a residual needs h", me);
  if (p->weight && !(p->eps >= 0.0)) return bad(MS_E_INVALID, "%s: eps must not be negative", me);
  if (p->q_stride < p->d) return bad(MS_E_INVALID, "%s: q_stride is smaller than a row", me);
  if ((p->h && p->h_stride < p->d) || (p->y && p->y_stride < p->d))
    return bad(MS_E_INVALID, "%s: h_stride or y_stride is smaller than a row", me);
  OnDevice on(p->device);
  if (on.err != cudaSuccess) return bad(MS_E_CUDA, "%s: device %d: %s", me, p->device, cudaGetErrorString(on.err));
  NormArgs a{};
  a.x = p->x, a.res = p->residual, a.w = p->weight, a.h = p->h, a.y = p->y;
  a.q = static_cast<uint8_t*>(p->q), a.s = p->scales;
  a.x_stride = p->x_stride, a.res_stride = p->residual_stride, a.h_stride = p->h_stride;
  a.y_stride = p->y_stride, a.q_stride = p->q_stride;
  a.T = p->T, a.d = p->d, a.eps = p->eps;
  return launched(me, launch_norm_fp8(a, p->dtype, sm_count(p->device), static_cast<cudaStream_t>(stream)));
}

extern "C" int ms_linear_fp8(const ms_fp8_linear* p, void* stream) {
  const char* me = "ms_linear_fp8";
  if (!p) return bad(MS_E_INVALID, "%s: the argument block is NULL", me);
  if (p->M < 0 || p->M > MS_FP8_MAX_ROWS) return bad(MS_E_INVALID, "%s: M must be in [0, %d]", me, MS_FP8_MAX_ROWS);
  if (p->M == 0) return MS_OK;
  if (!p->x || !p->x_scales || !p->w || !p->w_scales || !p->y)
    return bad(MS_E_INVALID, "%s: x, w, their scales or y is NULL", me);
  if (p->N < 1 || p->K < 1 || p->N > MS_FP8_MAX_ROWS || p->K > MS_FP8_MAX_ROWS)
    return bad(MS_E_INVALID, "%s: N and K must be in [1, %d]", me, MS_FP8_MAX_ROWS);
  if (p->out_dtype < MS_DT_BF16 || p->out_dtype > MS_DT_F32)
    return bad(MS_E_INVALID, "%s: unknown out_dtype %d", me, p->out_dtype);
  if (off16(p->x) || off16(p->w) || p->x_stride % 16 || p->w_stride % 16)
    return bad(MS_E_INVALID, "%s: the rows of x and w must start on 16-byte boundaries", me);
  if (p->x_stride < p->K || p->w_stride < p->K || p->y_stride < p->N || p->x_scales_stride < blocks(p->K))
    return bad(MS_E_INVALID, "%s: a stride is smaller than a row", me);
  OnDevice on(p->device);
  if (on.err != cudaSuccess) return bad(MS_E_CUDA, "%s: device %d: %s", me, p->device, cudaGetErrorString(on.err));
  LinearArgs a{};
  a.x = static_cast<const uint8_t*>(p->x), a.xs = p->x_scales;
  a.w = static_cast<const uint8_t*>(p->w), a.ws = p->w_scales;
  a.bias = p->bias, a.y = p->y;
  a.x_stride = p->x_stride, a.xs_stride = p->x_scales_stride, a.w_stride = p->w_stride, a.y_stride = p->y_stride;
  a.M = p->M, a.N = p->N, a.K = p->K;
  return launched(me, launch_linear_fp8(a, p->out_dtype, sm_count(p->device), static_cast<cudaStream_t>(stream)));
}

static int check_moe(const char* me, const ms_fp8_moe* p) {
  if (!p) return bad(MS_E_INVALID, "%s: the argument block is NULL", me);
  if (p->model != MS_MODEL_QWEN3 && p->model != MS_MODEL_GPTOSS)
    return bad(MS_E_INVALID, "%s: unknown model %d", me, p->model);
  if (p->T < 0 || p->T > MS_FP8_MAX_TOKENS)
    return bad(MS_E_INVALID, "%s: T must be in [0, %d]", me, MS_FP8_MAX_TOKENS);
  if (p->n_experts < 1 || p->n_experts > 256) return bad(MS_E_INVALID, "%s: n_experts must be in [1, 256]", me);
  if (p->top_k < 1 || p->top_k > 32 || p->top_k > p->n_experts)
    return bad(MS_E_INVALID, "%s: top_k must be in [1, min(32, n_experts)]", me);
  if (p->d_model < 16 || p->d_model % 16 || p->d_model > MS_FP8_MAX_FEATURES || p->d_ff < 16 || p->d_ff % 16 ||
      p->d_ff > MS_FP8_MAX_FEATURES)
    return bad(MS_E_INVALID, "%s: d_model and d_ff must be multiples of 16 in [16, %d]", me, MS_FP8_MAX_FEATURES);
  return MS_OK;
}

extern "C" int ms_moe_fp8_workspace(const ms_fp8_moe* p, size_t* bytes) {
  const char* me = "ms_moe_fp8_workspace";
  const int rc = check_moe(me, p);
  if (rc) return rc;
  if (!bytes) return bad(MS_E_INVALID, "%s: bytes is NULL", me);
  *bytes = moe_fp8_workspace(p->T, p->d_model, p->d_ff, p->n_experts, p->top_k);
  return MS_OK;
}

namespace {
using MoeLaunch = cudaError_t (*)(const MoeFp8Args&, int, cudaStream_t);

int moe_call(const char* me, const ms_fp8_moe* p, void* stream, MoeLaunch launch) {
  const int rc = check_moe(me, p);
  if (rc) return rc;
  if (p->T == 0) return MS_OK;
  if (!p->x || !p->router || !p->y || !p->workspace)
    return bad(MS_E_INVALID, "%s: x, router, y or workspace is NULL", me);
  for (int i = 0; i < 3; ++i) {
    if (!p->codes[i] || !p->scales[i]) return bad(MS_E_INVALID, "%s: codes or scales [%d] is NULL", me, i);
    if (off16(p->codes[i])) return bad(MS_E_INVALID, "%s: codes[%d] is not 16-byte aligned", me, i);
  }
  if (off16(p->x) || off16(p->router) || off16(p->y) || off16(p->workspace) || off16(p->residual))
    return bad(MS_E_INVALID, "%s: x, router, residual, y and workspace must be 16-byte aligned", me);
  if (p->workspace_bytes < moe_fp8_workspace(p->T, p->d_model, p->d_ff, p->n_experts, p->top_k))
    return bad(MS_E_INVALID, "%s: the workspace is too small (ms_moe_fp8_workspace)", me);
  OnDevice on(p->device);
  if (on.err != cudaSuccess) return bad(MS_E_CUDA, "%s: device %d: %s", me, p->device, cudaGetErrorString(on.err));
  MoeFp8Args a{};
  a.x = static_cast<const uint16_t*>(p->x), a.router = static_cast<const uint16_t*>(p->router);
  a.router_bias = p->router_bias;
  Fp8Matrix* m[3] = {&a.gate, &a.up, &a.down};
  for (int i = 0; i < 3; ++i)
    m[i]->q = static_cast<const uint8_t*>(p->codes[i]), m[i]->s = p->scales[i], m[i]->bias = p->bias[i];
  a.res = static_cast<const uint16_t*>(p->residual), a.y = static_cast<uint16_t*>(p->y);
  a.ws = static_cast<uint8_t*>(p->workspace);
  a.model = p->model, a.T = p->T, a.d = p->d_model, a.f = p->d_ff, a.E = p->n_experts, a.k = p->top_k;
  a.norm_topk = p->norm_topk_prob;
  return launched(me, launch(a, sm_count(p->device), static_cast<cudaStream_t>(stream)));
}
}  // namespace

extern "C" int ms_moe_fp8_layer(const ms_fp8_moe* p, void* stream) {
  return moe_call("ms_moe_fp8_layer", p, stream, launch_moe_fp8);
}

extern "C" int ms_fp8_selftest_wait(const ms_fp8_moe* p, void* stream) {
  const char* me = "ms_fp8_selftest_wait";
  const int rc = check_moe(me, p);
  if (rc) return rc;
  if (p->T <= MOE_FP8_ROUTED_HERE)
    return bad(MS_E_INVALID, "%s: T must be above %d (fewer tokens are routed without a wait)", me, MOE_FP8_ROUTED_HERE);
  return moe_call(me, p, stream, launch_moe_fp8_lost);
}

namespace {

// Reads and clears both words in one step each: what a kernel on another
// stream records is either in this answer or left for the next.
__global__ void k_take_status(int* linear, int* moe, volatile int* answer) {
  answer[0] = atomicExch(linear, 0);
  answer[1] = atomicExch(moe, 0);
}

// Pinned words for an answer, mapped on every device: two ints, and while they
// are not in use the next free ones. They are kept from call to call (freeing
// them would wait for the device), as many as calls were ever under way at once;
// those of a call that gave up waiting are not used again, as its kernel may
// yet write them.
struct Answer {
  int st[2];
  Answer* next;
};
std::mutex g_answers_mutex;
Answer* g_answers = nullptr;

// What this thread does is no part of a capture, another thread's included: that
// one stays whole though this one allocates or loads a kernel meanwhile.
struct BesideCaptures {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  BesideCaptures() { cudaThreadExchangeStreamCaptureMode(&mode); }
  ~BesideCaptures() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

Answer* take_answer() {
  {
    std::lock_guard<std::mutex> lock(g_answers_mutex);
    if (Answer* a = g_answers) {
      g_answers = a->next;
      return a;
    }
  }
  void* p = nullptr;
  if (cudaHostAlloc(&p, sizeof(Answer), cudaHostAllocPortable | cudaHostAllocMapped) == cudaSuccess)
    return static_cast<Answer*>(p);
  cudaGetLastError();
  return nullptr;
}
void give_answer(Answer* a) {
  std::lock_guard<std::mutex> lock(g_answers_mutex);
  a->next = g_answers;
  g_answers = a;
}

}  // namespace

extern "C" int ms_fp8_status(int device, int* status, void* stream) {
  const char* me = "ms_fp8_status";
  if (!status) return bad(MS_E_INVALID, "%s: status is NULL", me);
  *status = MS_OK;
  OnDevice on(device);
  if (on.err != cudaSuccess) return bad(MS_E_CUDA, "%s: device %d: %s", me, device, cudaGetErrorString(on.err));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaStreamCaptureStatus capturing;
  cudaError_t e = cudaStreamIsCapturing(s, &capturing);
  if (e != cudaSuccess || capturing != cudaStreamCaptureStatusNone)
    return bad(MS_E_INVALID, "%s: not for use in a capture", me);
  BesideCaptures beside;
  int* at[2] = {};
  if (linear_fp8_status(&at[0]) != cudaSuccess || moe_fp8_status(&at[1]) != cudaSuccess)
    return bad(MS_E_CUDA, "%s: the status words have no address", me);
  // The stream's work first: while it has not finished, nothing is taken.
  e = stream_wait_bounded(s);
  int st[2] = {};
  if (e == cudaSuccess) {
    Answer* answer = take_answer();
    if (!answer) return bad(MS_E_CUDA, "%s: no pinned memory for the answer", me);
    k_take_status<<<1, 1, 0, s>>>(at[0], at[1], answer->st);
    e = cudaGetLastError();
    const bool asked = e == cudaSuccess;
    if (asked) e = stream_wait_bounded(s);
    if (e == cudaSuccess) {
      const volatile int* v = answer->st;
      st[0] = v[0], st[1] = v[1];
    }
    if (e == cudaSuccess || !asked) give_answer(answer);
  }
  if (e == cudaErrorTimeout)
    return bad(MS_E_TIMEOUT, "%s: the stream did not finish within the host wait limit (MS_HOST_WAIT_S)", me);
  if (e != cudaSuccess) return bad(MS_E_CUDA, "%s: %s", me, cudaGetErrorString(e));
  *status = st[0] ? st[0] : st[1];
  return *status == MS_OK ? MS_OK : bad(*status, "an fp8 operator's bounded wait ran out: its output is not valid");
}
