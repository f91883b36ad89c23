// C ABI of the dense projection, the expert router and the mixture-of-experts layer
// (declarations in include/ffn_b200.h).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstring>
#include <new>

#include "../../include/ffn_b200.h"
#include "layers_simple.cuh"

namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t pitch_of(int64_t cols) { return (cols + 7) / 8 * 8; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool bad_rows(const void* p, int64_t ld, int64_t cols) { return !aligned16(p) || ld % 8 != 0 || ld < cols; }
constexpr int64_t kMaxDim = 65535;

// Makes `device` current for one call and puts the caller's device back.
struct DeviceScope {
  int before = -1;
  bool ok = true;
  explicit DeviceScope(int device) {
    int cur = 0;
    ok = cudaGetDevice(&cur) == cudaSuccess;
    if (ok && cur != device) {
      ok = cudaSetDevice(device) == cudaSuccess;
      if (ok) before = cur;
    }
  }
  ~DeviceScope() {
    if (before >= 0) cudaSetDevice(before);
  }
};

int launched() {
  if (cudaGetLastError() == cudaSuccess) return FFN_B200_OK;
  return FFN_B200_ERR_CUDA;
}

int device_sms(int given, int* sms) {
  *sms = given;
  if (given > 0) return FFN_B200_OK;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return FFN_B200_ERR_DEVICE;
  }
  int maj = 0, min = 0;
  return ffn_b200_device_info(dev, sms, &maj, &min);
}

int check_device(int device) {
  int sms = 0, maj = 0, min = 0;
  const int rc = ffn_b200_device_info(device, &sms, &maj, &min);
  if (rc) return rc;
  return maj == 10 && min == 0 ? FFN_B200_OK : FFN_B200_ERR_DEVICE;
}

int check_linear(const ffn_b200_linear_problem& p) {
  if (p.m <= 0 || p.k <= 0 || p.n <= 0 || p.k > kMaxDim || p.n > kMaxDim || p.m > (int64_t(1) << 31) - 16)
    return FFN_B200_ERR_INVALID;
  if (p.dtype != FFN_B200_F16 && p.dtype != FFN_B200_BF16) return FFN_B200_ERR_INVALID;
  if (p.activation < 0 || p.activation > FFN_B200_IDENTITY || p.activation == FFN_B200_SWIGLU)
    return FFN_B200_ERR_INVALID;
  if (p.block_num < 0 || p.reserved || p.tile < 0 || p.tile > 2) return FFN_B200_ERR_INVALID;
  return FFN_B200_OK;
}

int check_router(const ffn_b200_router_problem& p) {
  if (p.m <= 0 || p.k <= 0 || p.k > kMaxDim || p.m > (int64_t(1) << 31) - 16) return FFN_B200_ERR_INVALID;
  if (p.experts < 1 || p.experts > FFN_B200_MAX_EXPERTS || p.top_k < 1 || p.top_k > FFN_B200_MAX_TOP_K ||
      p.top_k > p.experts)
    return FFN_B200_ERR_INVALID;
  if (p.dtype != FFN_B200_F16 && p.dtype != FFN_B200_BF16) return FFN_B200_ERR_INVALID;
  if ((p.weight_f32 | p.sigmoid | p.renormalize) & ~1 || p.reserved) return FFN_B200_ERR_INVALID;
  return FFN_B200_OK;
}

int check_moe(const ffn_b200_moe_problem& p) {
  if (p.m <= 0 || p.k <= 0 || p.h <= 0 || p.n <= 0 || p.k > kMaxDim || p.h > kMaxDim || p.n > kMaxDim)
    return FFN_B200_ERR_INVALID;
  if (p.m > FFN_B200_MOE_MAX_TOKENS) return FFN_B200_ERR_TOO_LARGE;
  if (p.experts < 1 || p.experts > FFN_B200_MAX_EXPERTS || p.top_k < 1 || p.top_k > FFN_B200_MAX_TOP_K ||
      p.top_k > p.experts)
    return FFN_B200_ERR_INVALID;
  if (p.dtype != FFN_B200_F16 && p.dtype != FFN_B200_BF16) return FFN_B200_ERR_INVALID;
  if (p.activation < 0 || p.activation > FFN_B200_SWIGLU || p.block_num < 0) return FFN_B200_ERR_INVALID;
  return FFN_B200_OK;
}

}  // namespace

struct ffn_b200_linear {
  ffn_b200_linear_problem prob;
  ffn_b200_linear_plan plan;
  int device;
  const void* w;
  int64_t ldw;
  const void* bias;
};

struct ffn_b200_moe {
  ffn_b200_moe_problem prob;
  ffn_b200_moe_plan plan;
  ffn_b200_moe_buffers buf;
  int device;
  uint64_t wait_limit_ns;
  int inject;
};

extern "C" {

// ---- dense projection ----------------------------------------------------------------------
int ffn_b200_linear_make_plan(const ffn_b200_linear_problem* pr, ffn_b200_linear_plan* out) {
  if (!pr || !out) return FFN_B200_ERR_INVALID;
  int rc = check_linear(*pr);
  if (rc) return rc;
  int sms = 0;
  rc = device_sms(pr->sm_count, &sms);
  if (rc) return rc;
  std::memset(out, 0, sizeof(*out));
  out->block_num = sms;
  out->split = 1;
  return FFN_B200_OK;
}

int ffn_b200_linear_prepare(const ffn_b200_linear_problem* pr, const void* w, int64_t ldw, const void* bias,
                            float* workspace, uint32_t* counters, int device, ffn_b200_linear** out) {
  if (!pr || !w || !out) return FFN_B200_ERR_INVALID;
  *out = nullptr;
  ffn_b200_linear_plan plan;
  int rc = check_device(device);
  if (!rc) rc = ffn_b200_linear_make_plan(pr, &plan);
  if (rc) return rc;
  if (bad_rows(w, ldw, pr->k)) return FFN_B200_ERR_ALIGNMENT;
  auto* h = new (std::nothrow) ffn_b200_linear();
  if (!h) return FFN_B200_ERR_INVALID;
  h->prob = *pr;
  h->plan = plan;
  h->device = device;
  h->w = w;
  h->ldw = ldw;
  h->bias = bias;
  *out = h;
  return FFN_B200_OK;
}

int ffn_b200_linear_run(ffn_b200_linear* h, const void* x, int64_t ldx, const void* res, int64_t ldr, void* y,
                        int64_t ldy, void* stream) {
  if (!h || !x || !y) return FFN_B200_ERR_INVALID;
  const ffn_b200_linear_problem& p = h->prob;
  if (bad_rows(x, ldx, p.k) || bad_rows(y, ldy, p.n) || (res && bad_rows(res, ldr, p.n))) return FFN_B200_ERR_ALIGNMENT;
  DeviceScope scope(h->device);
  if (!scope.ok) return FFN_B200_ERR_DEVICE;
  const int64_t blocks = cdiv(p.m * p.n, 256);
  if (blocks >= (int64_t(1) << 31)) return FFN_B200_ERR_TOO_LARGE;
  auto* kern = p.dtype == FFN_B200_BF16 ? ffnb200::simple_linear<true> : ffnb200::simple_linear<false>;
  kern<<<static_cast<unsigned>(blocks), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      x, ldx, h->w, h->ldw, h->bias, res, ldr, y, ldy, p.m, static_cast<int>(p.k), static_cast<int>(p.n), p.activation);
  return launched();
}

int ffn_b200_linear_destroy(ffn_b200_linear* h) {
  delete h;
  return FFN_B200_OK;
}

// ---- expert router -------------------------------------------------------------------------
int ffn_b200_router_scratch(const ffn_b200_router_problem* pr, int64_t* logit_doubles, int64_t* counter_words) {
  if (!pr || !logit_doubles || !counter_words) return FFN_B200_ERR_INVALID;
  const int rc = check_router(*pr);
  if (rc) return rc;
  *logit_doubles = pr->m * pr->experts;
  *counter_words = cdiv(pr->m, 8);
  return FFN_B200_OK;
}

int ffn_b200_router_run(const ffn_b200_router_problem* pr, const void* x, int64_t ldx, const void* w, int64_t ldw,
                        const float* cbias, const uint8_t* mask, int32_t* ids, float* weights, double* logits,
                        uint32_t* counters, void* stream) {
  if (!pr || !x || !w || !ids || !weights || !logits || !counters) return FFN_B200_ERR_INVALID;
  const int rc = check_router(*pr);
  if (rc) return rc;
  if (bad_rows(x, ldx, pr->k) || bad_rows(w, ldw, pr->k)) return FFN_B200_ERR_ALIGNMENT;
  auto* kern = pr->dtype == FFN_B200_BF16
                   ? (pr->weight_f32 ? ffnb200::simple_route<true, true> : ffnb200::simple_route<true, false>)
                   : (pr->weight_f32 ? ffnb200::simple_route<false, true> : ffnb200::simple_route<false, false>);
  kern<<<static_cast<unsigned>(pr->m), 128, 0, static_cast<cudaStream_t>(stream)>>>(
      x, ldx, w, ldw, cbias, mask, ids, weights, logits, static_cast<int>(pr->k), pr->experts, pr->top_k, pr->sigmoid,
      pr->renormalize, pr->scale);
  return launched();
}

// ---- mixture-of-experts layer --------------------------------------------------------------
int ffn_b200_moe_make_plan(const ffn_b200_moe_problem* pr, ffn_b200_moe_plan* out) {
  if (!pr || !out) return FFN_B200_ERR_INVALID;
  int rc = check_moe(*pr);
  if (rc) return rc;
  int sms = 0;
  rc = device_sms(pr->sm_count, &sms);
  if (rc) return rc;
  std::memset(out, 0, sizeof(*out));
  out->block_num = pr->block_num ? pr->block_num : sms;
  out->hidden_rows = pr->m * pr->top_k;
  out->hidden_pitch = pitch_of(pr->h);
  out->workspace_floats = 4;
  out->counter_words = 4;
  out->status_words = 4;
  return FFN_B200_OK;
}

int ffn_b200_moe_prepare(const ffn_b200_moe_problem* pr, const ffn_b200_moe_buffers* b, int device,
                         ffn_b200_moe** out) {
  if (!pr || !b || !out) return FFN_B200_ERR_INVALID;
  *out = nullptr;
  ffn_b200_moe_plan plan;
  int rc = check_device(device);
  if (!rc) rc = ffn_b200_moe_make_plan(pr, &plan);
  if (rc) return rc;
  if (!b->w1 || !b->w2 || !b->hidden || !b->workspace || !b->counters || !b->status) return FFN_B200_ERR_INVALID;
  if (bad_rows(b->w1, b->ldw1, pr->k) || bad_rows(b->w2, b->ldw2, pr->h) || b->stride1 % 8 || b->stride2 % 8)
    return FFN_B200_ERR_ALIGNMENT;
  auto* h = new (std::nothrow) ffn_b200_moe();
  if (!h) return FFN_B200_ERR_INVALID;
  h->prob = *pr;
  h->plan = plan;
  h->buf = *b;
  h->device = device;
  h->wait_limit_ns = 4000000000ull;
  h->inject = 0;
  *out = h;
  return FFN_B200_OK;
}

int ffn_b200_moe_run(ffn_b200_moe* h, const void* x, int64_t ldx, const int32_t* ids, const float* weights,
                     const void* res, int64_t ldr, void* y, int64_t ldy, void* stream) {
  if (!h || !x || !ids || !weights || !y) return FFN_B200_ERR_INVALID;
  const ffn_b200_moe_problem& p = h->prob;
  const ffn_b200_moe_buffers& b = h->buf;
  if (bad_rows(x, ldx, p.k) || bad_rows(y, ldy, p.n) || (res && bad_rows(res, ldr, p.n))) return FFN_B200_ERR_ALIGNMENT;
  DeviceScope scope(h->device);
  if (!scope.ok) return FFN_B200_ERR_DEVICE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf = p.dtype == FFN_B200_BF16;
  const int k = static_cast<int>(p.k), hh = static_cast<int>(p.h), n = static_cast<int>(p.n);
  const dim3 up(static_cast<unsigned>(cdiv(hh, 128)), static_cast<unsigned>(p.m * p.top_k));
  const dim3 dn(static_cast<unsigned>(cdiv(n, 128)), static_cast<unsigned>(p.m));
  (bf ? ffnb200::simple_expert_up<true> : ffnb200::simple_expert_up<false>)<<<up, 128, 0, st>>>(
      x, ldx, ids, p.experts, b.w1, b.ldw1, b.stride1, b.hidden, h->plan.hidden_pitch, p.top_k, k, hh, p.activation);
  (bf ? ffnb200::simple_expert_down<true> : ffnb200::simple_expert_down<false>)<<<dn, 128, 0, st>>>(
      b.hidden, h->plan.hidden_pitch, ids, weights, p.experts, b.w2, b.ldw2, b.stride2, res, ldr, y, ldy, p.top_k, hh, n);
  return launched();
}

int ffn_b200_moe_reset(ffn_b200_moe* h, void* stream) {
  if (!h) return FFN_B200_ERR_INVALID;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (cudaMemsetAsync(h->buf.counters, 0, 4 * h->plan.counter_words, st) != cudaSuccess ||
      cudaMemsetAsync(h->buf.status, 0, 4 * h->plan.status_words, st) != cudaSuccess) {
    cudaGetLastError();
    return FFN_B200_ERR_CUDA;
  }
  return FFN_B200_OK;
}

int ffn_b200_moe_set_wait_limit(ffn_b200_moe* h, uint64_t ns) {
  if (!h || ns == 0) return FFN_B200_ERR_INVALID;
  h->wait_limit_ns = ns;
  return FFN_B200_OK;
}

int ffn_b200_moe_set_fault_injection(ffn_b200_moe* h, int mode) {
  if (!h || mode < 0 || mode > 1) return FFN_B200_ERR_INVALID;
  h->inject = mode;
  return FFN_B200_OK;
}

int ffn_b200_moe_destroy(ffn_b200_moe* h) {
  delete h;
  return FFN_B200_OK;
}

}  // extern "C"
