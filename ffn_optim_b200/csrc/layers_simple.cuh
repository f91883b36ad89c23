// Plain CUDA-core forms of the dense projection, the expert router and the routed experts:
// one output per thread, sums in fp32 (the router's in fp64).
#pragma once

#include "ffn_kernel.cuh"

namespace ffnb200 {

template <bool BF16>
__device__ __forceinline__ float elem(const void* p, size_t i) {
  return unpack_lo<BF16>(static_cast<uint32_t>(static_cast<const uint16_t*>(p)[i]));
}
__device__ __forceinline__ float apply_act(float z, int act) {
  if (act == 0) return gelu_rational(z);
  if (act == 1) return gelu_erf(z);
  if (act == 2) return silu(z);
  return z;
}

template <bool BF16>
__global__ void simple_linear(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                              const void* res, int64_t ldr, void* y, int64_t ldy, int64_t m, int k, int n, int act) {
  const int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
  if (i >= m * n) return;
  const int64_t t = i / n;
  const int c = static_cast<int>(i % n);
  float z = 0.f;
  for (int j = 0; j < k; ++j) z = fmaf(elem<BF16>(x, t * ldx + j), elem<BF16>(w, c * ldw + j), z);
  if (bias) z += elem<BF16>(bias, c);
  z = apply_act(z, act);
  if (res) z += elem<BF16>(res, t * ldr + c);
  static_cast<uint16_t*>(y)[t * ldy + c] = cvt1<BF16>(z);
}

template <bool BF16, bool W32>
__global__ void simple_route(const void* x, int64_t ldx, const void* w, int64_t ldw, const float* cbias,
                             const uint8_t* mask, int32_t* ids, float* weights, double* logits, int k, int experts,
                             int top, int sigmoid, int renorm, float scale) {
  const int64_t t = blockIdx.x;
  double* row = logits + t * experts;
  if (mask && !mask[t]) {
    for (int j = threadIdx.x; j < top; j += blockDim.x) ids[t * top + j] = -1, weights[t * top + j] = 0.f;
    return;
  }
  for (int e = threadIdx.x; e < experts; e += blockDim.x) {
    double z = 0.0;
    for (int j = 0; j < k; ++j) {
      const float wv = W32 ? static_cast<const float*>(w)[e * ldw + j] : elem<BF16>(w, e * ldw + j);
      z = fma(static_cast<double>(elem<BF16>(x, t * ldx + j)), static_cast<double>(wv), z);
    }
    row[e] = z;
  }
  __syncthreads();
  if (threadIdx.x) return;
  if (sigmoid) {
    for (int e = 0; e < experts; ++e) row[e] = 1.0 / (1.0 + exp(-row[e]));
  } else {
    double top_z = -INFINITY, sum = 0.0;
    for (int e = 0; e < experts; ++e) top_z = row[e] > top_z || row[e] != row[e] ? row[e] : top_z;
    for (int e = 0; e < experts; ++e) sum += row[e] = exp(row[e] - top_z);
    for (int e = 0; e < experts; ++e) row[e] /= sum;
  }
  double total = 0.0;
  for (int j = 0; j < top; ++j) {
    int best = -1;
    double bk = 0.0;
    for (int e = 0; e < experts; ++e) {
      bool used = false;
      for (int q = 0; q < j; ++q) used |= ids[t * top + q] == e;
      if (used) continue;
      double key = row[e] + (cbias ? static_cast<double>(cbias[e]) : 0.0);
      if (key != key) key = -INFINITY;
      if (best < 0 || key > bk) best = e, bk = key;
    }
    ids[t * top + j] = best;
    total += row[best];
  }
  for (int j = 0; j < top; ++j)
    weights[t * top + j] = static_cast<float>(row[ids[t * top + j]] / (renorm ? total : 1.0) * static_cast<double>(scale));
}

}  // namespace ffnb200
