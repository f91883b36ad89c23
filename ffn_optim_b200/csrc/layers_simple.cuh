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

}  // namespace ffnb200
