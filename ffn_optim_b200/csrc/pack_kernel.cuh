// Copies a strided [rows, cols] view of 16-bit values into rows of a 16-byte pitch, for operands whose
// own rows the TMA cannot address (odd pitch or base, transposed or strided views).  Tiles of 32
// rows x 32 columns go through shared memory, so that both sides move whole sectors when either
// the rows or the columns of the source are contiguous.  Bound by the launch for small views,
// by the source's sectors else.
#pragma once

#include "ffn_kernel.cuh"

namespace ffnb200 {

constexpr int kPackTile = 32;

__global__ void __launch_bounds__(256) pack_rows_kernel(const uint16_t* __restrict__ src, long long row_stride,
                                                        long long col_stride, long long rows, int cols,
                                                        uint16_t* __restrict__ dst, long long ld) {
  __shared__ uint16_t tile[kPackTile][kPackTile + 2];
  if (threadIdx.x == 0) grid_dep_launch();
  grid_dep_wait();
  const int a = threadIdx.x & 31, b = threadIdx.x >> 5;
  const long long r0 = static_cast<long long>(blockIdx.x) * kPackTile;
  const int c0 = static_cast<int>(blockIdx.y) * kPackTile;
  const bool by_rows = col_stride > row_stride;  // neighbouring rows lie closer than neighbouring columns
#pragma unroll
  for (int i = 0; i < kPackTile; i += 8) {
    const int r = by_rows ? a : b + i, c = by_rows ? b + i : a;
    if (r0 + r < rows && c0 + c < cols) tile[r][c] = src[(r0 + r) * row_stride + (c0 + c) * col_stride];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPackTile; i += 8)
    if (r0 + b + i < rows && c0 + a < cols) dst[(r0 + b + i) * ld + c0 + a] = tile[b + i][a];
}

}  // namespace ffnb200
