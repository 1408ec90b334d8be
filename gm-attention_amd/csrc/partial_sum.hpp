// The sums of workgroups' partial rows, in double and in a fixed order.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"

namespace gm {

constexpr int kPartialColumns = 8, kPartialParts = 32;

// out[c] = sum over rows of partial (rows, columns): a workgroup eight columns, 32 parts of the rows, whose loads do
// not wait for each other.
template <typename T>
__global__ __launch_bounds__(256) void partial_sum_kernel(const T* partial, int64_t rows, int columns, T* out) {
  __shared__ double sums[kPartialParts][kPartialColumns + 1];
  const int c = threadIdx.x % kPartialColumns, part = threadIdx.x / kPartialColumns;
  const int column = blockIdx.x * kPartialColumns + c;
  double s = 0.0;
  if (column < columns) {
#pragma unroll 8
    for (int64_t r = part; r < rows; r += kPartialParts) s += (double)partial[r * columns + column];
  }
  sums[part][c] = s;
  __syncthreads();
  if (part == 0 && column < columns) {
    double t = 0.0;
    for (int i = 0; i < kPartialParts; ++i) t += sums[i][c];
    out[column] = (T)t;
  }
}

template <typename T>
void launch_partial_sum(const T* partial, int64_t rows, int columns, T* out, hipStream_t stream) {
  const int groups = (columns + kPartialColumns - 1) / kPartialColumns;
  hipLaunchKernelGGL(partial_sum_kernel<T>, dim3((unsigned)groups), dim3(256), 0, stream, partial, rows, columns, out);
}

}  // namespace gm
