// The sums of workgroups' partial rows, in double and in a fixed order.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"

namespace gm {

// out[c] = sum over rows of partial (rows, columns): a workgroup sixteen columns, sixteen parts of the rows.
template <typename T>
__global__ __launch_bounds__(256) void partial_sum_kernel(const T* partial, int64_t rows, int columns, T* out) {
  __shared__ double sums[16][17];
  const int c = threadIdx.x & 15, part = threadIdx.x >> 4, column = blockIdx.x * 16 + c;
  double s = 0.0;
  if (column < columns)
    for (int64_t r = part; r < rows; r += 16) s += (double)partial[r * columns + column];
  sums[part][c] = s;
  __syncthreads();
  if (part == 0 && column < columns) {
    double t = 0.0;
    for (int i = 0; i < 16; ++i) t += sums[i][c];
    out[column] = (T)t;
  }
}

template <typename T>
void launch_partial_sum(const T* partial, int64_t rows, int columns, T* out, hipStream_t stream) {
  hipLaunchKernelGGL(partial_sum_kernel<T>, dim3((unsigned)((columns + 15) / 16)), dim3(256), 0, stream, partial, rows,
                     columns, out);
}

}  // namespace gm
