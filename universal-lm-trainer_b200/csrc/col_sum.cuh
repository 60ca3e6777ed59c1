// Column sums of per-CTA partial rows (sm_100a).
#pragma once

#include "common.cuh"

namespace ulm {
namespace {

// dw[c] = sum over the partial rows, in a fixed order: a CTA takes 32 columns, its 32 x 32 threads each add
// every 32nd partial row of one column (coalesced 128-byte reads, short independent chains), and the 32
// sub-sums of a column are added in index order.
__global__ void __launch_bounds__(1024)
col_sum_kernel(const float* partial, float* dw, int nparts, int d) {
  __shared__ float sub[32][33];
  grid_dependency_wait();                                // at once where the launch is an ordinary one
  const int c = blockIdx.x * 32 + threadIdx.x;
  float t = 0.f;
  if (c < d)
    for (int p = threadIdx.y; p < nparts; p += 32) t += partial[(int64_t)p * d + c];
  sub[threadIdx.y][threadIdx.x] = t;
  __syncthreads();
  if (threadIdx.y == 0 && c < d) {
    float sum = 0.f;
#pragma unroll
    for (int g = 0; g < 32; ++g) sum += sub[g][threadIdx.x];
    dw[c] = sum;
  }
}

}  // namespace
}  // namespace ulm
