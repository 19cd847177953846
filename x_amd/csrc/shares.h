// Sums of the workgroups' shares of a small gradient, in a fixed order.
#pragma once
#include "common.h"

namespace atlhip {
namespace {

// out[c] = sum over n shares part (n, D): 16 columns a workgroup, 64 interleaved runs of the shares side by side.
constexpr int kSumChannels = 16, kSumRuns = 64;
__global__ void __launch_bounds__(kSumChannels* kSumRuns) k_sum_shares(const float* __restrict__ part, int n, int64_t D,
                                                                       float* __restrict__ out) {
  __shared__ float lds[kSumRuns][kSumChannels];
  const int ch = threadIdx.x % kSumChannels, run = threadIdx.x / kSumChannels;
  const int64_t c = (int64_t)blockIdx.x * kSumChannels + ch;
  float sum = 0.f;
  if (c < D)
#pragma unroll 4
    for (int b = run; b < n; b += kSumRuns) sum += part[b * D + c];
  lds[run][ch] = sum;
  __syncthreads();
  for (int half = kSumRuns / 2; half >= 1; half /= 2) {
    if (run < half) lds[run][ch] += lds[run + half][ch];
    __syncthreads();
  }
  if (run == 0 && c < D) out[c] = lds[0][ch];
}

}  // namespace
}  // namespace atlhip
