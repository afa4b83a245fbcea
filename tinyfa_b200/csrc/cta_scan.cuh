// Prefix sum over a CTA of up to 1024 threads.
#pragma once

#include <cuda_runtime.h>

namespace tfa_b200 {

// Inclusive sum; every thread gets the CTA's total as well.  sWarp: 32 words of shared memory, free again on return.
__device__ __forceinline__ long long cta_scan(long long v, long long* sWarp, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  if (lane == 31) sWarp[warp] = v;
  __syncthreads();
  if (warp == 0) {
    long long w = lane < warps ? sWarp[lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += o;
    }
    sWarp[lane] = w;
  }
  __syncthreads();
  total = sWarp[31];
  if (warp > 0) v += sWarp[warp - 1];
  __syncthreads();
  return v;
}

}  // namespace tfa_b200
