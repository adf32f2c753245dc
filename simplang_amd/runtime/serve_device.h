// serve_device.h -- device helpers of the kernels that serve a batch of sequences
// (attention.hip, kv8.hip).
#pragma once

#include "rt_device.h"

namespace simp {

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }

// 2^x, below 2^-126 as 0
__device__ __forceinline__ float pow2(float x) { return __builtin_amdgcn_exp2f(x); }

// The last s of 0 .. n-1 for which f(s) holds, where it holds up to some s and not
// behind it; 0 where it holds for none.  The 64 lanes look at 64 places at a time, so up
// to 64 sequences cost one round trip to memory.  Every lane of the wave takes part.
template <class F>
__device__ __forceinline__ int last_of(int n, F f) {
  const int lane = threadIdx.x & 63;
  int lo = 0;
  while (n > 1) {
    const int step = (n + 63) >> 6;
    const unsigned long long yes = __ballot(lane * step < n && f(lo + lane * step));
    if (!yes) break;
    const int k = 63 - __clzll((long long)yes);
    lo += k * step;
    n = min(step, n - k * step);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

}  // namespace simp
