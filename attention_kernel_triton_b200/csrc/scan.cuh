// Prefix sums over a block of 1024 threads.
#pragma once
#include <stdint.h>

namespace akt {

// Exclusive prefix sum of x over the block; total through `total`.  sums: 33 of them.
template <typename S>
__device__ __forceinline__ S block_scan(S x, S* sums, S& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  S v = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const S y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  if (warp == 0) {
    S w = sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const S y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    sums[lane] = w;
  }
  __syncthreads();
  total = sums[31];
  const S before = warp ? sums[warp - 1] : 0;
  __syncthreads();
  return before + v - x;
}

}  // namespace akt
