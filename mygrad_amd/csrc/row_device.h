// What the kernels over rows (layer norm, log probabilities, distillation) share: sums over a block, and the types sums are carried in.
#pragma once

#include "internal.h"

namespace mg {

template <typename C>
__device__ __forceinline__ C wave_add(C v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

// The sums of N values over a block of up to 16 wavefronts, for all of its threads; `space` is N * 16 values of LDS.
template <int N, typename C>
__device__ __forceinline__ void block_add(C (&v)[N], C *space) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = wave_add(v[n]);
  if (waves == 1) return;
  __syncthreads();  // whoever still reads what was there before
  if (lane == 0)
#pragma unroll
    for (int n = 0; n < N; ++n) space[n * 16 + wave] = v[n];
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    v[n] = 0;
    for (int w = 0; w < waves; ++w) v[n] += space[n * 16 + w];
  }
}

}  // namespace mg
