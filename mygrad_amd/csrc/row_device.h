// What the kernels over rows (embedding, layer norm, log probabilities, distillation) share: pieces of a row that a lane loads at once, and
// sums over wavefronts and blocks.
#pragma once

#include "internal.h"

namespace mg {

// V neighbouring values of a row, 16 bytes.  Rows begin wherever their length puts them: the vector instructions take any address, and a
// row of 50001 halves moves as fast as one of 50000.
template <typename T>
struct Piece {
  static constexpr int V = 16 / sizeof(T);
  typedef T Held __attribute__((ext_vector_type(V), aligned(sizeof(T))));

  // From `at` on, of which `count` values are there (as many as V or more: all of them); the others are `otherwise`.
  static __device__ __forceinline__ Held load(const T *at, long long count, T otherwise) {
    Held v;
    if (count >= V) return *reinterpret_cast<const Held *>(at);
#pragma unroll
    for (int n = 0; n < V; ++n) v[n] = n < count ? at[n] : otherwise;
    return v;
  }
  static __device__ __forceinline__ void store(T *at, long long count, const Held &v) {
    if (count >= V) {
      *reinterpret_cast<Held *>(at) = v;
      return;
    }
#pragma unroll
    for (int n = 0; n < V; ++n)
      if (n < count) at[n] = v[n];
  }
};

// What another lane of a row of sixteen has, by a move within the vector unit.
template <int CONTROL>
__device__ __forceinline__ int from_lane(int v) {
  return __builtin_amdgcn_mov_dpp(v, CONTROL, 0xf, 0xf, true);
}
template <int CONTROL>
__device__ __forceinline__ float from_lane(float v) {
  return __builtin_bit_cast(float, from_lane<CONTROL>(__builtin_bit_cast(int, v)));
}
template <int CONTROL>
__device__ __forceinline__ double from_lane(double v) {
  typedef int Two __attribute__((ext_vector_type(2)));
  Two q = __builtin_bit_cast(Two, v);
  q[0] = __builtin_amdgcn_mov_dpp(q[0], CONTROL, 0xf, 0xf, true), q[1] = __builtin_amdgcn_mov_dpp(q[1], CONTROL, 0xf, 0xf, true);
  return __builtin_bit_cast(double, q);
}

// The sum over each run of `lanes` lanes, a power of two, for all of them.
template <typename C>
__device__ __forceinline__ C lanes_add(C v, int lanes) {
  if (lanes > 1) v += from_lane<0xb1>(v);   // lanes 1 0 3 2 of four
  if (lanes > 2) v += from_lane<0x4e>(v);   // 2 3 0 1
  if (lanes > 4) v += from_lane<0x141>(v);  // eight from behind
  if (lanes > 8) v += from_lane<0x140>(v);  // sixteen from behind
  if (lanes > 16) v += __shfl_xor(v, 16);
  if (lanes > 32) v += __shfl_xor(v, 32);
  return v;
}
// What the lanes of a wavefront wrote is there for all of them.
__device__ __forceinline__ void wave_sees() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <typename C>
__device__ __forceinline__ C wave_add(C v) {
  return lanes_add(v, 64);
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
