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
  // PAST: whole pieces do not stay in the last-level cache.
  template <bool PAST = false>
  static __device__ __forceinline__ void store(T *at, long long count, const Held &v) {
    if (count >= V) {
      if (PAST) __builtin_nontemporal_store(v, reinterpret_cast<Held *>(at));
      else *reinterpret_cast<Held *>(at) = v;
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
  typedef int Words __attribute__((ext_vector_type(2)));
  Words q = __builtin_bit_cast(Words, v);
  q[0] = __builtin_amdgcn_mov_dpp(q[0], CONTROL, 0xf, 0xf, true), q[1] = __builtin_amdgcn_mov_dpp(q[1], CONTROL, 0xf, 0xf, true);
  return __builtin_bit_cast(double, q);
}

// Of the two lanes of a wavefront that lie 16 (32) apart both values, the lower lane's first, by a move within the vector unit.
template <typename C>
struct Two {
  C low, high;
};
template <int APART>
__device__ __forceinline__ Two<int> pair_of(int v) {
  const auto both = APART == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return {(int)both[0], (int)both[1]};
}
template <int APART>
__device__ __forceinline__ Two<float> pair_of(float v) {
  const Two<int> both = pair_of<APART>(__builtin_bit_cast(int, v));
  return {__builtin_bit_cast(float, both.low), __builtin_bit_cast(float, both.high)};
}
template <int APART>
__device__ __forceinline__ Two<double> pair_of(double v) {
  typedef int Words __attribute__((ext_vector_type(2)));
  const Words words = __builtin_bit_cast(Words, v);
  const Two<int> first = pair_of<APART>(words[0]), second = pair_of<APART>(words[1]);
  return {__builtin_bit_cast(double, Words{first.low, second.low}), __builtin_bit_cast(double, Words{first.high, second.high})};
}

// `over` of each run of `lanes` lanes, a power of two, for all of them.
template <typename C, typename Over>
__device__ __forceinline__ C lanes_over(C v, int lanes, Over over) {
  if (lanes > 1) v = over(v, from_lane<0xb1>(v));   // lanes 1 0 3 2 of four
  if (lanes > 2) v = over(v, from_lane<0x4e>(v));   // 2 3 0 1
  if (lanes > 4) v = over(v, from_lane<0x141>(v));  // eight from behind
  if (lanes > 8) v = over(v, from_lane<0x140>(v));  // sixteen from behind
  if (lanes > 16) {
    const Two<C> both = pair_of<16>(v);
    v = over(both.low, both.high);
  }
  if (lanes > 32) {
    const Two<C> both = pair_of<32>(v);
    v = over(both.low, both.high);
  }
  return v;
}
template <typename C>
__device__ __forceinline__ C lanes_add(C v, int lanes) {
  return lanes_over(v, lanes, [](C a, C b) { return a + b; });
}
template <typename C>
__device__ __forceinline__ C lanes_max(C v, int lanes) {
  return lanes_over(v, lanes, [](C a, C b) { return max(a, b); });
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
