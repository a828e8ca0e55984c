// Sums, extremes, scans and sorts over a workgroup of TH threads (64 times a power of two, at most 1024). Every thread
// of the workgroup calls them, and the LDS they use may be used again after them without a barrier between. What is
// the same in all threads comes back in scalar registers.
#pragma once

#include "slg_common.h"

namespace slg {

// v of lane `lane` (the same lane in all threads).
template <typename T>
__device__ __forceinline__ T read_lane(T v, int lane) {
  static_assert(sizeof(T) == 4 || sizeof(T) == 8, "");
  union {
    T v;
    int i[sizeof(T) / 4];
  } u = {v};
#pragma unroll
  for (int k = 0; k < (int)sizeof(T) / 4; ++k) u.i[k] = __builtin_amdgcn_readlane(u.i[k], lane);
  return u.v;
}
template <typename T>
__device__ __forceinline__ T uniform(T v) {
  return read_lane(v, 0);
}
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

template <typename T, class F>
__device__ __forceinline__ T wave_reduce(T v, F f) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = f(v, __shfl_xor(v, d));
  return uniform(v);
}

// v of all threads joined by f, in one order; part: TH / 64 values of LDS.
template <int TH, typename T, class F>
__device__ __forceinline__ T block_reduce(T v, T* part, F f) {
  constexpr int W = TH / 64;
  v = wave_reduce(v, f);
  if constexpr (W > 1) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[threadIdx.x & (W - 1)];
#pragma unroll
    for (int d = W / 2; d; d >>= 1) v = f(v, __shfl_xor(v, d));
    v = uniform(v);
    __syncthreads();
  }
  return v;
}

// The sum of v over the threads before this one, and over all of them.
template <int TH>
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* part, uint64_t& total) {
  constexpr int W = TH / 64;
  const int lane = threadIdx.x & 63;
  uint64_t s = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t o = __shfl_up(s, d);
    if (lane >= d) s += o;
  }
  if constexpr (W == 1) {
    total = read_lane(s, 63);
    return s - v;
  } else {
    if (lane == 63) part[threadIdx.x >> 6] = s;
    __syncthreads();
    uint64_t w = part[lane & (W - 1)];
#pragma unroll
    for (int d = 1; d < W; d <<= 1) {
      const uint64_t o = __shfl_up(w, d);
      if ((lane & (W - 1)) >= d) w += o;
    }
    total = read_lane(w, W - 1);
    const int wave = wave_id();
    const uint64_t before = wave ? read_lane(w, wave - 1) : 0;
    __syncthreads();
    return before + s - v;
  }
}

// Values in falling order, one a thread; `size` (a power of two, at most TH, the same in all threads) of them count,
// the first threads'. buf: TH values of LDS. A bitonic network: neighbours up to a wave apart by shuffles, further
// ones through LDS.
template <int TH>
__device__ __forceinline__ uint64_t block_sort(uint64_t v, int size, uint64_t* buf) {
  const int t = threadIdx.x;
#pragma unroll 1
  for (int s = 2; s <= size; s <<= 1) {
#pragma unroll 1
    for (int d = s >> 1; d; d >>= 1) {
      uint64_t o;
      if (TH > 64 && d >= 64) {
        __syncthreads();
        buf[t] = v;
        __syncthreads();
        o = buf[t ^ d];
      } else {
        o = __shfl_xor(v, d);
      }
      const bool larger = ((t & s) == 0) == ((t & d) == 0);
      v = (v > o) == larger ? v : o;
    }
  }
  if constexpr (TH > 64) __syncthreads();
  return v;
}

}  // namespace slg
