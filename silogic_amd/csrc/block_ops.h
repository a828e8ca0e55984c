// Sums, extremes, scans and sorts over a workgroup of TH threads (a multiple of 64). Every thread of the workgroup
// calls them, and the arrays they use may be used again after them without a barrier between.
#pragma once

#include "slg_common.h"

namespace slg {

template <typename T, class F>
__device__ inline T wave_reduce(T v, F f) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = f(v, __shfl_xor(v, d));
  return v;
}

// v of all threads joined by f, in one order; part: TH / 64 values of LDS.
template <int TH, typename T, class F>
__device__ inline T block_reduce(T v, T* part, F f) {
  v = wave_reduce(v, f);
  if constexpr (TH > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < TH / 64; ++w) v = f(v, part[w]);
    __syncthreads();
  }
  return v;
}

// The sum of v over the threads before this one, and over all of them.
template <int TH>
__device__ inline uint64_t block_scan(uint64_t v, uint64_t* part, uint64_t& total) {
  const int lane = threadIdx.x & 63;
  uint64_t s = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t o = __shfl_up(s, d);
    if (lane >= d) s += o;
  }
  if constexpr (TH > 64) {
    if (lane == 63) part[threadIdx.x >> 6] = s;
    __syncthreads();
    uint64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < TH / 64; ++w) {
      if (w == (int)(threadIdx.x >> 6)) before = total;
      total += part[w];
    }
    __syncthreads();
    return before + s - v;
  } else {
    total = __shfl(s, 63);
    return s - v;
  }
}

// Values in falling order, one a thread; `size` (a power of two, at most TH, the same in all threads) of them count,
// the first threads'. buf: TH values of LDS. A bitonic network: neighbours up to a wave apart by shuffles, further
// ones through LDS.
template <int TH>
__device__ inline uint64_t block_sort(uint64_t v, int size, uint64_t* buf) {
  const int t = threadIdx.x;
  for (int s = 2; s <= size; s <<= 1) {
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
