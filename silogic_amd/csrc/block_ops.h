// Sums, extremes, scans and sorts over a workgroup of TH threads (64 times a power of two, at most 1024). Every thread
// of the workgroup calls them, and the LDS they use may be used again after them without a barrier between. What is
// the same in all threads comes back in scalar registers.
//
// Lanes exchange by DPP moves and swizzles, whose pattern is in the instruction: a shuffle by a lane's number takes
// four more instructions for the address and goes through LDS (64 largest of 4096 rows of 32000 bf16: 73 us with those,
// 53 without).
#pragma once

#include "slg_common.h"

namespace slg {

// A launch takes fewer than 2^32 threads along x: workgroups past the first kGridX go along y, and those past the last
// end at once.
constexpr uint32_t kGridX = 1u << 20;
inline dim3 grid_of(int64_t blocks) {
  return blocks <= kGridX ? dim3((unsigned)blocks) : dim3(kGridX, (unsigned)cdiv(blocks, kGridX));
}
__device__ __forceinline__ uint32_t block_id() { return blockIdx.y * kGridX + blockIdx.x; }   // blocks: at most 2^31

template <typename T, class F>
__device__ __forceinline__ T by_words(T v, F f) {
  static_assert(sizeof(T) % 4 == 0, "");
  union {
    T v;
    int i[sizeof(T) / 4];
  } u = {v};
#pragma unroll
  for (int k = 0; k < (int)(sizeof(T) / 4); ++k) u.i[k] = f(u.i[k]);
  return u.v;
}

// v of lane `lane` (the same lane in all threads).
template <typename T>
__device__ __forceinline__ T read_lane(T v, int lane) {
  return by_words(v, [&](int w) { return __builtin_amdgcn_readlane(w, lane); });
}
template <typename T>
__device__ __forceinline__ T uniform(T v) {
  return by_words(v, [](int w) { return __builtin_amdgcn_readfirstlane(w); });
}
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// v of the lane whose number differs in bit D.
template <int D, typename T>
__device__ __forceinline__ T lane_xor(T v) {
  static_assert(D == 1 || D == 2 || D == 4 || D == 8 || D == 16 || D == 32, "");
  if constexpr (D == 32) {
    const int at = (int)((threadIdx.x & 63) ^ 32) << 2;
    return by_words(v, [&](int w) { return __builtin_amdgcn_ds_bpermute(at, w); });
  } else {
    return by_words(v, [](int w) {
      if constexpr (D == 1) return __builtin_amdgcn_mov_dpp(w, 0xb1, 0xf, 0xf, true);        // quad_perm 1 0 3 2
      else if constexpr (D == 2) return __builtin_amdgcn_mov_dpp(w, 0x4e, 0xf, 0xf, true);   // quad_perm 2 3 0 1
      else if constexpr (D == 8) return __builtin_amdgcn_mov_dpp(w, 0x128, 0xf, 0xf, true);  // row_ror 8
      else return __builtin_amdgcn_ds_swizzle(w, (D << 10) | 0x1f);
    });
  }
}
// v of the lane N before within its row of 16; 0 where there is none.
template <int N, typename T>
__device__ __forceinline__ T row_shift(T v) {
  return by_words(v, [](int w) { return __builtin_amdgcn_update_dpp(0, w, 0x110 + N, 0xf, 0xf, true); });
}

template <int LANES = 64, typename T, class F>
__device__ __forceinline__ T lanes_reduce(T v, F f) {
  if constexpr (LANES > 1) v = f(v, lane_xor<1>(v));
  if constexpr (LANES > 2) v = f(v, lane_xor<2>(v));
  if constexpr (LANES > 4) v = f(v, lane_xor<4>(v));
  if constexpr (LANES > 8) v = f(v, lane_xor<8>(v));
  if constexpr (LANES > 16) v = f(v, lane_xor<16>(v));
  if constexpr (LANES > 32) v = f(v, lane_xor<32>(v));
  return v;
}
template <typename T, class F>
__device__ __forceinline__ T wave_reduce(T v, F f) {
  return uniform(lanes_reduce(v, f));
}

// v of all threads joined by f, in one order; part: TH / 64 values of LDS.
template <int TH, typename T, class F>
__device__ __forceinline__ T block_reduce(T v, T* part, F f) {
  constexpr int W = TH / 64;
  v = wave_reduce(v, f);
  if constexpr (W > 1) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = uniform(lanes_reduce<W>(part[threadIdx.x & (W - 1)], f));
    __syncthreads();
  }
  return v;
}

// Sums of v over the lanes up to this one.
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {
  v += row_shift<1>(v);
  v += row_shift<2>(v);
  v += row_shift<4>(v);
  v += row_shift<8>(v);
  const int lane = threadIdx.x & 63;
  const uint64_t r0 = read_lane(v, 15), r1 = read_lane(v, 31), r2 = read_lane(v, 47);
  return v + (lane < 16 ? 0 : lane < 32 ? r0 : lane < 48 ? r0 + r1 : r0 + r1 + r2);
}

// The sum of v over the threads before this one, and over all of them.
template <int TH>
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* part, uint64_t& total) {
  constexpr int W = TH / 64;
  const uint64_t s = wave_scan(v);
  if constexpr (W == 1) {
    total = read_lane(s, 63);
    return s - v;
  } else {
    if ((threadIdx.x & 63) == 63) part[threadIdx.x >> 6] = s;
    __syncthreads();
    uint64_t w = part[threadIdx.x & (W - 1)];   // the same in each row of 16 lanes
    w += row_shift<1>(w);
    w += row_shift<2>(w);
    w += row_shift<4>(w);
    w += row_shift<8>(w);
    total = read_lane(w, W - 1);
    const int wave = wave_id();
    const uint64_t before = wave ? read_lane(w, wave - 1) : 0;
    __syncthreads();
    return before + s - v;
  }
}

// Lanes whose number has bit D clear.
template <int D>
constexpr uint64_t kLanesWithout = D == 1    ? 0x5555555555555555ull
                                   : D == 2  ? 0x3333333333333333ull
                                   : D == 4  ? 0x0f0f0f0f0f0f0f0full
                                   : D == 8  ? 0x00ff00ff00ff00ffull
                                   : D == 16 ? 0x0000ffff0000ffffull
                                             : 0x00000000ffffffffull;
// One step of a bitonic network: the larger of v and the other thread's in the lanes of `larger`.
template <typename T>
__device__ __forceinline__ T sort_step(T v, T other, uint64_t larger) {
  return __builtin_amdgcn_inverse_ballot_w64(__ballot(v > other) ^ ~larger) ? v : other;
}
// Steps D, D / 2, .. 1 of runs whose lanes are `falling` or rising.
template <int D, typename T>
__device__ __forceinline__ T sort_lanes(T v, uint64_t falling) {
  v = sort_step(v, lane_xor<D>(v), ~(falling ^ kLanesWithout<D>));
  if constexpr (D > 1) v = sort_lanes<D / 2>(v, falling);
  return v;
}
// A wave's values in falling or in rising order.
template <typename T>
__device__ __forceinline__ T wave_sort(T v, bool falling) {
  v = sort_lanes<1>(v, kLanesWithout<2>);
  v = sort_lanes<2>(v, kLanesWithout<4>);
  v = sort_lanes<4>(v, kLanesWithout<8>);
  v = sort_lanes<8>(v, kLanesWithout<16>);
  v = sort_lanes<16>(v, kLanesWithout<32>);
  return sort_lanes<32>(v, falling ? ~0ull : 0);
}

// Values in falling order, one a thread; the first n threads' count (the same n in all threads, at most TH), the others
// hold 0. buf: TH values of LDS. Waves that hold nothing only wait.
template <int TH>
__device__ __forceinline__ uint64_t block_sort(uint64_t v, int n, uint64_t* buf) {
  const int t = threadIdx.x;
  int size = 64;
  while (size < n) size *= 2;
  const int first = wave_id() * 64;   // of the wave
  const bool mine = first < size;
  if (mine) v = wave_sort(v, (first & 64) == 0);
  if constexpr (TH > 64) {
#pragma unroll 1
    for (int s = 128; s <= size; s <<= 1) {
      const uint64_t falling = first & s ? 0 : ~0ull;
#pragma unroll 1
      for (int d = s >> 1; d >= 64; d >>= 1) {
        __syncthreads();
        if (mine) buf[t] = v;
        __syncthreads();
        if (mine) v = sort_step(v, buf[t ^ d], first & d ? ~falling : falling);
      }
      if (mine) v = sort_lanes<32>(v, falling);
    }
    __syncthreads();
  }
  return v;
}

}  // namespace slg
