// Stable radix sort of (key, index) pairs, the order in which sums over
// references or tokens run: entries in ascending keys, indices of one key
// ascending, the same on every call. Least significant digits first, at most
// 10 bits a pass; a pass is a count of every workgroup's digits and a scatter.
//
// A wave ranks 64 entries at a time: ballots over the digit's bits give each
// lane the lanes that share its digit, the first of them adds their number to
// the wave's counter in LDS and reads what was there (LDS operations of a wave
// stay in order, so all of a lane's entries are in flight at once). A
// workgroup's first place of a digit is the sum of all smaller digits and of
// the earlier workgroups' counts, which every workgroup sums for itself from
// counts stored digit by digit: 16-byte loads, all in flight, where a separate
// scan would be a launch (with one load at a time that sum was most of a pass:
// 41 us at 524288 entries). Where the counts are few, a scatter also counts the
// next pass's digits, by where it puts each entry: in LDS, then added to the
// other workgroups' (whole numbers: the order does not matter), a launch of 4.5
// us less (fp32 backward of 2000 -> 2000, K = 8, B = 256, captured: 72 us for 76;
// references placed by counters took it to 69 and cost up to milliseconds
// where they fell on few inputs). Up to 4096 entries are sorted by one
// workgroup in one launch, passes through LDS.
//
// Key sources are functors with `int key(int64_t i)`, 0 <= key < 2^31.
#pragma once
#include <algorithm>

#include "slg_common.h"

namespace slg {

constexpr int kRadixThreads = 512, kRadixWaves = kRadixThreads / 64;
constexpr int kRadixBits = 10, kRadixSmallBits = 9;  // of a digit, at most (the small sort's LDS holds entries too)
constexpr int kRadixScanBlocks = 4096;               // workgroups at most
constexpr int kRadixSmall = 8 * kRadixThreads;       // entries of the one-launch sort, at most
constexpr int kRadixNext = 4096;                     // counts that a scatter keeps for the next pass, at most

// A range of 4-byte words that the first launch clears beside its own work,
// and up to one more word.
struct RadixClear {
  void* p = nullptr;
  int64_t bytes = 0;
  int* word = nullptr;
};

struct RadixPlan {
  int64_t N;
  int64_t tile;  // entries a workgroup, whole rounds of kRadixThreads * items
  int blocks, nbp, items, passes, bits;
  bool scan;  // many workgroups: their first places by a launch of its own
  bool next;  // scatters count for the next pass
  // Workspace in 4-byte words: two entry arrays, the counts (of every pass, if
  // a scatter makes the next one's), the digits' sums.
  int64_t ent, hist;
  int64_t words() const { return 2 * ent + (next ? passes : 1) * hist + (1 << kRadixBits); }
  // Which of the two entry arrays holds the result.
  int result() const { return (passes - 1) & 1; }
};

// nkeys: keys are below it.
inline RadixPlan radix_plan(int64_t N, int64_t nkeys) {
  RadixPlan p{};
  p.N = N;
  int key = 1;
  while (key < 31 && ((nkeys - 1) >> key) != 0) ++key;
  const int most = N <= kRadixSmall ? kRadixSmallBits : kRadixBits;
  p.passes = (key + most - 1) / most;
  p.bits = (key + p.passes - 1) / p.passes;
  // short rounds spread few entries over more CUs. Past 256 workgroups each
  // would read too many counts: a launch scans them first, and several
  // workgroups a CU take a round each (a pass over 4.2 M entries by 9 bits: 55
  // us, in 256 workgroups of four rounds 79; at 524288 entries the launch is
  // the dearer, 25 to 21)
  p.scan = N > 256 * 4 * kRadixThreads;
  p.items = p.scan ? 8 : 4;
  const int64_t round = (int64_t)p.items * kRadixThreads;
  p.tile = std::max<int64_t>(1, cdiv(N, kRadixScanBlocks * round)) * round;
  p.blocks = (int)std::max<int64_t>(1, cdiv(N, p.tile));
  p.nbp = (p.blocks + 3) & ~3;
  p.ent = (2 * N + 3) & ~int64_t(3);
  p.hist = (int64_t)p.nbp << p.bits;
  p.next = !p.scan && p.passes > 1 && p.hist <= kRadixNext && N > kRadixSmall;
  return p;
}

// Lanes of this wave with the same digit (among valid lanes).
__device__ inline uint64_t radix_peers(int d, int bits, bool valid) {
  uint64_t m = __ballot(valid);
  for (int b = 0; b < bits; ++b) {
    const bool one = (d >> b) & 1;
    const uint64_t on = __ballot(one);
    m &= one ? on : ~on;
  }
  return m;
}

// Ranks of a lane's entries among the wave's of the same digit so far, counted
// in cnt (the wave's, LDS).
template <int I>
__device__ inline void radix_rank(const int (&d)[I], const bool (&valid)[I], int bits, int* cnt,
                                  int (&rank)[I]) {
  const int lane = threadIdx.x & 63;
  const uint64_t below = (1ull << lane) - 1;
  int first[I], old[I];
#pragma unroll
  for (int u = 0; u < I; ++u) {
    const uint64_t m = radix_peers(d[u], bits, valid[u]);
    rank[u] = __popcll(m & below);
    first[u] = m ? __ffsll((unsigned long long)m) - 1 : 0;
    old[u] = 0;
    if (valid[u] && first[u] == lane) old[u] = atomicAdd(&cnt[d[u]], __popcll(m));
  }
#pragma unroll
  for (int u = 0; u < I; ++u) rank[u] += __shfl(old[u], first[u], 64);
}

// Inclusive sum over the workgroup's threads (kRadixThreads; part: kRadixWaves ints of LDS).
__device__ inline int radix_scan(int v, int* part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  if (lane == 63) part[wave] = x;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRadixWaves; ++w) x += w < wave ? part[w] : 0;
  return x;
}

__device__ inline void radix_clear(const RadixClear& c, int64_t block, int64_t blocks) {
  if (block == 0 && threadIdx.x == 0 && c.word) *c.word = 0;
  const int64_t n = c.bytes >> 4, at = block * kRadixThreads + threadIdx.x;
  for (int64_t i = at; i < n; i += blocks * kRadixThreads)
    reinterpret_cast<uint4*>(c.p)[i] = make_uint4(0, 0, 0, 0);
  if (at < (c.bytes & 15)) static_cast<uint8_t*>(c.p)[(n << 4) + at] = 0;
}

static __global__ void __launch_bounds__(kRadixThreads) radix_clear_kernel(RadixClear clear) {
  radix_clear(clear, blockIdx.x, gridDim.x);
}

template <typename Src>
__device__ inline int2 radix_entry(const Src& src, const int2* in, int64_t i) {
  return in ? in[i] : make_int2(src.key(i), (int)i);
}

// All passes in one workgroup (N <= kRadixSmall); workgroups past the first clear.
template <typename Src>
__global__ void __launch_bounds__(kRadixThreads)
radix_small_kernel(Src src, int N, int passes, int bits, int2* __restrict__ out, RadixClear clear) {
  constexpr int I = kRadixSmall / kRadixThreads;
  __shared__ int cnt[kRadixWaves << kRadixSmallBits];
  __shared__ int2 ent[kRadixSmall];
  __shared__ int part[kRadixWaves];
  if (gridDim.x == 1 || blockIdx.x > 0)
    radix_clear(clear, gridDim.x == 1 ? 0 : blockIdx.x - 1, max((int)gridDim.x - 1, 1));
  if (blockIdx.x > 0) return;
  const int R = 1 << bits, tid = threadIdx.x, wave = tid >> 6;
  // a wave's entries are contiguous, as few rounds of 64 as N needs
  const int per = (N + kRadixThreads - 1) / kRadixThreads, w0 = wave * per * 64 + (tid & 63);
  for (int p = 0; p < passes; ++p) {
    for (int i = tid; i < kRadixWaves * R; i += kRadixThreads) cnt[i] = 0;
    int2 e[I];
    int d[I], rank[I];
    bool valid[I];
#pragma unroll
    for (int u = 0; u < I; ++u) {
      const int i = w0 + u * 64;
      valid[u] = u < per && i < N;
      e[u] = !valid[u] ? make_int2(0, 0) : p ? ent[i] : make_int2(src.key(i), i);
      d[u] = (e[u].x >> (p * bits)) & (R - 1);
    }
    __syncthreads();  // counters cleared, entries read
    radix_rank<I>(d, valid, bits, cnt + wave * R, rank);
    __syncthreads();
    int total = 0;
    if (tid < R)
      for (int w = 0; w < kRadixWaves; ++w) total += cnt[w * R + tid];
    int run = radix_scan(total, part) - total;
    if (tid < R)
      for (int w = 0; w < kRadixWaves; ++w) {
        const int c = cnt[w * R + tid];
        cnt[w * R + tid] = run;
        run += c;
      }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < I; ++u)
      if (valid[u]) {
        const int at = cnt[wave * R + d[u]] + rank[u];
        if (p + 1 < passes) ent[at] = e[u];
        else out[at] = e[u];
      }
    __syncthreads();  // counters read, entries written
  }
}

// Digit counts of each workgroup's entries: hist [digit][nbp], and zeros in the
// zeros words behind it. Workgroups past the sort's clear.
template <typename Src>
__global__ void __launch_bounds__(kRadixThreads)
radix_count_kernel(Src src, const int2* __restrict__ in, RadixPlan p, int shift, int* __restrict__ hist,
                   int zeros, RadixClear clear) {
  __shared__ int cnt[1 << kRadixBits];
  if ((int)blockIdx.x >= p.blocks) {
    radix_clear(clear, blockIdx.x - p.blocks, gridDim.x - p.blocks);
    return;
  }
  const int R = 1 << p.bits;
  for (int d = threadIdx.x; d < R; d += kRadixThreads) cnt[d] = 0;
  for (int i = blockIdx.x * kRadixThreads + threadIdx.x; i < zeros; i += p.blocks * kRadixThreads)
    hist[p.hist + i] = 0;
  __syncthreads();
  const int64_t i0 = blockIdx.x * p.tile, i1 = min(p.N, i0 + p.tile);
  const int lane = threadIdx.x & 63;
  for (int64_t i = i0 + threadIdx.x - lane; i < i1; i += 4 * kRadixThreads) {  // whole waves
    int k[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t at = i + u * kRadixThreads + lane;
      k[u] = at < i1 ? radix_entry(src, in, at).x : -1;
    }
    // peers count once: after the first pass neighbours share their digits
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int d = (k[u] >> shift) & (R - 1);
      const uint64_t m = radix_peers(d, p.bits, k[u] >= 0);
      if (k[u] >= 0 && __ffsll((unsigned long long)m) - 1 == lane) atomicAdd(&cnt[d], __popcll(m));
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < R; d += kRadixThreads) hist[(int64_t)d * p.nbp + blockIdx.x] = cnt[d];
  if (blockIdx.x == 0)  // the padding that the 16-byte loads read
    for (int d = threadIdx.x; d < R; d += kRadixThreads)
      for (int b = p.blocks; b < p.nbp; ++b) hist[(int64_t)d * p.nbp + b] = 0;
}

// Counts [digit][nbp] to first places within the digit, a workgroup a digit;
// tot: the digit's entries.
static __global__ void __launch_bounds__(kRadixThreads)
radix_scan_kernel(int nbp, int* __restrict__ hist, int* __restrict__ tot) {
  __shared__ int part[2][kRadixWaves];
  int* h = hist + (int64_t)blockIdx.x * nbp;
  int run = 0;
  for (int b0 = 0, k = 0; b0 < nbp; b0 += kRadixThreads, k ^= 1) {
    const int b = b0 + threadIdx.x, c = b < nbp ? h[b] : 0;
    const int x = radix_scan(c, part[k]);
    if (b < nbp) h[b] = run + x - c;
#pragma unroll
    for (int w = 0; w < kRadixWaves; ++w) run += part[k][w];
  }
  if (threadIdx.x == 0) tot[blockIdx.x] = run;
}

// NEXT: the counts of the next pass's digits are added to next (a workgroup's
// entries are I * kRadixThreads).
template <typename Src, int I, bool NEXT>
__global__ void __launch_bounds__(kRadixThreads)
radix_scatter_kernel(Src src, const int2* __restrict__ in, RadixPlan p, int shift,
                     const int* __restrict__ hist, const int* __restrict__ sums, int2* __restrict__ out,
                     int* __restrict__ next) {
  __shared__ int cnt[kRadixWaves << kRadixBits];
  __shared__ int ahead[NEXT ? kRadixNext : 1];
  __shared__ int tot[1 << kRadixBits], base[1 << kRadixBits], part[kRadixWaves];
  const int R = 1 << p.bits, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int mine = blockIdx.x;
  const int64_t i0 = mine * p.tile, i1 = min(p.N, i0 + p.tile);
  int2 e[I];
  auto begin = [&](int64_t r0) {  // a round's entries on their way, its counters cleared
#pragma unroll
    for (int u = 0; u < I; ++u) {
      const int64_t i = r0 + (wave * I + u) * 64 + lane;
      e[u] = i < i1 ? radix_entry(src, in, i) : make_int2(0, 0);
    }
    for (int i = tid; i < kRadixWaves * R; i += kRadixThreads) cnt[i] = 0;
  };
  begin(i0);
  if constexpr (NEXT)
    for (int i = tid; i < (int)p.hist; i += kRadixThreads) ahead[i] = 0;
  if (p.scan) {
    for (int d = tid; d < R; d += kRadixThreads) {
      tot[d] = sums[d];
      base[d] = hist[(int64_t)d * p.nbp + mine];
    }
  } else {  // P neighbouring threads to a digit
    const int P = max(1, min(kRadixThreads >> p.bits, 64)), q = tid % P, nq = p.nbp >> 2;
    for (int d0 = 0; d0 < R; d0 += kRadixThreads / P) {  // every lane takes part in the sums
      const int d = d0 + tid / P;
      int total = 0, before = 0;
      if (d < R) {
        const int4* h = reinterpret_cast<const int4*>(hist + (int64_t)d * p.nbp);
        constexpr int U = 8;
        for (int j0 = q; j0 < nq; j0 += U * P) {
          int4 c[U];
#pragma unroll
          for (int u = 0; u < U; ++u) c[u] = h[min(j0 + u * P, nq - 1)];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int j = j0 + u * P;
            if (j < nq) {
              const int b = 4 * j;
              total += c[u].x + c[u].y + c[u].z + c[u].w;
              before += (b < mine ? c[u].x : 0) + (b + 1 < mine ? c[u].y : 0) + (b + 2 < mine ? c[u].z : 0) +
                        (b + 3 < mine ? c[u].w : 0);
            }
          }
        }
      }
      for (int s = 1; s < P; s <<= 1) {
        total += __shfl_xor(total, s, 64);
        before += __shfl_xor(before, s, 64);
      }
      if (d < R && q == 0) {
        tot[d] = total;
        base[d] = before;
      }
    }
  }
  __syncthreads();
  {  // a thread's neighbouring digits
    const int per = max(1, R / kRadixThreads), d0 = min(tid * per, R), d1 = min(d0 + per, R);
    int t = 0;
    for (int d = d0; d < d1; ++d) t += tot[d];
    int x = radix_scan(t, part) - t;
    for (int d = d0; d < d1; ++d) {
      base[d] += x;
      x += tot[d];
    }
  }
  for (int64_t r0 = i0; r0 < i1; r0 += I * kRadixThreads) {
    int d[I], rank[I];
    bool valid[I];
#pragma unroll
    for (int u = 0; u < I; ++u) {
      valid[u] = r0 + (wave * I + u) * 64 + lane < i1;
      d[u] = (e[u].x >> shift) & (R - 1);
    }
    radix_rank<I>(d, valid, p.bits, cnt + wave * R, rank);
    __syncthreads();
    for (int b = tid; b < R; b += kRadixThreads) {
      int run = base[b];
#pragma unroll
      for (int w = 0; w < kRadixWaves; ++w) {
        const int c = cnt[w * R + b];
        cnt[w * R + b] = run;
        run += c;
      }
      base[b] = run;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < I; ++u)
      if (valid[u]) {
        const int at = cnt[wave * R + d[u]] + rank[u];
        out[at] = e[u];
        if constexpr (NEXT)
          atomicAdd(&ahead[((e[u].x >> (shift + p.bits)) & (R - 1)) * p.nbp + at / (I * kRadixThreads)], 1);
      }
    __syncthreads();
    if (r0 + I * kRadixThreads < i1) {
      begin(r0 + I * kRadixThreads);
      __syncthreads();
    }
  }
  if constexpr (NEXT)
    for (int i = tid; i < (int)p.hist; i += kRadixThreads)
      if (ahead[i]) atomicAdd(&next[i], ahead[i]);
}

// Sorts N > 0 entries; ws: plan.words() words at a multiple of 16 bytes. The
// result is ws + result() * ent words, as int2 (key, index).
template <typename Src>
inline const int2* radix_sort(const Src& src, const RadixPlan& p, int* ws, const RadixClear& clear,
                              hipStream_t st) {
  int2* ent[2] = {reinterpret_cast<int2*>(ws), reinterpret_cast<int2*>(ws + p.ent)};
  int *hist = ws + 2 * p.ent, *sums = hist + (p.next ? p.passes : 1) * p.hist;
  const int extra = (int)std::min<int64_t>(cdiv(clear.bytes, 16 * kRadixThreads), 2048);
  if (p.N <= kRadixSmall) {
    hipLaunchKernelGGL((radix_small_kernel<Src>), dim3(1 + extra), dim3(kRadixThreads), 0, st, src, (int)p.N,
                       p.passes, p.bits, ent[p.result()], clear);
    return ent[p.result()];
  }
  const int2* in = nullptr;
  for (int k = 0, shift = 0; k < p.passes; ++k, shift += p.bits) {
    const RadixClear c = k == 0 ? clear : RadixClear{};
    if (k == 0 || !p.next)
      hipLaunchKernelGGL((radix_count_kernel<Src>),
                         dim3(p.blocks + (k == 0 ? std::max(extra, clear.word ? 1 : 0) : 0)), dim3(kRadixThreads), 0,
                         st, src, in, p, shift, hist, p.next ? (int)((p.passes - 1) * p.hist) : 0, c);
    if (p.scan)
      hipLaunchKernelGGL(radix_scan_kernel, dim3(1 << p.bits), dim3(kRadixThreads), 0, st, p.nbp, hist, sums);
    auto scatter = p.items != 4                    ? radix_scatter_kernel<Src, 8, false>
                   : p.next && k + 1 < p.passes ? radix_scatter_kernel<Src, 4, true>
                                                : radix_scatter_kernel<Src, 4, false>;
    hipLaunchKernelGGL(scatter, dim3(p.blocks), dim3(kRadixThreads), 0, st, src, in, p, shift, hist, sums, ent[k & 1],
                       hist + p.hist);
    if (p.next) hist += p.hist;
    in = ent[k & 1];
  }
  return in;
}

}  // namespace slg
