// Rows of activations in 8 bits and back (rows8.h has the layout):
//   lo = min_i x_i, step = (max_i x_i - lo) / 255,
//   code_i = rint((x_i - lo) * (255 / (max - lo))),
// in fp32 with IEEE division, so the codes are defined to the bit. A row of
// equal values (or one so narrow that 255 / span overflows) has codes 0 and
// step 0, exact to within its span. Soft activations of a sample share one
// range; a sample's own lo and step use all 256 codes of it (deep layers
// crowd around 1/2), and rows of bits {0, 1} come back exactly. A value off by
// at most half a step: (max - min) / 510. A row that holds an infinity or a
// NaN, or whose span overflows, has lo = NaN: it comes back as NaN everywhere
// rather than as finite values that were not there.
//
// Both ways are bound by memory: 5 bytes a value. 4096 x 16380 (335 MB): packed
// in 74 us (4.6 TB/s; a copy of as much takes 71), unpacked in 54 (6.2 TB/s).
#include <algorithm>

#include "rows8.h"

namespace slg {

constexpr int64_t kRows8Grid = 1 << 20;  // workgroups at most; the rest in turn

// VU neighbouring values or words as one access, from any multiple of 4 bytes
// (aligned ones are as fast), so that odd widths take 16 bytes too: a row's
// last run is moved back to end with the row, the values that two threads then
// hold come out the same from both.
template <typename E, int VU>
struct Rows8Run {
  typedef E t __attribute__((ext_vector_type(VU), aligned(4)));
};
template <int VU>
__device__ inline void rows8_load(const float* __restrict__ p, float (&v)[VU]) {
  using R = typename Rows8Run<float, VU>::t;
  const R r = *reinterpret_cast<const R*>(p);
#pragma unroll
  for (int j = 0; j < VU; ++j) v[j] = VU == 1 ? ((const float*)&r)[0] : r[j];
}
template <typename E, int VU>
__device__ inline void rows8_store(E* __restrict__ p, const E (&v)[VU]) {
  using R = typename Rows8Run<E, VU>::t;
  R r;
#pragma unroll
  for (int j = 0; j < VU; ++j) r[j] = v[j];
  *reinterpret_cast<R*>(p) = r;
}

// One workgroup per tile of 4 samples. NU > 0: the tile's values stay in
// registers between the range and the codes (NU runs of VU inputs of each row
// a thread, D <= NU * VU * T); NU = 0: they are read again. D >= VU.
template <int NU, int VU, int T>
__global__ void __launch_bounds__(T)
rows8_pack_kernel(const float* __restrict__ x, int64_t B, int D, int ld, uint32_t* __restrict__ codes,
                  float* __restrict__ rows) {
  struct Ends { float lo, hi; };
  __shared__ Ends part[T / 64][kRows8Tile];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int64_t t = blockIdx.x; t * kRows8Tile < B; t += gridDim.x) {
    const int64_t b0 = t * kRows8Tile;
    const int nb = (int)min((int64_t)kRows8Tile, B - b0);
    const float* p[kRows8Tile];
#pragma unroll
    for (int v = 0; v < kRows8Tile; ++v) p[v] = x + min(b0 + v, B - 1) * D;  // past the batch: its last row
    Rows8Range r[kRows8Tile];
    float keep[NU > 0 ? NU : 1][kRows8Tile][VU];
    if constexpr (NU > 0) {
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const int i = min((tid + u * T) * VU, D - VU);  // past the row: its last values
#pragma unroll
        for (int v = 0; v < kRows8Tile; ++v) rows8_load<VU>(p[v] + i, keep[u][v]);
      }
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int v = 0; v < kRows8Tile; ++v)
#pragma unroll
          for (int j = 0; j < VU; ++j) r[v].take(keep[u][v][j]);
    } else {
      for (int i = tid * VU; i < D; i += T * VU)
#pragma unroll
        for (int v = 0; v < kRows8Tile; ++v) {
          rows8_load<VU>(p[v] + min(i, D - VU), keep[0][v]);
#pragma unroll
          for (int j = 0; j < VU; ++j) r[v].take(keep[0][v][j]);
        }
    }
#pragma unroll
    for (int v = 0; v < kRows8Tile; ++v) {
      r[v].wave();
      if (lane == 0) part[wave][v] = {r[v].lo, r[v].hi};
    }
    __syncthreads();
    float lo[kRows8Tile], inv[kRows8Tile];
#pragma unroll
    for (int v = 0; v < kRows8Tile; ++v) {
      Ends a = part[0][v];
#pragma unroll
      for (int w = 1; w < T / 64; ++w) {
        a.lo = fminf(a.lo, part[w][v].lo);
        a.hi = fmaxf(a.hi, part[w][v].hi);
      }
      float step;
      rows8_scale(a.lo, a.hi, lo[v], step, inv[v]);
      if (tid == 0 && v < nb) {
        rows[2 * (b0 + v)] = lo[v];
        rows[2 * (b0 + v) + 1] = step;
      }
      if (v >= nb) inv[v] = 0.0f;  // codes 0 past the batch
    }
    uint32_t* c = codes + t * ld;
    auto put = [&](int i, const float (&e)[kRows8Tile][VU]) {
      uint32_t w[VU];
#pragma unroll
      for (int j = 0; j < VU; ++j) {
        w[j] = 0;
#pragma unroll
        for (int v = 0; v < kRows8Tile; ++v) w[j] = rows8_code(w[j], v, e[v][j], lo[v], inv[v]);
      }
      rows8_store<uint32_t, VU>(c + i, w);
    };
    if constexpr (NU > 0) {
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const int i = (tid + u * T) * VU;
        if (i < D) put(min(i, D - VU), keep[u]);
      }
    } else {
      for (int k = tid * VU; k < D; k += T * VU) {
        const int i = min(k, D - VU);
#pragma unroll
        for (int v = 0; v < kRows8Tile; ++v) rows8_load<VU>(p[v] + i, keep[0][v]);
        put(i, keep[0]);
      }
    }
    if (tid < ld - D) c[D + tid] = 0u;
    __syncthreads();  // part is written again
  }
}

// Rows too wide for that: the tile's four rows one after the other, NU runs of
// 4 of one row a thread, while their codes gather in as many words (D <= 4096 *
// NU; 1024 threads). The next row's values are on their way as soon as the last
// one's are coded (behind the tile's last row that row again, from the caches,
// unused). 2048 x 32000: 73 us, with every value read twice 104 (1500 x
// 40960: 72 and 99; 64 x 20000: 10.1 and 9.5).
template <int NU>
__global__ void __launch_bounds__(1024)
rows8_pack_wide_kernel(const float* __restrict__ x, int64_t B, int D, int ld, uint32_t* __restrict__ codes,
                       float* __restrict__ rows) {
  constexpr int T = 1024, VU = 4, W = T / 64;
  struct Ends { float lo, hi; };
  __shared__ Ends part[2][W];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  float e[NU][VU];
  auto load = [&](const float* p, int u) { rows8_load<VU>(p + min((tid + u * T) * VU, D - VU), e[u]); };
  for (int64_t t = blockIdx.x; t * kRows8Tile < B; t += gridDim.x) {
    const int64_t b0 = t * kRows8Tile;
    const int nb = (int)min((int64_t)kRows8Tile, B - b0);
    uint32_t w[NU][VU];
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      load(x + b0 * D, u);
#pragma unroll
      for (int j = 0; j < VU; ++j) w[u][j] = 0;
    }
    for (int v = 0; v < nb; ++v) {
      Rows8Range r;
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int j = 0; j < VU; ++j) r.take(e[u][j]);
      r.wave();
      if (lane == 0) part[v & 1][wave] = {r.lo, r.hi};
      __syncthreads();  // part[v & 1] is written again two rows on, past the next one's
      Ends a = part[v & 1][0];
#pragma unroll
      for (int k = 1; k < W; ++k) {
        a.lo = fminf(a.lo, part[v & 1][k].lo);
        a.hi = fmaxf(a.hi, part[v & 1][k].hi);
      }
      float lo, step, inv;
      rows8_scale(a.lo, a.hi, lo, step, inv);
      if (tid == 0) {
        rows[2 * (b0 + v)] = lo;
        rows[2 * (b0 + v) + 1] = step;
      }
      const float* next = x + (b0 + min(v + 1, nb - 1)) * D;
#pragma unroll
      for (int u = 0; u < NU; ++u) {
#pragma unroll
        for (int j = 0; j < VU; ++j) w[u][j] |= rows8_code(0, 0, e[u][j], lo, inv) << (8 * v);
        load(next, u);
      }
    }
    uint32_t* c = codes + t * ld;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int i = (tid + u * T) * VU;
      if (i < D) rows8_store<uint32_t, VU>(c + min(i, D - VU), w[u]);
    }
    if (tid < ld - D) c[D + tid] = 0u;
  }
}

// Values that the codes stand for: a thread takes VU neighbouring words and
// writes four rows of them.
template <int VU>
__global__ void __launch_bounds__(256)
rows8_unpack_kernel(const uint32_t* __restrict__ codes, const float* __restrict__ rows, int64_t B, int D,
                    int ld, int per_tile, int64_t blocks, float* __restrict__ x) {
  using W = typename Rows8Run<uint32_t, VU>::t;
  for (int64_t k = blockIdx.x; k < blocks; k += gridDim.x) {
    const int64_t t = k / per_tile;
    const int i0 = ((int)(k - t * per_tile) * 256 + threadIdx.x) * VU, i = min(i0, D - VU);
    if (i0 >= D) continue;
    const W r = *reinterpret_cast<const W*>(codes + t * ld + i);
    uint32_t w[VU];
#pragma unroll
    for (int j = 0; j < VU; ++j) w[j] = VU == 1 ? ((const uint32_t*)&r)[0] : r[j];
#pragma unroll
    for (int v = 0; v < kRows8Tile; ++v) {
      const int64_t b = t * kRows8Tile + v;
      if (b >= B) break;
      const float lo = rows[2 * b], step = rows[2 * b + 1];
      float e[VU];
#pragma unroll
      for (int j = 0; j < VU; ++j) e[j] = fmaf((float)((w[j] >> (8 * v)) & 255u), step, lo);
      rows8_store<float, VU>(x + b * D + i, e);
    }
  }
}

template <int NU, int VU, int T>
static void launch_pack(const float* x, int64_t B, int64_t D, uint32_t* codes, float* rows, hipStream_t st) {
  hipLaunchKernelGGL((rows8_pack_kernel<NU, VU, T>),
                     dim3((unsigned)std::min<int64_t>(cdiv(B, kRows8Tile), kRows8Grid)), dim3(T), 0, st, x, B,
                     (int)D, (int)rows8_ld(D), codes, rows);
}

template <int NU>
static void launch_pack_wide(const float* x, int64_t B, int64_t D, uint32_t* codes, float* rows, hipStream_t st) {
  hipLaunchKernelGGL((rows8_pack_wide_kernel<NU>), dim3((unsigned)std::min<int64_t>(cdiv(B, kRows8Tile), kRows8Grid)),
                     dim3(1024), 0, st, x, B, (int)D, (int)rows8_ld(D), codes, rows);
}

// The fewest threads that hold a tile in 16 values of each row a thread (32
// for the widest): fewer, longer threads have less of the range's sums over
// lanes and waves to do. Measured (us; threads x values a thread):
//   65536 x 256     64 x 4   15.7   256 x 4    44    read again by 64    21
//   32768 x 1000    64 x 16  26.2   256 x 4    27.5  read again by 256   38
//   16384 x 2000   256 x 8   26.3  1024 x 4    67    read again by 256   42
//   8192 x 4001    256 x 16  26.1  1024 x 4    39    read again by 256   43
//   4096 x 8001    512 x 16  26.6  1024 x 8    29    read again by 512   43
//   4096 x 16380   512 x 32  68.7  1024 x 16   72    read again by 1024  85
// Wider rows go row by row, and those past 40960 (what a workgroup's registers
// hold) are read again.
void rows8_pack(const float* x, int64_t B, int64_t D, uint32_t* codes, float* rows, hipStream_t st) {
  if (D < 4) launch_pack<1, 1, 64>(x, B, D, codes, rows, st);
  else if (D <= 256) launch_pack<1, 4, 64>(x, B, D, codes, rows, st);
  else if (D <= 512) launch_pack<2, 4, 64>(x, B, D, codes, rows, st);
  else if (D <= 1024) launch_pack<4, 4, 64>(x, B, D, codes, rows, st);
  else if (D <= 2048) launch_pack<2, 4, 256>(x, B, D, codes, rows, st);
  else if (D <= 4096) launch_pack<4, 4, 256>(x, B, D, codes, rows, st);
  else if (D <= 8192) launch_pack<4, 4, 512>(x, B, D, codes, rows, st);
  else if (D <= 16384) launch_pack<8, 4, 512>(x, B, D, codes, rows, st);
  else if (D <= 24576) launch_pack_wide<6>(x, B, D, codes, rows, st);
  else if (D <= 32768) launch_pack_wide<8>(x, B, D, codes, rows, st);
  else if (D <= 40960) launch_pack_wide<10>(x, B, D, codes, rows, st);
  else launch_pack<0, 4, 512>(x, B, D, codes, rows, st);
}

}  // namespace slg

using namespace slg;

extern "C" {

int64_t slg_rows8_ld(int64_t D) { return rows8_ld(D); }

int slg_rows8_pack(const float* x, int64_t B, int64_t D, uint8_t* codes, float* rows, slg_stream_t stream) {
  SLG_REQUIRE((x && codes && rows) || B == 0, SLG_E_ARG, "rows8_pack: null pointer");
  SLG_REQUIRE(B >= 0 && D > 0 && D < (1LL << 28) && B < (1LL << 31) && B * D < (1LL << 40), SLG_E_SHAPE,
              "rows8_pack: B %lld, D %lld", (long long)B, (long long)D);
  SLG_REQUIRE((uintptr_t)codes % 16 == 0, SLG_E_ARG, "rows8_pack: codes not at a multiple of 16 bytes");
  if (B == 0) return 0;
  rows8_pack(x, B, D, reinterpret_cast<uint32_t*>(codes), rows, as_stream(stream));
  SLG_LAUNCH_CHECK("rows8_pack");
  return 0;
}

int slg_rows8_unpack(const uint8_t* codes, const float* rows, int64_t B, int64_t D, float* x,
                     slg_stream_t stream) {
  SLG_REQUIRE((x && codes && rows) || B == 0, SLG_E_ARG, "rows8_unpack: null pointer");
  SLG_REQUIRE(B >= 0 && D > 0 && D < (1LL << 28) && B < (1LL << 31) && B * D < (1LL << 40), SLG_E_SHAPE,
              "rows8_unpack: B %lld, D %lld", (long long)B, (long long)D);
  SLG_REQUIRE((uintptr_t)codes % 16 == 0, SLG_E_ARG, "rows8_unpack: codes not at a multiple of 16 bytes");
  if (B == 0) return 0;
  const bool vec = D >= 4;
  const int64_t per = cdiv(D, vec ? 1024 : 256), blocks = cdiv(B, kRows8Tile) * per;
  hipLaunchKernelGGL(vec ? rows8_unpack_kernel<4> : rows8_unpack_kernel<1>,
                     dim3((unsigned)std::min(blocks, kRows8Grid)), dim3(256), 0, as_stream(stream),
                     reinterpret_cast<const uint32_t*>(codes), rows, B, (int)D, (int)rows8_ld(D), (int)per, blocks,
                     x);
  SLG_LAUNCH_CHECK("rows8_unpack");
  return 0;
}

}  // extern "C"
