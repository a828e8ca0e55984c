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
#include <algorithm>

#include "rows8.h"

namespace slg {

constexpr int64_t kRows8Grid = 1 << 20;  // workgroups at most; the rest in turn

// VU neighbouring values or words as one access.
template <int VU>
__device__ inline void rows8_load(const float* __restrict__ p, float (&v)[VU]) {
  if constexpr (VU == 4) {
    const float4 r = *reinterpret_cast<const float4*>(p);
    v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
  } else {
    v[0] = *p;
  }
}

// One workgroup per tile of 4 samples. NU > 0: the tile's values stay in
// registers between the range and the codes (NU runs of VU inputs of each row
// a thread, D <= NU * VU * T); NU = 0: they are read again. VU = 4: D a
// multiple of 4 and x at one of 16 bytes.
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
    for (int v = 0; v < kRows8Tile; ++v) p[v] = x + (b0 + min(v, nb - 1)) * D;  // past the batch: its last row
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
          rows8_load<VU>(p[v] + i, keep[0][v]);
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
      if constexpr (VU == 4) *reinterpret_cast<uint4*>(c + i) = make_uint4(w[0], w[1], w[2], w[3]);
      else c[i] = w[0];
    };
    if constexpr (NU > 0) {
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const int i = (tid + u * T) * VU;
        if (i < D) put(i, keep[u]);
      }
    } else {
      for (int i = tid * VU; i < D; i += T * VU) {
#pragma unroll
        for (int v = 0; v < kRows8Tile; ++v) rows8_load<VU>(p[v] + i, keep[0][v]);
        put(i, keep[0]);
      }
    }
    if (tid < ld - D) c[D + tid] = 0u;
    __syncthreads();  // part is written again
  }
}

// Values that the codes stand for: a thread takes VU neighbouring words and
// writes four rows of them (VU = 4: as above).
template <int VU>
__global__ void __launch_bounds__(256)
rows8_unpack_kernel(const uint32_t* __restrict__ codes, const float* __restrict__ rows, int64_t B, int D,
                    int ld, int per_tile, int64_t blocks, float* __restrict__ x) {
  for (int64_t k = blockIdx.x; k < blocks; k += gridDim.x) {
    const int64_t t = k / per_tile;
    const int i = ((int)(k - t * per_tile) * 256 + threadIdx.x) * VU;
    if (i >= D) continue;
    uint32_t w[VU];
    if constexpr (VU == 4) {
      const uint4 r = *reinterpret_cast<const uint4*>(codes + t * ld + i);
      w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w;
    } else {
      w[0] = codes[t * ld + i];
    }
#pragma unroll
    for (int v = 0; v < kRows8Tile; ++v) {
      const int64_t b = t * kRows8Tile + v;
      if (b >= B) break;
      const float lo = rows[2 * b], step = rows[2 * b + 1];
      float e[VU];
#pragma unroll
      for (int j = 0; j < VU; ++j) e[j] = fmaf((float)((w[j] >> (8 * v)) & 255u), step, lo);
      if constexpr (VU == 4) *reinterpret_cast<float4*>(x + b * D + i) = make_float4(e[0], e[1], e[2], e[3]);
      else x[b * D + i] = e[0];
    }
  }
}

template <int NU, int VU, int T>
static void launch_pack(const float* x, int64_t B, int64_t D, uint32_t* codes, float* rows, hipStream_t st) {
  hipLaunchKernelGGL((rows8_pack_kernel<NU, VU, T>),
                     dim3((unsigned)std::min<int64_t>(cdiv(B, kRows8Tile), kRows8Grid)), dim3(T), 0, st, x, B,
                     (int)D, (int)rows8_ld(D), codes, rows);
}

// Workgroups that hold a tile in registers: 16 values of each row a thread at
// most.
template <int VU>
static void launch_pack_v(const float* x, int64_t B, int64_t D, uint32_t* codes, float* rows, hipStream_t st) {
  constexpr int Q = 4 / VU;  // runs that make 4 values
  if (D <= 256 * VU) launch_pack<1, VU, 256>(x, B, D, codes, rows, st);
  else if (D <= 4096 && Q * VU * 256 >= D) launch_pack<Q, VU, 256>(x, B, D, codes, rows, st);
  else if (D <= 4096) launch_pack<Q, VU, 1024>(x, B, D, codes, rows, st);
  else if (D <= 8192) launch_pack<2 * Q, VU, 1024>(x, B, D, codes, rows, st);
  else if (D <= 16384) launch_pack<4 * Q, VU, 1024>(x, B, D, codes, rows, st);
  else launch_pack<0, VU, 1024>(x, B, D, codes, rows, st);
}

static bool rows8_vector(const float* x, int64_t D) { return D % 4 == 0 && (uintptr_t)x % 16 == 0; }

void rows8_pack(const float* x, int64_t B, int64_t D, uint32_t* codes, float* rows, hipStream_t st) {
  if (rows8_vector(x, D)) launch_pack_v<4>(x, B, D, codes, rows, st);
  else launch_pack_v<1>(x, B, D, codes, rows, st);
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
  const bool vec = rows8_vector(x, D);
  const int64_t per = cdiv(D, vec ? 1024 : 256), blocks = cdiv(B, kRows8Tile) * per;
  hipLaunchKernelGGL(vec ? rows8_unpack_kernel<4> : rows8_unpack_kernel<1>,
                     dim3((unsigned)std::min(blocks, kRows8Grid)), dim3(256), 0, as_stream(stream),
                     reinterpret_cast<const uint32_t*>(codes), rows, B, (int)D, (int)rows8_ld(D), (int)per, blocks,
                     x);
  SLG_LAUNCH_CHECK("rows8_unpack");
  return 0;
}

}  // extern "C"
