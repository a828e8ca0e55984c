// Activations in 8 bits (rows8.hip): what a layer keeps of its input between
// the forward and the backward.
//   codes [ceil(B / 4)][ld] uint32: byte v of word (t, i) is the code of
//         sample 4 t + v, input i (0 past the batch and past the row);
//   rows  [B][2] float: a sample's offset lo and step; a code stands for
//         lo + code * step.
#pragma once
#include "slg_common.h"

namespace slg {

constexpr int kRows8Tile = 4;  // samples a word

// Words from one tile's row to the next: whole quads, so that every row
// starts at a multiple of 16 bytes.
inline int64_t rows8_ld(int64_t D) { return (D + 3) & ~int64_t(3); }

// A row's range; a value that is not finite makes `odd` NaN.
struct Rows8Range {
  float lo = INFINITY, hi = -INFINITY, odd = 0.0f;
  __device__ void take(float v) {
    lo = fminf(lo, v);
    hi = fmaxf(hi, v);
    odd = fmaf(v, 0.0f, odd);
  }
  // Over the wave, as two values: hi = infinity where the row is not finite.
  __device__ void wave() {
    if (!(odd == 0.0f)) hi = INFINITY;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      lo = fminf(lo, __shfl_xor(lo, d, 64));
      hi = fmaxf(hi, __shfl_xor(hi, d, 64));
    }
  }
};

// Offset, step and reciprocal step of a row with range lo..hi.
__device__ inline void rows8_scale(float lo, float hi, float& lo_out, float& step, float& inv) {
  const float span = hi - lo;
  const bool bad = !(span <= 3.402823466e38f);  // not finite, or a span that is not
  inv = 255.0f / span;
  step = span / 255.0f;
  if (!(span > 0.0f) || !(inv <= 3.402823466e38f) || bad) inv = step = 0.0f;
  lo_out = bad ? __int_as_float(0x7fc00000) : lo;
}

// `word` with byte v set to x's code. (x - lo) * inv is at most 255 (1 + 2^-23)
// and rounds to a code; the conversion truncates a whole number.
__device__ inline uint32_t rows8_code(uint32_t word, int v, float x, float lo, float inv) {
  const float q = rintf((x - lo) * inv);
  // inv = 0: a constant or not finite row, code 0
  return __builtin_amdgcn_cvt_pk_u8_f32(inv > 0.0f ? q : 0.0f, v, word);
}

// Where a forward kernel puts the codes and rows of its input (codes null: nowhere).
struct Rows8Out {
  uint32_t* codes;
  float* rows;
  int ld;
};

// LDS floats that rows8_pack_tile takes for S samples and W waves.
constexpr int rows8_scratch(int S, int W) { return 2 * S * W; }

// Codes and rows of the S samples from b0 on (S and b0 multiples of 4) that a
// workgroup has in LDS, transposed: tile[g * IN + i] holds samples b0 + 4 g ..
// of input i.
template <int S, typename V4>
__device__ inline void rows8_pack_tile(const V4* tile, int IN, int b0, int B, float* scratch, const Rows8Out& o) {
  constexpr int G = S / kRows8Tile;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, W = blockDim.x >> 6, T = blockDim.x;
  Rows8Range r[S];
  constexpr int U = 8 / G;  // reads in flight
  for (int i0 = tid; i0 < IN; i0 += U * T) {
    V4 v[U][G];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int g = 0; g < G; ++g) v[u][g] = tile[g * IN + min(i0 + u * T, IN - 1)];  // past the row: its last
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int s = 0; s < S; ++s) r[s].take(v[u][s / 4][s % 4]);
  }
#pragma unroll
  for (int s = 0; s < S; ++s) {
    r[s].wave();
    if (lane == 0) {
      scratch[2 * (wave * S + s)] = r[s].lo;
      scratch[2 * (wave * S + s) + 1] = r[s].hi;
    }
  }
  __syncthreads();
  float lo[S], inv[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    float a = INFINITY, z = -INFINITY, step;
    for (int w = 0; w < W; ++w) {
      a = fminf(a, scratch[2 * (w * S + s)]);
      z = fmaxf(z, scratch[2 * (w * S + s) + 1]);
    }
    rows8_scale(a, z, lo[s], step, inv[s]);
    if (b0 + s >= B) {
      inv[s] = 0.0f;
    } else if (tid == 0) {
      o.rows[2 * (int64_t)(b0 + s)] = lo[s];
      o.rows[2 * (int64_t)(b0 + s) + 1] = step;
    }
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
    if (b0 + 4 * g >= B) break;
    uint32_t* c = o.codes + ((int64_t)(b0 / 4) + g) * o.ld;
    for (int i0 = tid; i0 < IN; i0 += 4 * T) {
      V4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = tile[g * IN + min(i0 + u * T, IN - 1)];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) w = rows8_code(w, e, v[u][e], lo[4 * g + e], inv[4 * g + e]);
        if (i0 + u * T < IN) c[i0 + u * T] = w;
      }
    }
    if (tid < o.ld - IN) c[IN + tid] = 0u;
  }
}

// slg_rows8_pack's launch.
void rows8_pack(const float* x, int64_t B, int64_t D, uint32_t* codes, float* rows, hipStream_t st);

}  // namespace slg
