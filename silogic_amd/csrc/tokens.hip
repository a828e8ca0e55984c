// Token encoder for gfx950: a learned row of D soft bits per token id.
//   soft   y[n, d] = sigmoid(scale * E[t_n, d]) (ste: 1 where E > 0, else 0)
//   hard   bit (n, d) = E[t_n, d] > 0, the soft form past 1/2
//   back   gE[v, d] = scale * sigmoid'(scale * E[v, d]) * sum over n with t_n = v of gy[n, d]
// A token that is the padding id, or that no row of the table has (negative,
// or V and above), is absent: its values and bits are 0 and it adds to no
// gradient. The derivative depends on the table's entry alone, so it stays
// outside the sum: the backward reads gy once and neither y nor the table per
// token.
//
// Tables are fp32, bf16 or fp16 (rounded once, on the gradient's write);
// values, sums and gy are fp32.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>

#include "slg_common.h"

namespace slg {

enum { kTabF32 = 0, kTabBf16 = 1, kTabF16 = 2 };

template <int DT> struct TabType;
template <> struct TabType<kTabF32> { using t = float; };
template <> struct TabType<kTabBf16> { using t = uint16_t; };
template <> struct TabType<kTabF16> { using t = _Float16; };

template <int DT>
__device__ inline float tab_get(typename TabType<DT>::t v) {
  if constexpr (DT == kTabBf16) return __uint_as_float((uint32_t)v << 16);
  else return (float)v;
}

// Round to nearest even; a NaN stays one.
template <int DT>
__device__ inline typename TabType<DT>::t tab_put(float v) {
  if constexpr (DT == kTabBf16) {
    const uint32_t u = __float_as_uint(v);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
  } else {
    return (typename TabType<DT>::t)v;
  }
}

// The row of token n, or V where it is absent.
template <typename IdT>
__device__ inline int tok_row(const IdT* __restrict__ ids, int64_t n, int V, int64_t pad) {
  const int64_t t = (int64_t)ids[n];
  return (t >= 0 && t < V && t != pad) ? (int)t : V;
}

__device__ inline float tok_value(float e, float scale, bool ste) {
  if (ste) return e > 0.0f ? 1.0f : 0.0f;
  return 1.0f / (1.0f + expf(-scale * e));
}

// scale * sigmoid'(scale e), from exp(-|z|): no difference of values near 1.
__device__ inline float tok_slope(float e, float scale) {
  const float t = expf(-fabsf(scale * e)), u = 1.0f + t;
  return scale * (t / (u * u));
}

// One thread per unit of VU values of one token (D a multiple of VU).
template <int DT, typename IdT, int VU>
__global__ void __launch_bounds__(256)
tok_encode_kernel(const IdT* __restrict__ ids, int64_t units, int upr, int V, int64_t pad,
                  const typename TabType<DT>::t* __restrict__ tab, float scale, int ste, float* __restrict__ y) {
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < units; u += (int64_t)gridDim.x * 256) {
    const int64_t n = u / upr;
    const int c = (int)(u - n * upr);
    const int r = tok_row(ids, n, V, pad);
#pragma unroll
    for (int j = 0; j < VU; ++j) {
      const float e = r < V ? tab_get<DT>(tab[((int64_t)r * upr + c) * VU + j]) : 0.0f;
      y[u * VU + j] = r < V ? tok_value(e, scale, ste != 0) : 0.0f;
    }
  }
}

// ---------------------------------------------------------------------------
// Sorting tokens: entries (row, token) in ascending rows, tokens of one row in
// ascending order (a stable least-significant-digit radix sort), so that every
// sum has one order. Absent tokens (row V) come last.
// ---------------------------------------------------------------------------
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kSortBlocks = 128;      // workgroups at most: each reads every one's counts
constexpr int kSortMinTile = 4096;    // entries a workgroup at least
constexpr int kSortMaxBits = 9;       // digits of at most 512 values: 32 KB of counts in LDS

struct SortArgs {
  int64_t N;
  int64_t tile;        // entries a workgroup (a multiple of 1024)
  int V;
  int64_t pad;
  int shift, bits;
};

template <typename IdT>
__device__ inline int2 sort_entry(const IdT* ids, const int2* in, int64_t i, const SortArgs& a) {
  return in ? in[i] : make_int2(tok_row(ids, i, a.V, a.pad), (int)i);
}

// Lanes of this wave with the same digit (among valid lanes).
__device__ inline uint64_t same_digit(int d, int bits, bool valid) {
  uint64_t m = __ballot(valid);
  for (int b = 0; b < bits; ++b) {
    const uint64_t on = __ballot((d >> b) & 1);
    m &= (d >> b) & 1 ? on : ~on;
  }
  return m;
}

// Digit counts of each workgroup's entries: hist [workgroup][1 << bits].
template <typename IdT>
__global__ void __launch_bounds__(kSortThreads)
tok_hist_kernel(SortArgs a, const IdT* __restrict__ ids, const int2* __restrict__ in, int* __restrict__ hist) {
  __shared__ int cnt[1 << kSortMaxBits];
  const int R = 1 << a.bits;
  for (int d = threadIdx.x; d < R; d += kSortThreads) cnt[d] = 0;
  __syncthreads();
  const int64_t i0 = blockIdx.x * a.tile, i1 = min(a.N, i0 + a.tile);
  for (int64_t i = i0 + threadIdx.x; i < i1; i += kSortThreads)
    atomicAdd(&cnt[(sort_entry(ids, in, i, a).x >> a.shift) & (R - 1)], 1);
  __syncthreads();
  for (int d = threadIdx.x; d < R; d += kSortThreads) hist[(int64_t)blockIdx.x * R + d] = cnt[d];
}

// One pass: each workgroup's entries to their places. A wave takes a
// contiguous part of the tile in order, 64 entries at a time.
template <typename IdT>
__global__ void __launch_bounds__(kSortThreads)
tok_scatter_kernel(SortArgs a, const IdT* __restrict__ ids, const int2* __restrict__ in,
                   const int* __restrict__ hist, int2* __restrict__ out) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int R = 1 << a.bits;
  volatile int* cnt = reinterpret_cast<int*>(smem);  // [waves][R]
  __shared__ int scan[kSortWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int d = tid; d < kSortWaves * R; d += kSortThreads) cnt[d] = 0;
  __syncthreads();
  const int64_t i0 = blockIdx.x * a.tile, i1 = min(a.N, i0 + a.tile);
  const int64_t w0 = i0 + wave * (a.tile / kSortWaves), w1 = min(i1, w0 + a.tile / kSortWaves);
  volatile int* mine = cnt + wave * R;
  const uint64_t below = (1ull << lane) - 1;
  for (int64_t i = w0; i < w1; i += 64) {  // this wave's counts
    const bool valid = i + lane < w1;
    const int d = valid ? (sort_entry(ids, in, i + lane, a).x >> a.shift) & (R - 1) : 0;
    const uint64_t m = same_digit(d, a.bits, valid);
    if (valid && (m & below) == 0) mine[d] += __popcll(m);
  }
  __syncthreads();
  // digit d's first place: all smaller digits, then earlier workgroups'
  // entries of d, then earlier waves'
  int total = 0, before = 0;
  if (tid < R) {
    for (int g = 0; g < (int)gridDim.x; ++g) {
      const int c = hist[(int64_t)g * R + tid];
      total += c;
      before += g < (int)blockIdx.x ? c : 0;
    }
  }
  int x = total;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  if (lane == 63) scan[wave] = x;
  __syncthreads();
  int base = x - total + before;
  for (int w = 0; w < wave; ++w) base += scan[w];
  if (tid < R) {
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = cnt[w * R + tid];
      cnt[w * R + tid] = base;
      base += c;
    }
  }
  __syncthreads();
  for (int64_t i = w0; i < w1; i += 64) {
    const bool valid = i + lane < w1;
    const int2 e = valid ? sort_entry(ids, in, i + lane, a) : make_int2(0, 0);
    const int d = (e.x >> a.shift) & (R - 1);
    const uint64_t m = same_digit(d, a.bits, valid);
    int at = 0;
    if (valid) {
      at = mine[d] + __popcll(m & below);
      out[at] = e;
    }
    __builtin_amdgcn_wave_barrier();
    if (valid && (m & below) == 0) mine[d] = at + __popcll(m);
    __builtin_amdgcn_wave_barrier();
  }
}

// ---------------------------------------------------------------------------
// Sums of the sorted tokens' gradients
// ---------------------------------------------------------------------------
constexpr int kSegChunk = 32;  // entries a group of lanes sums in order

struct SegArgs {
  int64_t N, chunks;
  int V, D;
  float scale;
};

template <typename T>
__global__ void __launch_bounds__(256) tok_zero_kernel(T* __restrict__ p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = (T)0;
}

template <int DT>
__device__ inline void seg_write(const SegArgs& a, int v, int d, float sum,
                                 const typename TabType<DT>::t* __restrict__ tab,
                                 typename TabType<DT>::t* __restrict__ gtab) {
  const int64_t at = (int64_t)v * a.D + d;
  gtab[at] = tab_put<DT>(sum * tok_slope(tab_get<DT>(tab[at]), a.scale));
}

// A group of G lanes sums a chunk of kSegChunk entries over G columns. A run
// of one row that lies inside the chunk is written; a run that the chunk
// before it began goes to edge[0][chunk], one that begins here and goes on to
// edge[1][chunk], for tok_join_kernel.
template <int DT>
__global__ void __launch_bounds__(256)
tok_segment_kernel(SegArgs a, int G, const int2* __restrict__ ent, const float* __restrict__ gy,
                   const typename TabType<DT>::t* __restrict__ tab,
                   typename TabType<DT>::t* __restrict__ gtab, float* __restrict__ edge) {
  const int per = 256 / G;
  const int64_t c = (int64_t)blockIdx.x * per + threadIdx.x / G;
  if (c >= a.chunks) return;
  const int64_t i0 = c * kSegChunk, i1 = min(a.N, i0 + kSegChunk);
  for (int d = threadIdx.x % G; d < a.D; d += G) {
    int row = ent[i0].x;
    bool from_before = i0 > 0 && ent[i0 - 1].x == row;
    float sum = 0.0f;
    for (int64_t i = i0; i < i1; ++i) {
      const int2 e = ent[i];
      if (e.x != row) {
        if (from_before) edge[c * a.D + d] = sum;
        else if (row < a.V) seg_write<DT>(a, row, d, sum, tab, gtab);
        row = e.x;
        from_before = false;
        sum = 0.0f;
      }
      if (row >= a.V) break;
      sum += gy[(int64_t)(uint32_t)e.y * a.D + d];
    }
    if (row >= a.V) continue;
    const bool goes_on = i1 < a.N && ent[i1].x == row;
    if (from_before) edge[c * a.D + d] = sum;
    else if (goes_on) edge[(a.chunks + c) * a.D + d] = sum;
    else seg_write<DT>(a, row, d, sum, tab, gtab);
  }
}

// The runs that cross chunks: the workgroup of the chunk where one begins
// adds the chunks' parts in order.
template <int DT>
__global__ void __launch_bounds__(256)
tok_join_kernel(SegArgs a, const int2* __restrict__ ent, const float* __restrict__ edge,
                const typename TabType<DT>::t* __restrict__ tab,
                typename TabType<DT>::t* __restrict__ gtab) {
  const int64_t c = blockIdx.x, i0 = c * kSegChunk, i1 = min(a.N, i0 + kSegChunk);
  const int row = ent[i1 - 1].x;
  if (row >= a.V || i1 >= a.N || ent[i1].x != row) return;      // nothing goes on
  if (i0 > 0 && ent[i0].x == row && ent[i0 - 1].x == row) return;  // begun before this chunk
  int64_t last = c + 1;  // the run's last chunk
  while (last + 1 < a.chunks && ent[(last + 1) * kSegChunk].x == row) ++last;
  for (int d = threadIdx.x; d < a.D; d += 256) {
    float sum = edge[(a.chunks + c) * a.D + d];
    for (int64_t k = c + 1; k <= last; ++k) sum += edge[k * a.D + d];
    seg_write<DT>(a, row, d, sum, tab, gtab);
  }
}

// ---------------------------------------------------------------------------
// Hard bits
// ---------------------------------------------------------------------------
// bits [V][DW] words: bit d % 64 of word d / 64 of a row = E > 0. A wave per word.
template <int DT>
__global__ void __launch_bounds__(256)
tok_bits_kernel(const typename TabType<DT>::t* __restrict__ tab, int64_t words, int D, int DW,
                uint64_t* __restrict__ bits) {
  const int lane = threadIdx.x & 63;
  for (int64_t k = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); k < words; k += (int64_t)gridDim.x * 4) {
    const int64_t v = k / DW;
    const int d = (int)(k - v * DW) * 64 + lane;
    const uint64_t w = __ballot(d < D && tab_get<DT>(tab[v * D + min(d, D - 1)]) > 0.0f);
    if (lane == 0) bits[k] = w;
  }
}

// Bits as uint8 [N, D].
template <typename IdT>
__global__ void __launch_bounds__(256)
tok_bytes_kernel(const IdT* __restrict__ ids, int64_t N, int V, int64_t pad, int D, int DW,
                 const uint64_t* __restrict__ bits, uint8_t* __restrict__ out) {
  const int64_t n_all = N * D;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n_all; i += (int64_t)gridDim.x * 256) {
    const int64_t n = i / D;
    const int d = (int)(i - n * D), r = tok_row(ids, n, V, pad);
    out[i] = r < V ? (uint8_t)((bits[(int64_t)r * DW + (d >> 6)] >> (d & 63)) & 1u) : 0;
  }
}

// Bits packed 64 samples a word: a wave takes 64 samples' word dw of token l
// and writes the transpose, word j = bit j of the 64 samples.
template <typename IdT, bool WM>
__global__ void __launch_bounds__(256)
tok_packed_kernel(const IdT* __restrict__ ids, int64_t B, int64_t L, int V, int64_t pad, int D, int DW,
                  int64_t nw, const uint64_t* __restrict__ bits, uint64_t* __restrict__ out) {
  const int lane = threadIdx.x & 63;
  const int64_t F = L * D, jobs = nw * L * DW;
  for (int64_t k = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); k < jobs; k += (int64_t)gridDim.x * 4) {
    const int64_t w = k / (L * DW);
    const int64_t r = k - w * (L * DW);
    const int64_t l = r / DW;
    const int dw = (int)(r - l * DW);
    const int64_t b = w * 64 + lane;
    const int row = b < B ? tok_row(ids, b * L + l, V, pad) : V;
    const uint64_t m = row < V ? bits[(int64_t)row * DW + dw] : 0ull;
    uint64_t mine = 0;
    for (int j = 0; j < 64; ++j) {
      const uint64_t t = __ballot((m >> j) & 1);
      if (lane == j) mine = t;
    }
    const int d = dw * 64 + lane;
    if (d < D) {
      const int64_t f = l * D + d;
      out[WM ? w * F + f : f * nw + w] = mine;
    }
  }
}

static unsigned grid_of(int64_t blocks) { return (unsigned)std::min<int64_t>(std::max<int64_t>(blocks, 1), 1 << 16); }

static bool tok_sizes(int64_t N, int64_t V, int64_t D) {
  return N >= 0 && N < (1LL << 31) - 8192 && V > 0 && V < (1LL << 30) && D > 0 && D < (1LL << 24) &&
         N * D < (1LL << 40) && V * D < (1LL << 40);
}

// f(table type tag, id type tag)
template <typename F>
static void tok_dispatch(int dtype, int id_bytes, F&& f) {
  auto ids = [&](auto dt) {
    if (id_bytes == 8) f(dt, (int64_t)0);
    else f(dt, (int32_t)0);
  };
  if (dtype == kTabF32) ids(std::integral_constant<int, kTabF32>{});
  else if (dtype == kTabBf16) ids(std::integral_constant<int, kTabBf16>{});
  else ids(std::integral_constant<int, kTabF16>{});
}

struct TokBwdPlan {
  int64_t blocks, tile, chunks;
  int passes, bits;
  int64_t ent, hist, edge;  // 4-byte words of one entry array, the counts, the edges
  int64_t total() const { return 2 * ent + hist + edge; }
};

static TokBwdPlan tok_bwd_plan(int64_t N, int64_t V, int64_t D) {
  TokBwdPlan p{};
  auto round4 = [](int64_t n) { return (n + 3) & ~int64_t(3); };
  p.tile = std::max<int64_t>(kSortMinTile, cdiv(cdiv(N, kSortBlocks), 1024) * 1024);
  p.blocks = std::max<int64_t>(1, cdiv(N, p.tile));
  int key = 1;  // bits of the largest key, V
  while (key < 31 && (V >> key) != 0) ++key;
  p.passes = (key + kSortMaxBits - 1) / kSortMaxBits;
  p.bits = (key + p.passes - 1) / p.passes;
  p.chunks = cdiv(N, kSegChunk);
  p.ent = round4(2 * N);
  p.hist = round4(p.blocks << p.bits);
  p.edge = round4(2 * p.chunks * D);
  return p;
}

}  // namespace slg

using namespace slg;

#define TOK_CHECK(name)                                                                              \
  SLG_REQUIRE(dtype >= 0 && dtype <= 2, SLG_E_ARG, name ": table dtype %d", dtype);                  \
  SLG_REQUIRE(id_bytes == 4 || id_bytes == 8, SLG_E_ARG, name ": ids of %d bytes", id_bytes);        \
  SLG_REQUIRE(tok_sizes(N, V, D), SLG_E_SHAPE, name ": N %lld, V %lld, D %lld", (long long)N,        \
              (long long)V, (long long)D)

extern "C" {

int slg_token_encode(const void* ids, int32_t id_bytes, int64_t N, int64_t V, int64_t D, int64_t pad,
                     const void* table, int32_t dtype, float scale, int32_t ste, float* y,
                     slg_stream_t stream) {
  SLG_REQUIRE(table && ((ids && y) || N == 0), SLG_E_ARG, "token_encode: null pointer");
  TOK_CHECK("token_encode");
  if (N == 0) return 0;
  hipStream_t st = as_stream(stream);
  tok_dispatch(dtype, id_bytes, [&](auto dt, auto it) {
    using Id = decltype(it);
    using T = typename TabType<decltype(dt)::value>::t;
    hipLaunchKernelGGL((tok_encode_kernel<decltype(dt)::value, Id, 1>), dim3(grid_of(cdiv(N * D, 256))),
                       dim3(256), 0, st, static_cast<const Id*>(ids), N * D, (int)D, (int)V, pad,
                       static_cast<const T*>(table), scale, ste, y);
  });
  SLG_LAUNCH_CHECK("token_encode");
  return 0;
}

int64_t slg_token_encode_bwd_workspace(int64_t N, int64_t V, int64_t D) {
  return tok_sizes(N, V, D) ? tok_bwd_plan(N, V, D).total() : -1;
}

int slg_token_encode_bwd(const void* ids, int32_t id_bytes, int64_t N, int64_t V, int64_t D, int64_t pad,
                         const void* table, int32_t dtype, float scale, const float* gy, void* gtable,
                         int32_t* workspace, int64_t workspace_words, slg_stream_t stream) {
  SLG_REQUIRE(table && gtable && ((ids && gy && workspace) || N == 0), SLG_E_ARG,
              "token_encode_bwd: null pointer");
  TOK_CHECK("token_encode_bwd");
  const TokBwdPlan p = tok_bwd_plan(N, V, D);
  SLG_REQUIRE(workspace_words >= p.total() && (uintptr_t)workspace % 16 == 0, SLG_E_ARG,
              "token_encode_bwd: workspace of %lld words, %lld at a multiple of 16 bytes needed",
              (long long)workspace_words, (long long)p.total());
  hipStream_t st = as_stream(stream);
  int2* ent[2] = {reinterpret_cast<int2*>(workspace), reinterpret_cast<int2*>(workspace + p.ent)};
  int* hist = workspace + 2 * p.ent;
  float* edge = reinterpret_cast<float*>(hist + p.hist);
  const size_t lds = sizeof(int) * kSortWaves << p.bits;
  int rc = 0;
  tok_dispatch(dtype, id_bytes, [&](auto dt, auto it) {
    using Id = decltype(it);
    constexpr int DT = decltype(dt)::value;
    using T = typename TabType<DT>::t;
    hipLaunchKernelGGL((tok_zero_kernel<T>), dim3(grid_of(cdiv(V * D, 256))), dim3(256), 0, st,
                       static_cast<T*>(gtable), V * D);
    if (N == 0) return;
    SortArgs a{N, p.tile, (int)V, pad, 0, p.bits};
    const int2* in = nullptr;
    for (int k = 0; k < p.passes; ++k, a.shift += p.bits) {
      hipLaunchKernelGGL((tok_hist_kernel<Id>), dim3((unsigned)p.blocks), dim3(kSortThreads), 0, st, a,
                         static_cast<const Id*>(ids), in, hist);
      hipLaunchKernelGGL((tok_scatter_kernel<Id>), dim3((unsigned)p.blocks), dim3(kSortThreads), lds, st, a,
                         static_cast<const Id*>(ids), in, hist, ent[k & 1]);
      in = ent[k & 1];
    }
    const SegArgs s{N, p.chunks, (int)V, (int)D, scale};
    int G = 16;
    while (G < 64 && G < D) G *= 2;
    hipLaunchKernelGGL((tok_segment_kernel<DT>), dim3((unsigned)cdiv(p.chunks, 256 / G)), dim3(256), 0, st, s, G,
                       in, gy, static_cast<const T*>(table), static_cast<T*>(gtable), edge);
    hipLaunchKernelGGL((tok_join_kernel<DT>), dim3((unsigned)p.chunks), dim3(256), 0, st, s, in, edge,
                       static_cast<const T*>(table), static_cast<T*>(gtable));
  });
  if (rc) return rc;
  SLG_LAUNCH_CHECK("token_encode_bwd");
  return 0;
}

int slg_token_bits(const void* table, int32_t dtype, int64_t V, int64_t D, uint64_t* bits, slg_stream_t stream) {
  SLG_REQUIRE(table && bits, SLG_E_ARG, "token_bits: null pointer");
  SLG_REQUIRE(dtype >= 0 && dtype <= 2, SLG_E_ARG, "token_bits: table dtype %d", dtype);
  SLG_REQUIRE(tok_sizes(0, V, D), SLG_E_SHAPE, "token_bits: V %lld, D %lld", (long long)V, (long long)D);
  const int64_t DW = cdiv(D, 64);
  tok_dispatch(dtype, 8, [&](auto dt, auto) {
    using T = typename TabType<decltype(dt)::value>::t;
    hipLaunchKernelGGL((tok_bits_kernel<decltype(dt)::value>), dim3(grid_of(cdiv(V * DW, 4))), dim3(256), 0,
                       as_stream(stream), static_cast<const T*>(table), V * DW, (int)D, (int)DW, bits);
  });
  SLG_LAUNCH_CHECK("token_bits");
  return 0;
}

int slg_token_encode_hard(const void* ids, int32_t id_bytes, int64_t B, int64_t L, int64_t V, int64_t D,
                          int64_t pad, const uint64_t* bits, int32_t layout, void* out, slg_stream_t stream) {
  SLG_REQUIRE(bits && ((ids && out) || B == 0 || L == 0), SLG_E_ARG, "token_encode_hard: null pointer");
  SLG_REQUIRE(layout >= 0 && layout <= 2, SLG_E_ARG, "token_encode_hard: layout %d", layout);
  SLG_REQUIRE(B >= 0 && L >= 0 && B < (1LL << 31) && L < (1LL << 31), SLG_E_SHAPE,
              "token_encode_hard: B %lld, L %lld", (long long)B, (long long)L);
  const int64_t N = B * L;
  const int32_t dtype = 0;
  TOK_CHECK("token_encode_hard");
  if (N == 0) return 0;
  hipStream_t st = as_stream(stream);
  const int64_t DW = cdiv(D, 64), nw = cdiv(B, 64);
  tok_dispatch(0, id_bytes, [&](auto, auto it) {
    using Id = decltype(it);
    const Id* id = static_cast<const Id*>(ids);
    if (layout == 2) {
      hipLaunchKernelGGL((tok_bytes_kernel<Id>), dim3(grid_of(cdiv(N * D, 256))), dim3(256), 0, st, id, N, (int)V,
                         pad, (int)D, (int)DW, bits, static_cast<uint8_t*>(out));
      return;
    }
    const dim3 grid(grid_of(cdiv(nw * L * DW, 4)));
    if (layout == 1)
      hipLaunchKernelGGL((tok_packed_kernel<Id, true>), grid, dim3(256), 0, st, id, B, L, (int)V, pad, (int)D,
                         (int)DW, nw, bits, static_cast<uint64_t*>(out));
    else
      hipLaunchKernelGGL((tok_packed_kernel<Id, false>), grid, dim3(256), 0, st, id, B, L, (int)V, pad, (int)D,
                         (int)DW, nw, bits, static_cast<uint64_t*>(out));
  });
  SLG_LAUNCH_CHECK("token_encode_hard");
  return 0;
}

}  // extern "C"
