// Token encoder for gfx950: a learned row of D soft bits per token id.
//   soft   y[n, d] = sigmoid(scale * E[t_n, d]) (ste: 1 where E > 0, else 0)
//   hard   bit (n, d) = E[t_n, d] > 0, the soft form past 1/2 (scale > 0: a
//          negative one would put the soft form and the bits at odds)
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

#include "radix_sort.h"

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

// sigmoid(z) of a table's entry, from t = -z log2 e: 1 / (1 + 2^t) with the
// hardware exp2 and reciprocal (about an ulp each).
__device__ inline float tok_value(float e, float nlog2, bool ste) {
  if (ste) return e > 0.0f ? 1.0f : 0.0f;
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(e * nlog2));
}

// scale * sigmoid'(scale e) = scale t / (1 + t)^2, t = exp(-|scale e|): no
// difference of values near 1; exp2 and reciprocal as above (with expf and a
// division the writes of short runs took as long as their loads).
__device__ inline float tok_slope(float e, float scale) {
  const float t = __builtin_amdgcn_exp2f(-fabsf(e * (scale * 1.44269504f))), r = __builtin_amdgcn_rcpf(1.0f + t);
  return scale * (t * r) * r;
}

// VU neighbouring values of a table's row or of a gradient's, from any element
// on: a row's last group is moved back to end with the row (the columns that
// two lanes then hold come out the same from both). RAG = false: rows of whole
// groups, aligned as such.
template <int DT, int VU, bool RAG = true>
struct RowVec {
  using T = typename TabType<DT>::t;
  typedef T t __attribute__((ext_vector_type(VU), aligned(sizeof(T) * (RAG ? 1 : VU))));
};
template <int DT, int VU, bool RAG = true>
__device__ inline void tab_load(const typename TabType<DT>::t* __restrict__ p, float (&v)[VU]) {
  using T = typename TabType<DT>::t;
  const typename RowVec<DT, VU, RAG>::t r = *reinterpret_cast<const typename RowVec<DT, VU, RAG>::t*>(p);
#pragma unroll
  for (int j = 0; j < VU; ++j) v[j] = tab_get<DT>(VU == 1 ? ((const T*)&r)[0] : r[j]);
}
template <int DT, int VU, bool RAG = true, bool NT = false>
__device__ inline void tab_store(typename TabType<DT>::t* __restrict__ p, const float (&v)[VU]) {
  using Vt = typename RowVec<DT, VU, RAG>::t;
  Vt r;
#pragma unroll
  for (int j = 0; j < VU; ++j) r[j] = tab_put<DT>(v[j]);
  if constexpr (NT) __builtin_nontemporal_store(r, reinterpret_cast<Vt*>(p));
  else *reinterpret_cast<Vt*>(p) = r;
}
// The first column of group c.
template <int VU, bool RAG = true>
__device__ inline int group_col(int c, int D) {
  return RAG ? min(c * VU, D - VU) : c * VU;
}

// A thread takes kEncUnits units of VU values of one token, a workgroup's units
// next to each other (upr units a row). The values stream past the caches,
// which are left to the table's rows (524288 tokens of 128 values, 25.6 MB of
// table: 55 against 68 us). Idx: the type that counts units.
constexpr int kEncUnits = 4;
template <int DT, typename IdT, int VU, bool RAG>
__global__ void __launch_bounds__(256)
tok_encode_kernel(const IdT* __restrict__ ids, int64_t units, int64_t upr, int D, int V, int64_t pad,
                  const typename TabType<DT>::t* __restrict__ tab, float nlog2, int ste, float* __restrict__ y) {
  for (int64_t u0 = (int64_t)blockIdx.x * (256 * kEncUnits) + threadIdx.x; u0 < units;
       u0 += (int64_t)gridDim.x * (256 * kEncUnits)) {
    int r[kEncUnits], col[kEncUnits];
    int64_t at[kEncUnits];
    float e[kEncUnits][VU];
#pragma unroll
    for (int k = 0; k < kEncUnits; ++k) {
      const int64_t u = min(u0 + k * 256, units - 1), n = u / upr;
      col[k] = group_col<VU, RAG>((int)(u - n * upr), D);
      at[k] = n * D + col[k];
      r[k] = tok_row(ids, n, V, pad);
    }
#pragma unroll
    for (int k = 0; k < kEncUnits; ++k)  // an absent token reads row 0
      tab_load<DT, VU, RAG>(tab + (int64_t)(r[k] < V ? r[k] : 0) * D + col[k], e[k]);
#pragma unroll
    for (int k = 0; k < kEncUnits; ++k) {
      if (u0 + k * 256 < units) {
        float v[VU];
#pragma unroll
        for (int j = 0; j < VU; ++j) v[j] = r[k] < V ? tok_value(e[k][j], nlog2, ste != 0) : 0.0f;
        tab_store<kTabF32, VU, RAG, true>(y + at[k], v);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Gradient of the table: tokens sorted by row (radix_sort.h; absent ones, of
// row V, come last), then summed in that order.
// ---------------------------------------------------------------------------
template <typename IdT>
struct TokenKeys {
  const IdT* ids;
  int V;
  int64_t pad;
  __device__ int key(int64_t i) const { return tok_row(ids, i, V, pad); }
};

struct SegArgs {
  int64_t N, chunks;
  int V, D, C, G;  // C entries a chunk, G lanes a row
  float scale;
};

template <int DT, int VU>
__device__ inline void seg_write(const SegArgs& a, int v, int d, const float (&sum)[VU], const float (&e)[VU],
                                 typename TabType<DT>::t* __restrict__ gtab) {
  float g[VU];
#pragma unroll
  for (int j = 0; j < VU; ++j) g[j] = sum[j] * tok_slope(e[j], a.scale);
  tab_store<DT, VU>(gtab + (int64_t)v * a.D + d, g);
}

// G lanes sum a chunk of C entries, VU columns each, kSegAhead rows of the
// gradient in flight together with the table's rows that the runs ending among
// them are multiplied by. A run of one row inside the chunk is written; one
// that the chunk before it began goes to edge[0][chunk], one that begins here
// and goes on to edge[1][chunk] and on the list of tok_join_kernel (whose
// order does not matter: every run is summed by itself), to which a workgroup
// adds its runs at once (one atomic a run on one address took most of the
// kernel: 17 us at 65536 tokens of 64 values).
constexpr int kSegAhead = 4;
template <int DT, int VU>
__global__ void __launch_bounds__(256)
tok_segment_kernel(SegArgs a, const int2* __restrict__ ent, const float* __restrict__ gy,
                   const typename TabType<DT>::t* __restrict__ tab,
                   typename TabType<DT>::t* __restrict__ gtab, float* __restrict__ edge,
                   int* __restrict__ list, int* __restrict__ listed) {
  __shared__ int runs[256], n_runs, at_list;
  if (threadIdx.x == 0) n_runs = 0;
  __syncthreads();
  const int per = 256 / a.G, l = threadIdx.x % a.G;
  const int64_t c = (int64_t)blockIdx.x * per + threadIdx.x / a.G;
  const int64_t i0 = min(c * a.C, a.N - 1), i1 = min(a.N, c * a.C + a.C);
  const int first = ent[i0].x;
  const bool begun = i0 > 0 && ent[i0 - 1].x == first;
  const int after = i1 < a.N ? ent[i1].x : -1;
  // absent tokens from the chunk's start to the end: nothing
  for (int q = c < a.chunks && first < a.V ? l : a.D; q * VU < a.D; q += a.G) {
    const int d = group_col<VU>(q, a.D);
    bool from_before = begun;
    float sum[VU];
#pragma unroll
    for (int j = 0; j < VU; ++j) sum[j] = 0.0f;
    int2 next[kSegAhead];  // the next rows' entries, a batch ahead of their gradients
#pragma unroll
    for (int u = 0; u < kSegAhead; ++u) next[u] = ent[min(i0 + u, i1 - 1)];
    for (int64_t i = i0; i < i1; i += kSegAhead) {
      int2 e[kSegAhead];
      float g[kSegAhead][VU], t[kSegAhead][VU];
      bool ends[kSegAhead];
#pragma unroll
      for (int u = 0; u < kSegAhead; ++u) {
        e[u] = next[u];
        tab_load<kTabF32, VU>(gy + (int64_t)(uint32_t)e[u].y * a.D + d, g[u]);
      }
#pragma unroll
      for (int u = 0; u < kSegAhead; ++u) next[u] = ent[min(i + kSegAhead + u, i1 - 1)];
#pragma unroll
      for (int u = 0; u < kSegAhead; ++u) {
        const int64_t at = i + u + 1;
        const int then = at < i1 ? (u + 1 < kSegAhead ? e[(u + 1) % kSegAhead].x : next[0].x) : after;
        ends[u] = i + u < i1 && e[u].x < a.V && e[u].x != then;
        if (ends[u]) tab_load<DT, VU>(tab + (int64_t)e[u].x * a.D + d, t[u]);
      }
#pragma unroll
      for (int u = 0; u < kSegAhead; ++u) {
        if (i + u >= i1 || e[u].x >= a.V) break;
#pragma unroll
        for (int j = 0; j < VU; ++j) sum[j] += g[u][j];
        if (ends[u]) {
          if (from_before) tab_store<kTabF32, VU>(edge + c * a.D + d, sum);
          else seg_write<DT, VU>(a, e[u].x, d, sum, t[u], gtab);
          from_before = false;
#pragma unroll
          for (int j = 0; j < VU; ++j) sum[j] = 0.0f;
        }
      }
      if (e[kSegAhead - 1].x >= a.V) break;
    }
    const int row = ent[i1 - 1].x;
    if (row < a.V && after == row) {  // the last run goes on
      if (from_before) {
        tab_store<kTabF32, VU>(edge + c * a.D + d, sum);
      } else {
        tab_store<kTabF32, VU>(edge + (a.chunks + c) * a.D + d, sum);
        if (q == 0) runs[atomicAdd(&n_runs, 1)] = (int)c;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) at_list = n_runs ? atomicAdd(listed, n_runs) : 0;
  __syncthreads();
  for (int k = threadIdx.x; k < n_runs; k += 256) list[at_list + k] = runs[k];
}

// The runs that cross chunks. A group of G lanes takes a run of up to kJoinNear
// chunks past the one where it begins; the workgroup then takes its groups'
// longer runs one by one, their chunks' parts dealt to the groups (each in
// ascending order), whose sums are added in order. T = 1024 for few long runs
// (tok_join_threads).
constexpr int kJoinNear = 8;
template <int DT, int VU, int T>
__global__ void __launch_bounds__(T)
tok_join_kernel(SegArgs a, const int2* __restrict__ ent, const float* __restrict__ edge,
                const typename TabType<DT>::t* __restrict__ tab,
                typename TabType<DT>::t* __restrict__ gtab, const int* __restrict__ list,
                const int* __restrict__ listed) {
  constexpr int W = T / 64;
  __shared__ float red[T * VU];
  __shared__ int end[W], far[T], n_far;
  const int tid = threadIdx.x, wave = tid >> 6;
  const int P = T / a.G, part = tid / a.G, l = tid % a.G;
  const int n = *listed;
  // runs dealt to the workgroups one by one, so that long ones meet in few
  for (int64_t k0 = blockIdx.x; k0 < n; k0 += (int64_t)gridDim.x * P) {
    if (tid == 0) n_far = 0;
    __syncthreads();
    const int64_t k = k0 + (int64_t)part * gridDim.x;
    if (k < n) {
      const int64_t c = list[k];
      int x[kJoinNear];
#pragma unroll
      for (int u = 0; u < kJoinNear; ++u) x[u] = ent[min(c + 1 + u, a.chunks - 1) * a.C].x;
      const int row = ent[(c + 1) * a.C - 1].x;
      int m = 0;  // chunks past c that begin with the row
#pragma unroll
      for (int u = 0; u < kJoinNear; ++u) m += m == u && c + 1 + u < a.chunks && x[u] == row;
      if (m == kJoinNear) {
        if (l == 0) far[atomicAdd(&n_far, 1)] = (int)c;
      } else {
        for (int q = l; q * VU < a.D; q += a.G) {
          const int d = group_col<VU>(q, a.D);
          float s[VU], e[VU], g[kJoinNear - 1][VU];
          tab_load<kTabF32, VU>(edge + (a.chunks + c) * a.D + d, s);
          tab_load<DT, VU>(tab + (int64_t)row * a.D + d, e);
#pragma unroll
          for (int u = 0; u < kJoinNear - 1; ++u)
            tab_load<kTabF32, VU>(edge + (c + 1 + min(u, m - 1)) * a.D + d, g[u]);
#pragma unroll
          for (int u = 0; u < kJoinNear - 1; ++u)
#pragma unroll
            for (int j = 0; j < VU; ++j) s[j] += u < m ? g[u][j] : 0.0f;
          seg_write<DT, VU>(a, row, d, s, e, gtab);
        }
      }
    }
    __syncthreads();
    for (int f = 0; f < n_far; ++f) {
      const int64_t c = far[f];
      const int row = ent[(c + 1) * a.C - 1].x;
      int64_t last = c + kJoinNear;
      for (bool more = true; more;) {
        const int64_t q = last + 1 + tid;
        const uint64_t off = __ballot(q >= a.chunks || ent[min(q, a.chunks - 1) * a.C].x != row);
        if ((tid & 63) == 0) end[wave] = off ? __ffsll((unsigned long long)off) - 1 : 64;
        __syncthreads();
        int m = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          m += more ? end[w] : 0;
          more &= end[w] == 64;
        }
        __syncthreads();
        last += m;
      }
      for (int q0 = 0; q0 * VU < a.D; q0 += a.G) {
        const bool on = (q0 + l) * VU < a.D;
        const int d = on ? group_col<VU>(q0 + l, a.D) : 0;
        float sum[VU];
#pragma unroll
        for (int j = 0; j < VU; ++j) sum[j] = 0.0f;
        if (on) {
          constexpr int U = 8;
          for (int64_t q = c + 1 + part; q <= last; q += (int64_t)U * P) {
            float g[U][VU];
#pragma unroll
            for (int u = 0; u < U; ++u)
              tab_load<kTabF32, VU>(edge + min(q + (int64_t)u * P, last) * a.D + d, g[u]);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
              for (int j = 0; j < VU; ++j) sum[j] += q + (int64_t)u * P <= last ? g[u][j] : 0.0f;
          }
        }
#pragma unroll
        for (int j = 0; j < VU; ++j) red[(part * a.G + l) * VU + j] = sum[j];
        __syncthreads();
        if (part == 0 && on) {
          float s[VU], e[VU];
          tab_load<kTabF32, VU>(edge + (a.chunks + c) * a.D + d, s);
          tab_load<DT, VU>(tab + (int64_t)row * a.D + d, e);
          for (int p = 0; p < P; ++p)
#pragma unroll
            for (int j = 0; j < VU; ++j) s[j] += red[(p * a.G + l) * VU + j];
          seg_write<DT, VU>(a, row, d, s, e, gtab);
        }
        __syncthreads();
      }
    }
    __syncthreads();  // n_far is cleared
  }
}

// ---------------------------------------------------------------------------
// Hard bits
// ---------------------------------------------------------------------------
// bits [V][DW] words: bit d % 64 of word d / 64 of a row = E > 0. A wave per word,
// with one load of 64 values in flight: 32000 x 64 in fp32 7 us (8.4 MB, 1.2
// TB/s), once a version of the weight.
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

// Bits as uint8 [N, D], VU of a token a thread (D >= VU), written at any byte;
// a token's last run is moved back to end with it. 4.2 M tokens of 100 bits:
// 132 us with 16 bits a thread, 250 with 4 (and 8.4 M of 6: 82 us a bit a
// thread, 48 with 4).
template <typename IdT, int VU>
__global__ void __launch_bounds__(256)
tok_bytes_kernel(const IdT* __restrict__ ids, int64_t units, int upr, int D, int V, int64_t pad, int DW,
                 const uint64_t* __restrict__ bits, uint8_t* __restrict__ out) {
  constexpr int VW = VU < 4 ? 1 : VU / 4;
  typedef uint32_t run __attribute__((ext_vector_type(VW), aligned(1)));
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < units; i += (int64_t)gridDim.x * 256) {
    const int64_t n = i / upr;
    const int d = group_col<VU>((int)(i - n * upr), D), r = tok_row(ids, n, V, pad), s = d & 63;
    uint32_t b = 0;
    if (r < V) {
      const uint64_t* w = bits + (int64_t)r * DW + (d >> 6);
      b = (uint32_t)(w[0] >> s);
      if (s + VU > 64) b |= (uint32_t)(w[1] << (64 - s));
    }
    if constexpr (VU >= 4) {
      run v;
#pragma unroll
      for (int j = 0; j < VW; ++j) v[j] = (((b >> (4 * j)) & 15u) * 0x00204081u) & 0x01010101u;  // bit j to byte j
      *reinterpret_cast<run*>(out + n * D + d) = v;
    } else {
      out[i] = (uint8_t)(b & 1u);
    }
  }
}

// The wave's 64 x 64 bits transposed: lane j's word becomes bit j of every
// lane's word (six exchanges of halves; a ballot per bit took 5 times the
// instructions).
__device__ inline uint64_t wave_transpose(uint64_t m) {
  const int lane = threadIdx.x & 63;
  uint32_t lo = (uint32_t)m, hi = (uint32_t)(m >> 32);
  const uint32_t got = (uint32_t)__shfl_xor((int)(lane & 32 ? lo : hi), 32, 64);
  if (lane & 32) lo = got; else hi = got;
  auto halves = [&](int s, uint32_t keep) {
    const uint32_t ylo = (uint32_t)__shfl_xor((int)lo, s, 64), yhi = (uint32_t)__shfl_xor((int)hi, s, 64);
    if (lane & s) {
      lo = (lo & ~keep) | ((ylo >> s) & keep);
      hi = (hi & ~keep) | ((yhi >> s) & keep);
    } else {
      lo = (lo & keep) | ((ylo & keep) << s);
      hi = (hi & keep) | ((yhi & keep) << s);
    }
  };
  halves(16, 0x0000ffffu);
  halves(8, 0x00ff00ffu);
  halves(4, 0x0f0f0f0fu);
  halves(2, 0x33333333u);
  halves(1, 0x55555555u);
  return (uint64_t)hi << 32 | lo;
}

constexpr int kPackTokens = 4;
// The rows of kPackTokens neighbouring tokens of which n are there (the rest:
// absent), as 16-byte loads where all are.
template <typename IdT>
__device__ inline void tok_rows(const IdT* __restrict__ p, int64_t n, int V, int64_t pad, int (&row)[kPackTokens]) {
  IdT t[kPackTokens];
  if (n >= kPackTokens) {
    typedef IdT t4 __attribute__((ext_vector_type(kPackTokens), aligned(sizeof(IdT))));
    const t4 r = *reinterpret_cast<const t4*>(p);
#pragma unroll
    for (int u = 0; u < kPackTokens; ++u) t[u] = r[u];
  } else {
#pragma unroll
    for (int u = 0; u < kPackTokens; ++u) t[u] = u < n ? p[u] : (IdT)-1;
  }
#pragma unroll
  for (int u = 0; u < kPackTokens; ++u) row[u] = tok_row(t, u, V, pad);
}
// Bits packed 64 samples a word. A wave takes 64 samples' word dw of kPackTokens
// neighbouring tokens (whose ids share memory lines) and transposes each: lane
// j then holds feature j's word. Word-major rows of features are written as
// they are; for the rows [F][nw] a workgroup's waves take TW neighbouring
// words, which leave through LDS in runs of TW. Bound by the loads of
// single rows of bits, a line each: 65536 x 16 tokens of 64 bits 9.7 us (17 MB
// of ids and words, 1.8 TB/s; with the ids loaded one by one 13.4), 65536 x 128
// of 2 bits 43. Word-major the same to 5% (calls of 65536 x 64 x 100 bits: 42.5
// us, word-major 39.9).
template <typename IdT, bool WM, int TW>
__global__ void __launch_bounds__(64 * TW)
tok_packed_kernel(const IdT* __restrict__ ids, int64_t B, int64_t L, int V, int64_t pad, int D, int DW,
                  int64_t nw, const uint64_t* __restrict__ bits, uint64_t* __restrict__ out) {
  __shared__ uint64_t tile[WM ? 1 : kPackTokens][WM ? 1 : 64][WM ? 1 : TW + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t F = L * D, wt = (nw + TW - 1) / TW, lt = (L + kPackTokens - 1) / kPackTokens, jobs = wt * lt * DW;
  // the jobs that share ids' lines on one XCD, whose L2 then reads them once
  for (int64_t k = xcd_logical_id(blockIdx.x, gridDim.x); k < jobs; k += gridDim.x) {
    const int64_t t = k / (lt * DW), r = k - t * (lt * DW), l0 = r / DW * kPackTokens;
    const int dw = (int)(r % DW);
    const int64_t w = t * TW + wave, b = w * 64 + lane;
    int row[kPackTokens];
    uint64_t m[kPackTokens];
    tok_rows(ids + min(b, B - 1) * L + l0, L - l0, V, pad, row);
    if (b >= B)
#pragma unroll
      for (int u = 0; u < kPackTokens; ++u) row[u] = V;
#pragma unroll
    for (int u = 0; u < kPackTokens; ++u) m[u] = row[u] < V ? bits[(int64_t)row[u] * DW + dw] : 0ull;
    const int d = dw * 64 + lane;
#pragma unroll
    for (int u = 0; u < kPackTokens; ++u) {
      const uint64_t v = wave_transpose(m[u]);
      if constexpr (WM) {
        if (w < nw && d < D && l0 + u < L) out[w * F + (l0 + u) * D + d] = v;
      } else {
        tile[u][lane][wave] = v;
      }
    }
    if constexpr (!WM) {
      __syncthreads();
      const int j = threadIdx.x / TW, i = threadIdx.x % TW;
      if (t * TW + i < nw && dw * 64 + j < D)
#pragma unroll
        for (int u = 0; u < kPackTokens; ++u)
          if (l0 + u < L) out[((l0 + u) * D + dw * 64 + j) * nw + t * TW + i] = tile[u][j][i];
      __syncthreads();
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


// Threads of a join's workgroup: 256, or 1024 where a few rows have all tokens,
// whose runs a workgroup each then reads (131072 tokens of 512 values over 2
// rows: 243 us in all with 256, 185 with 1024; 65536 x 64 over 32000 rows: the
// join 7 and 17 us; 4.1 M tokens of one value over 1000 rows: 271 and 332 in
// all).
static int tok_join_threads(int64_t chunks, int64_t V) { return V <= 256 && chunks >= 32 * V ? 1024 : 256; }

struct TokBwdPlan {
  RadixPlan sort;
  int64_t chunks, edge, list;
  int C, G, VU;
  int64_t total() const { return sort.words() + edge + list; }
};

// Lanes a row: a power of two up to the wave. Chunks: 256 entries, fewer where
// that leaves less than 16 waves a CU (524288 x 128 tokens: 64; 65536 x 64: 8,
// of which 16 and 32 took 1 and 7 us longer with their joins).
static TokBwdPlan tok_bwd_plan(int64_t N, int64_t V, int64_t D) {
  TokBwdPlan p{};
  p.sort = radix_plan(N, V + 1);
  p.VU = D >= 4 ? 4 : 1;
  p.G = 1;
  while (p.G < 64 && p.G * p.VU < D) p.G *= 2;
  p.C = 256;
  while (p.C > 8 && cdiv(N, p.C) * p.G < 262144) p.C /= 2;
  p.chunks = cdiv(N, p.C);
  p.edge = (2 * p.chunks * D + 3) & ~int64_t(3);
  p.list = p.chunks + 1;
  return p;
}

}  // namespace slg

using namespace slg;

#define TOK_CHECK(name)                                                                              \
  SLG_REQUIRE(dtype >= 0 && dtype <= 2, SLG_E_ARG, name ": table dtype %d", dtype);                  \
  SLG_REQUIRE(id_bytes == 4 || id_bytes == 8, SLG_E_ARG, name ": ids of %d bytes", id_bytes);        \
  SLG_REQUIRE(tok_sizes(N, V, D), SLG_E_SHAPE, name ": N %lld, V %lld, D %lld", (long long)N,        \
              (long long)V, (long long)D)

// scale log2 e has to be finite too: 0 times an infinity has no value.
#define TOK_CHECK_SCALE(name) \
  SLG_REQUIRE(scale > 0.0f && scale <= 2e38f, SLG_E_ARG, name ": scale %g outside (0, 2e38]", (double)scale)

extern "C" {

int slg_token_encode(const void* ids, int32_t id_bytes, int64_t N, int64_t V, int64_t D, int64_t pad,
                     const void* table, int32_t dtype, float scale, int32_t ste, float* y,
                     slg_stream_t stream) {
  SLG_REQUIRE(table && ((ids && y) || N == 0), SLG_E_ARG, "token_encode: null pointer");
  TOK_CHECK("token_encode");
  TOK_CHECK_SCALE("token_encode");
  if (N == 0) return 0;
  hipStream_t st = as_stream(stream);
  const float nlog2 = (float)(-1.4426950408889634 * (double)scale);
  tok_dispatch(dtype, id_bytes, [&](auto dt, auto it) {
    constexpr int DT = decltype(dt)::value;
    using Id = decltype(it);
    using T = typename TabType<DT>::t;
    auto go = [&](auto kern, int vu) {
      const int64_t upr = cdiv(D, vu), units = N * upr;
      hipLaunchKernelGGL(kern, dim3(grid_of(cdiv(units, 256 * kEncUnits))), dim3(256), 0, st,
                         static_cast<const Id*>(ids), units, upr, (int)D, (int)V, pad,
                         static_cast<const T*>(table), nlog2, ste, y);
    };
    // whole aligned groups (524288 x 256: 84 us, taken as ragged ones 92), any
    // rows of 4 values (2.4 M x 27: 62 us, a value a thread 102), narrower ones
    const bool whole = D % 4 == 0 && (uintptr_t)table % (4 * sizeof(T)) == 0 && (uintptr_t)y % 16 == 0;
    if (whole) go(tok_encode_kernel<DT, Id, 4, false>, 4);
    else if (D >= 4) go(tok_encode_kernel<DT, Id, 4, true>, 4);
    else go(tok_encode_kernel<DT, Id, 1, true>, 1);
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
  TOK_CHECK_SCALE("token_encode_bwd");
  const TokBwdPlan p = tok_bwd_plan(N, V, D);
  SLG_REQUIRE(workspace_words >= p.total() && (uintptr_t)workspace % 16 == 0, SLG_E_ARG,
              "token_encode_bwd: workspace of %lld words, %lld at a multiple of 16 bytes needed",
              (long long)workspace_words, (long long)p.total());
  hipStream_t st = as_stream(stream);
  SLG_REQUIRE((uintptr_t)gtable % 16 == 0, SLG_E_ARG, "token_encode_bwd: gtable not at a multiple of 16 bytes");
  float* edge = reinterpret_cast<float*>(workspace + p.sort.words());
  int* listed = workspace + p.sort.words() + p.edge;
  tok_dispatch(dtype, id_bytes, [&](auto dt, auto it) {
    using Id = decltype(it);
    constexpr int DT = decltype(dt)::value;
    using T = typename TabType<DT>::t;
    const RadixClear clear{gtable, V * D * (int64_t)sizeof(T), N > 0 ? listed : nullptr};
    if (N == 0) {
      hipLaunchKernelGGL(radix_clear_kernel, dim3(grid_of(cdiv(clear.bytes, 16 * kRadixThreads))),
                         dim3(kRadixThreads), 0, st, clear);
      return;
    }
    const int2* ent = radix_sort(TokenKeys<Id>{static_cast<const Id*>(ids), (int)V, pad}, p.sort, workspace, clear, st);
    auto go = [&](auto vu) {
      constexpr int VU = decltype(vu)::value;
      const SegArgs s{N, p.chunks, (int)V, (int)D, p.C, p.G, scale};
      hipLaunchKernelGGL((tok_segment_kernel<DT, VU>), dim3((unsigned)cdiv(p.chunks, 256 / p.G)), dim3(256), 0, st, s,
                         ent, gy, static_cast<const T*>(table), static_cast<T*>(gtable), edge, listed + 1, listed);
      const int T2 = tok_join_threads(p.chunks, V);
      hipLaunchKernelGGL((T2 == 1024 ? tok_join_kernel<DT, VU, 1024> : tok_join_kernel<DT, VU, 256>),
                         dim3((unsigned)std::min<int64_t>(p.chunks, 512 * 1024 / T2)), dim3(T2), 0, st, s, ent, edge,
                         static_cast<const T*>(table), static_cast<T*>(gtable), listed + 1, listed);
    };
    if (p.VU == 4) go(std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, 1>{});
  });
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
      auto go = [&](auto kern, int64_t vu) {
        const int64_t upr = cdiv(D, vu), units = N * upr;
        hipLaunchKernelGGL(kern, dim3(grid_of(cdiv(units, 256))), dim3(256), 0, st, id, units, (int)upr, (int)D,
                           (int)V, pad, (int)DW, bits, static_cast<uint8_t*>(out));
      };
      if (D >= 16) go(tok_bytes_kernel<Id, 16>, 16);
      else if (D >= 4) go(tok_bytes_kernel<Id, 4>, 4);
      else go(tok_bytes_kernel<Id, 1>, 1);
      return;
    }
    auto go = [&](auto kern, int tw) {
      hipLaunchKernelGGL(kern, dim3(grid_of(cdiv(cdiv(nw, tw) * cdiv(L, kPackTokens) * DW, 8) * 8)), dim3(64 * tw), 0, st, id, B, L, (int)V, pad,
                         (int)D, (int)DW, nw, bits, static_cast<uint64_t*>(out));
    };
    // as many neighbouring words a workgroup as there are, so that no wave
    // idles (one word's tokens, 64 x 20000 x 64 bits: 11 us; with 4 and 8
    // words a workgroup 15 and 27), up to 8, whose rows leave in runs of 64
    // bytes (65536 x 64 x 100 bits: 32 us; with 4 the same, with 1 52). One
    // word a feature lies the same in both layouts.
    if (nw == 1) go(tok_packed_kernel<Id, false, 1>, 1);
    else if (layout == 1) go(tok_packed_kernel<Id, true, 4>, 4);
    else if (nw <= 4) go(tok_packed_kernel<Id, false, 4>, 4);
    else go(tok_packed_kernel<Id, false, 8>, 8);
  });
  SLG_LAUNCH_CHECK("token_encode_hard");
  return 0;
}

}  // extern "C"
