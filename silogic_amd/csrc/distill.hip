// The loss of a student's logits against a teacher's largest ones, with its gradient (gfx950). Row s of V logits,
// the teacher's values t_j at tokens i_j (K of them), temperature T:
//   q_j  = softmax(t / T) over the entries that are there: an id in 0..V-1 and a value other than -inf
//   p    = softmax(s / T),  p1 = softmax(s)
//   loss = a_s T^2 sum_j q_j (log q_j - log p[i_j]) - a_h log p1[label]
//   grad = a_s T (p - sum of q_j with i_j = .) + a_h (p1 - [. = label])
// a_s = 1 - alpha and a_h = alpha with labels, else 1 and 0. A term whose entries or label are missing counts 0, and
// so does a row of logits that are all -inf; "mean" is over the rows that have an entry or a label. A token named
// twice gets both entries' probabilities.
//
// Both softmaxes share their maximum m: what is kept of a row is m, 1/Z and 1/Z1 (and the teacher's own), so that a
// probability is exp((s - m) / T) / Z with the difference exact where it matters. Sums are fp32, those over rows 64
// bits; the gradient is rounded once.
#include <algorithm>

#include "block_ops.h"
#include "float_types.h"

namespace slg {

constexpr float kLog2e = 1.44269504f;
constexpr int kMaxEntries = 1024;
constexpr int kKept = 8;   // floats kept of a row: m, 1/Z, 1/Z1, the teacher's maximum and 1/sum, a_s T, a_h, unused

struct Distill {
  const void* logits;
  int64_t N, V, ld;
  const void* values;
  int vtype;
  const void* ids;
  int id_bytes, K;
  const void* labels;   // null: none
  int label_bytes;
  float T, inv_t, alpha;
};

__device__ inline float load_as(const void* p, int dtype, int64_t i) {
  if (dtype == kTabF32) return static_cast<const float*>(p)[i];
  if (dtype == kTabBf16) return tab_get<kTabBf16>(static_cast<const uint16_t*>(p)[i]);
  return (float)static_cast<const _Float16*>(p)[i];
}
__device__ inline int64_t load_id(const void* p, int bytes, int64_t i) {
  return bytes == 8 ? static_cast<const int64_t*>(p)[i] : (int64_t)static_cast<const int32_t*>(p)[i];
}
// Token of the teacher's entry j of row n, or -1, and its value.
__device__ inline int entry(const Distill& a, int64_t n, int j, float& t) {
  const int64_t id = load_id(a.ids, a.id_bytes, n * a.K + j);
  t = load_as(a.values, a.vtype, n * a.K + j);
  return id >= 0 && id < a.V && t != -INFINITY ? (int)id : -1;
}
__device__ inline int label_of(const Distill& a, int64_t n) {
  if (!a.labels) return -1;
  const int64_t y = load_id(a.labels, a.label_bytes, n);
  return y >= 0 && y < a.V ? (int)y : -1;
}

struct Sums {   // maximum and sums of exp((s - m) / T), exp(s - m)
  float m, z, z1;
};
// exp2((from - to) c) for a change of the maximum; a maximum of -inf has sums of 0.
__device__ inline Sums join(Sums a, Sums b, float c) {
  const float m = fmaxf(a.m, b.m), r = m == -INFINITY ? 0.0f : m;
  const float fa = (a.m - r), fb = (b.m - r);
  return {m, a.z * exp2f(fa * c) + b.z * exp2f(fb * c), a.z1 * exp2f(fa * kLog2e) + b.z1 * exp2f(fb * kLog2e)};
}

template <int DT, class F>
__device__ inline void each_in(const typename TabType<DT>::t* row, int64_t a, int64_t b, int threads, F f) {
  for (int64_t i = a + threadIdx.x; i < b; i += threads) f(i, tab_get<DT>(row[i]));
}

template <int TH>
__device__ inline Sums block_sums(Sums v, float c, Sums* part) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v = join(v, Sums{__shfl_xor(v.m, d), __shfl_xor(v.z, d), __shfl_xor(v.z1, d)}, c);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[0];
  for (int w = 1; w < TH / 64; ++w) v = join(v, part[w], c);
  __syncthreads();
  return v;
}

// The row's loss and what is kept of it, from its sums.
template <int DT, int TH>
__device__ inline void finish_row(const Distill& a, int64_t n, Sums s, float* part, float* loss, float* kept, float& a_s,
                                  float& a_h, float& top, float& rtot) {
  const auto* row = static_cast<const typename TabType<DT>::t*>(a.logits) + n * a.ld;
  const auto add = [](float x, float y) { return x + y; };
  top = -INFINITY;
  bool any = false, nan = false;
  for (int j = threadIdx.x; j < a.K; j += TH) {
    float t;
    if (entry(a, n, j, t) >= 0) {
      any = true;
      nan |= t != t;
      top = fmaxf(top, t);
    }
  }
  top = block_reduce<TH>(top, part, [](float x, float y) { return fmaxf(x, y); });
  const float some = block_reduce<TH>(any ? 1.0f : 0.0f, part, add);
  const float bad = block_reduce<TH>(nan ? 1.0f : 0.0f, part, add);
  const bool alive = s.z != 0.0f;   // a NaN stays
  const int y = label_of(a, n);
  const bool soft = some > 0.0f && alive, hard = y >= 0 && alive;
  float tot = 0.0f;
  for (int j = threadIdx.x; j < a.K; j += TH) {
    float t;
    if (entry(a, n, j, t) >= 0) tot += expf((t - top) * a.inv_t);
  }
  tot = block_reduce<TH>(tot, part, add);
  rtot = bad > 0.0f ? NAN : 1.0f / tot;
  const float logs = logf(s.z) - logf(tot);
  float l = 0.0f;
  for (int j = threadIdx.x; j < a.K; j += TH) {
    float t;
    const int i = entry(a, n, j, t);
    if (i < 0) continue;
    const float q = expf((t - top) * a.inv_t) * rtot;
    if (q != 0.0f) l += q * ((t - top) * a.inv_t - (tab_get<DT>(row[i]) - s.m) * a.inv_t + logs);
  }
  l = block_reduce<TH>(l, part, add);
  const float share = a.labels ? 1.0f - a.alpha : 1.0f;
  a_s = soft ? share * a.T : 0.0f;
  a_h = hard ? a.alpha : 0.0f;
  if (threadIdx.x == 0) {
    float v = soft ? share * a.T * a.T * l : 0.0f;
    if (hard) v += a.alpha * (logf(s.z1) - (tab_get<DT>(row[y]) - s.m));
    loss[n] = v;
    if (kept) {
      float* k = kept + n * kKept;
      k[0] = s.m, k[1] = 1.0f / s.z, k[2] = 1.0f / s.z1, k[3] = top, k[4] = rtot, k[5] = a_s, k[6] = a_h;
      k[7] = some > 0.0f || y >= 0 ? 1.0f : 0.0f;
    }
  }
}

template <int DT>
__global__ void __launch_bounds__(256) distill_fwd_kernel(Distill a, float* loss, float* kept) {
  __shared__ Sums parts[4];
  __shared__ float part[4];
  const int64_t n = blockIdx.x;
  const auto* row = static_cast<const typename TabType<DT>::t*>(a.logits) + n * a.ld;
  const float c = a.inv_t * kLog2e;
  Sums s{-INFINITY, 0.0f, 0.0f};
  each_in<DT>(row, 0, a.V, 256, [&](int64_t, float x) {
    const float m = fmaxf(s.m, x), r = m == -INFINITY ? 0.0f : m;
    s.z = s.z * exp2f((s.m - r) * c) + exp2f((x - r) * c);
    s.z1 = s.z1 * exp2f((s.m - r) * kLog2e) + exp2f((x - r) * kLog2e);
    s.m = m;
  });
  s = block_sums<256>(s, c, parts);
  float a_s, a_h, top, rtot;
  finish_row<DT, 256>(a, n, s, part, loss, kept, a_s, a_h, top, rtot);
}

// Sum of the rows' losses, or over the rows that count: out[0]; out[1] is what an upstream gradient is multiplied by.
__global__ void __launch_bounds__(1024) distill_mean_kernel(const float* loss, const float* kept, int64_t N, int mean, float* out,
                                                            float* factor) {
  __shared__ double part[16];
  double s = 0.0, c = 0.0;
  for (int64_t n = threadIdx.x; n < N; n += 1024) {
    s += (double)loss[n];
    c += (double)kept[n * kKept + 7];
  }
  const auto add = [](double x, double y) { return x + y; };
  s = block_reduce<1024>(s, part, add);
  c = block_reduce<1024>(c, part, add);
  if (threadIdx.x == 0) {
    const double f = mean ? 1.0 / fmax(c, 1.0) : 1.0;
    out[0] = (float)(s * f);
    *factor = (float)f;
  }
}

// grad of `chunk` logits of a row: all of them from their probabilities, then those that the teacher or the label
// names once more, each by the first entry that names it.
template <int DT>
__global__ void __launch_bounds__(256)
distill_bwd_kernel(Distill a, const float* kept, const float* upstream, int per_row, const float* factor, float scale, int64_t chunk,
                   int chunks, void* grad) {
  __shared__ int id[kMaxEntries + 1];
  __shared__ float share[kMaxEntries + 1];
  const int64_t n = blockIdx.x / chunks, from = (blockIdx.x % chunks) * chunk, to = min(a.V, from + chunk);
  const auto* row = static_cast<const typename TabType<DT>::t*>(a.logits) + n * a.ld;
  auto* out = static_cast<typename TabType<DT>::t*>(grad) + n * a.V;
  const float* k = kept + n * kKept;
  float g = scale;
  if (upstream) g *= upstream[per_row ? n : 0];
  if (factor) g *= *factor;
  const float m = k[0], top = k[3], rtot = k[4], c = a.inv_t * kLog2e;
  const float a_s = k[5], a_h = k[6], w = g * a_s * k[1], w1 = g * a_h * k[2];
  if (g == 0.0f || (a_s == 0.0f && a_h == 0.0f)) {
    for (int64_t i = from + threadIdx.x; i < to; i += 256) out[i] = tab_put<DT>(0.0f);
    return;
  }
  const auto at = [&](float x) {
    float v = 0.0f;
    if (a_s != 0.0f) v = w * exp2f((x - m) * c);
    if (a_h != 0.0f) v += w1 * exp2f((x - m) * kLog2e);
    return v;
  };
  for (int j = threadIdx.x; j < a.K; j += 256) {
    float t;
    const int i = a_s != 0.0f ? entry(a, n, j, t) : -1;
    id[j] = i;
    share[j] = i < 0 ? 0.0f : g * a_s * expf((t - top) * a.inv_t) * rtot;
  }
  if (threadIdx.x == 0) id[a.K] = a_h != 0.0f ? label_of(a, n) : -1, share[a.K] = g * a_h;
  each_in<DT>(row, from, to, 256, [&](int64_t i, float x) { out[i] = tab_put<DT>(at(x)); });
  __syncthreads();
  for (int j = threadIdx.x; j <= a.K; j += 256) {
    const int i = id[j];
    if (i < from || i >= to) continue;
    float q = 0.0f;
    bool first = true;
    for (int o = 0; o <= a.K; ++o) {
      if (id[o] != i) continue;
      first &= o >= j;
      q += share[o];
    }
    if (first) out[i] = tab_put<DT>(at(tab_get<DT>(row[i])) - q);
  }
}

}  // namespace slg

using namespace slg;

namespace {

template <class F>
void by_type(int dtype, F f) {
  if (dtype == kTabF32) f(std::integral_constant<int, kTabF32>{});
  else if (dtype == kTabBf16) f(std::integral_constant<int, kTabBf16>{});
  else f(std::integral_constant<int, kTabF16>{});
}

int check(const Distill& a, int dtype, const char* name) {
  SLG_REQUIRE((a.logits && a.values && a.ids) || a.N == 0, SLG_E_ARG, "%s: null pointer", name);
  SLG_REQUIRE(dtype >= 0 && dtype <= 2 && a.vtype >= 0 && a.vtype <= 2, SLG_E_ARG, "%s: types %d and %d", name, dtype, a.vtype);
  SLG_REQUIRE((a.id_bytes == 4 || a.id_bytes == 8) && (!a.labels || a.label_bytes == 4 || a.label_bytes == 8), SLG_E_ARG,
              "%s: ids of %d bytes, labels of %d", name, a.id_bytes, a.label_bytes);
  SLG_REQUIRE(a.T >= 1e-4f && a.T <= 1e4f, SLG_E_ARG, "%s: temperature %g outside [1e-4, 1e4]", name, (double)a.T);
  SLG_REQUIRE(a.alpha >= 0.0f && a.alpha <= 1.0f, SLG_E_ARG, "%s: alpha %g outside [0, 1]", name, (double)a.alpha);
  SLG_REQUIRE(a.N >= 0 && a.N < (1LL << 31) && a.V >= 1 && a.V < (1LL << 31) && a.ld >= 0 && a.K >= 1 && a.K <= kMaxEntries,
              SLG_E_SHAPE, "%s: N %lld, V %lld, K %d", name, (long long)a.N, (long long)a.V, a.K);
  return 0;
}

Distill args(const void* logits, int64_t N, int64_t V, int64_t ld, const void* values, int32_t vtype, const void* ids, int32_t id_bytes,
             int32_t K, const void* labels, int32_t label_bytes, float T, float alpha) {
  return {logits, N, V, ld, values, vtype, ids, id_bytes, K, labels, label_bytes, T, 1.0f / T, alpha};
}

// grid of the gradient: rows in chunks of 8192 logits
constexpr int64_t kChunk = 8192;

}  // namespace

extern "C" {

int64_t slg_distill_kept(int64_t N) { return N < 0 || N >= (1LL << 31) ? -1 : N * (kKept + 1) + 1; }

int slg_distill_fwd(const void* logits, int32_t dtype, int64_t N, int64_t V, int64_t ld, const void* values, int32_t vtype,
                    const void* ids, int32_t id_bytes, int32_t K, const void* labels, int32_t label_bytes, float T, float alpha,
                    int32_t reduction, float* loss, float* kept, slg_stream_t stream) {
  const Distill a = args(logits, N, V, ld, values, vtype, ids, id_bytes, K, labels, label_bytes, T, alpha);
  if (const int rc = check(a, dtype, "distill_fwd")) return rc;
  SLG_REQUIRE(reduction >= 0 && reduction <= 2, SLG_E_ARG, "distill_fwd: reduction %d", reduction);
  SLG_REQUIRE(((loss || N == 0) && kept) || (N == 0 && !reduction), SLG_E_ARG, "distill_fwd: null pointer");
  if (N == 0 && !reduction) return 0;
  hipStream_t st = as_stream(stream);
  float *rows = reduction ? kept + N * kKept : loss, *factor = kept + N * (kKept + 1);
  if (N)
    by_type(dtype, [&](auto dt) {
      hipLaunchKernelGGL((distill_fwd_kernel<decltype(dt)::value>), dim3((unsigned)N), dim3(256), 0, st, a, rows, kept);
    });
  if (reduction)
    hipLaunchKernelGGL(distill_mean_kernel, dim3(1), dim3(1024), 0, st, rows, kept, N, reduction == 2, loss, factor);
  SLG_LAUNCH_CHECK("distill_fwd");
  return 0;
}

int slg_distill_bwd(const void* logits, int32_t dtype, int64_t N, int64_t V, int64_t ld, const void* values, int32_t vtype,
                    const void* ids, int32_t id_bytes, int32_t K, const void* labels, int32_t label_bytes, float T, float alpha,
                    int32_t reduction, const float* kept, const float* upstream, float scale, void* grad, slg_stream_t stream) {
  const Distill a = args(logits, N, V, ld, values, vtype, ids, id_bytes, K, labels, label_bytes, T, alpha);
  if (const int rc = check(a, dtype, "distill_bwd")) return rc;
  SLG_REQUIRE(reduction >= 0 && reduction <= 2, SLG_E_ARG, "distill_bwd: reduction %d", reduction);
  SLG_REQUIRE((kept && grad) || N == 0, SLG_E_ARG, "distill_bwd: null pointer");
  const int64_t chunks = cdiv(V, kChunk);
  SLG_REQUIRE(N * chunks < (1LL << 31), SLG_E_SHAPE, "distill_bwd: N %lld, V %lld", (long long)N, (long long)V);
  if (N == 0) return 0;
  by_type(dtype, [&](auto dt) {
    hipLaunchKernelGGL((distill_bwd_kernel<decltype(dt)::value>), dim3((unsigned)(N * chunks)), dim3(256), 0, as_stream(stream), a,
                       kept, upstream, reduction == 0, reduction ? kept + N * (kKept + 1) : nullptr, scale, kChunk, (int)chunks, grad);
  });
  SLG_LAUNCH_CHECK("distill_bwd");
  return 0;
}

int slg_distill_loss_grad(const void* logits, int32_t dtype, int64_t N, int64_t V, int64_t ld, const void* values, int32_t vtype,
                          const void* ids, int32_t id_bytes, int32_t K, const void* labels, int32_t label_bytes, float T, float alpha,
                          int32_t reduction, float scale, float* loss, void* grad, float* kept, slg_stream_t stream) {
  SLG_REQUIRE(grad || N == 0, SLG_E_ARG, "distill_loss_grad: null pointer");
  SLG_REQUIRE(isfinite(scale), SLG_E_ARG, "distill_loss_grad: scale %g", (double)scale);
  if (const int rc = slg_distill_fwd(logits, dtype, N, V, ld, values, vtype, ids, id_bytes, K, labels, label_bytes, T, alpha, reduction,
                                     loss, kept, stream))
    return rc;
  return slg_distill_bwd(logits, dtype, N, V, ld, values, vtype, ids, id_bytes, K, labels, label_bytes, T, alpha, reduction, kept,
                         nullptr, scale, grad, stream);
}

}  // extern "C"
