// The loss of a student's logits against a teacher's largest ones, with its gradient (gfx950). Row s of V logits,
// the teacher's values t_j at tokens i_j (K of them), temperature T:
//   q_j  = softmax(t / T) over the entries that are there: an id in 0..V-1 and a value other than -inf
//   p    = softmax(s / T),  p1 = softmax(s)
//   loss = a_s T^2 sum_j q_j (log q_j - log p[i_j]) - a_h log p1[label]
//   grad = a_s T (p - sum of q_j with i_j = .) + a_h (p1 - [. = label])
// a_s = 1 - alpha and a_h = alpha with labels, else 1 and 0. A term whose entries or label are missing, or whose
// share is 0, counts 0 whatever its values are, and so does a row of logits that are all -inf; "mean" is over the
// rows that have an entry or a label. A token named twice gets both entries' probabilities, and the loss both terms
// of the sum over entries.
//
// Both softmaxes share their maximum m: what is kept of a row is m, 1/Z and 1/Z1 (and the teacher's own), so that a
// probability is exp((s - m) / T) / Z with the difference exact where it matters. Sums are fp32, those over rows 64
// bits; the gradient is rounded once. With long rows all kernels are bound by the logits' bytes: one pass for the
// loss (the running maximum and sums of each thread joined at the end), another with the write for the gradient. Both
// from one call hold the row in registers between them. Times below are of 4096 x 32000 and 64 entries, on a card
// whose copies reach 5.0 to 5.4 TB/s.
//
// Roundings: an exponential's argument (s - m) log2 e / T takes four (the difference, 1 / T, the factor, the product) and
// the exponential one, so that a probability is off by some 2^-22 of itself times 1 + (m - s) / T, and by its row's sum,
// which chains of V / threads additions and as many rescaled maxima make. Under 2^-126 of the largest it is 0.
#include <algorithm>
#include <type_traits>

#include "block_ops.h"
#include "float_types.h"

namespace slg {

constexpr float kLog2e = 1.44269504f;
constexpr int kMaxEntries = 1024;
constexpr int kKept = 8;      // floats kept of a row: m, 1/Z, 1/Z1, the teacher's maximum and 1/sum, a_s T, a_h, counted
constexpr int kCounts = 256;  // workgroups that count the rows of a mean
// More rows than these are summed by kCounts workgroups before the last one: the loss of 32768 x 49 takes 25 us so and 38
// without, of 16384 x 49 17 and 22, of 250 x 257 9 and 7.
constexpr int kManyRows = 16384;
// Past this temperature a small soft loss is summed without cancellation (close_loss): the factor T^2 would bring the
// roundings of the logarithms, some 2^-20, to the loss's own size at T = 1000. Up to it they come to 2^-16 at most.
constexpr float kFarT = 4.0f;
constexpr int kParts = 1024;  // parts of rows that the loss's first pass is cut into where there are fewer rows

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

__device__ __forceinline__ float load_as(const void* p, int dtype, int64_t i) {
  if (dtype == kTabF32) return static_cast<const float*>(p)[i];
  if (dtype == kTabBf16) return tab_get<kTabBf16>(static_cast<const uint16_t*>(p)[i]);
  return (float)static_cast<const _Float16*>(p)[i];
}
__device__ __forceinline__ int64_t load_id(const void* p, int bytes, int64_t i) {
  return bytes == 8 ? static_cast<const int64_t*>(p)[i] : (int64_t)static_cast<const int32_t*>(p)[i];
}
// Token of the teacher's entry j of row n, or -1, and its value.
__device__ __forceinline__ int entry(const Distill& a, int64_t n, int j, float& t) {
  const int64_t id = load_id(a.ids, a.id_bytes, n * a.K + j);
  t = load_as(a.values, a.vtype, n * a.K + j);
  return id >= 0 && id < a.V && t != -INFINITY ? (int)id : -1;
}
__device__ __forceinline__ int label_of(const Distill& a, int64_t n) {
  if (!a.labels) return -1;
  const int64_t y = load_id(a.labels, a.label_bytes, n);
  return y >= 0 && y < a.V ? (int)y : -1;
}

// The soft term's share of the loss.
__device__ __forceinline__ float soft_share(const Distill& a) { return a.labels ? 1.0f - a.alpha : 1.0f; }

// Under 2^-126 it is 0.
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Which exponentials are summed: of one softmax, of two, or of two at temperature 2, where one is the other's square.
enum Form { kOne, kTwo, kSquare };

struct Sums {   // maximum and sums of exp((s - m) / T), exp(s - m)
  float m, z, z1;
};
// A maximum of -inf has sums of 0; of a NaN they are NaN.
__device__ __forceinline__ Sums join(Sums a, Sums b, float c) {
  const float m = fmaxf(a.m, b.m), r = m == -INFINITY ? 0.0f : m;
  const float fa = a.m - r, fb = b.m - r;
  return {m, a.z * exp2_fast(fa * c) + b.z * exp2_fast(fb * c), a.z1 * exp2_fast(fa * kLog2e) + b.z1 * exp2_fast(fb * kLog2e)};
}

// Groups of 16 bytes of a row, from any element on.
template <int DT>
struct Group {
  using T = typename TabType<DT>::t;
  static constexpr int U = 16 / (int)sizeof(T);
  typedef T Vec __attribute__((ext_vector_type(U), aligned(sizeof(T))));
  static __device__ __forceinline__ void get(const T* p, float (&v)[U]) {
    const Vec x = *reinterpret_cast<const Vec*>(p);
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = tab_get<DT>(x[u]);
  }
  static __device__ __forceinline__ T round(float v) {
    if constexpr (DT == kTabBf16) return __builtin_bit_cast(uint16_t, (__bf16)v);
    else return (T)v;
  }
  static __device__ __forceinline__ void put(T* p, const float (&v)[U]) {
    Vec x;
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = round(v[u]);
    __builtin_nontemporal_store(x, reinterpret_cast<Vec*>(p));
  }
};

template <Form FORM>
__device__ __forceinline__ void add_exp(float d, float c, float& z, float& z1) {
  const float e = exp2_fast(d * c);
  z += e;
  if (FORM == kTwo) z1 += exp2_fast(d * kLog2e);
  if (FORM == kSquare) z1 = fmaf(e, e, z1);
}

// n more values of the running sums.
template <Form FORM, int n>
__device__ __forceinline__ void take(Sums& s, const float (&v)[n], float c) {
  float m = s.m;
#pragma unroll
  for (int u = 0; u < n; ++u) m = fmaxf(m, v[u]);
  const float r = m == -INFINITY ? 0.0f : m;
  s.z *= exp2_fast((s.m - r) * c);
  if (FORM != kOne) s.z1 *= exp2_fast((s.m - r) * kLog2e);
  s.m = m;
#pragma unroll
  for (int u = 0; u < n; ++u) add_exp<FORM>(v[u] - r, c, s.z, s.z1);
}

// Sums of the row's values from `from` to `to` by TH threads, four groups of a thread in flight.
template <int DT, int TH, Form FORM>
__device__ __forceinline__ Sums sums_of(const typename TabType<DT>::t* row, int64_t from, int64_t to, float c) {
  using G = Group<DT>;
  constexpr int64_t kStep = (int64_t)TH * G::U;
  Sums s{-INFINITY, 0.0f, 0.0f};
  int64_t i = from + (int64_t)threadIdx.x * G::U;
  for (; i + 3 * kStep + G::U <= to; i += 4 * kStep) {
    float v[4][G::U];
#pragma unroll
    for (int k = 0; k < 4; ++k) G::get(row + i + k * kStep, v[k]);
#pragma unroll
    for (int k = 0; k < 4; ++k) take<FORM>(s, v[k], c);
  }
  for (; i + G::U <= to; i += kStep) {
    float v[G::U];
    G::get(row + i, v);
    take<FORM>(s, v, c);
  }
  if (i < to) {   // the row's end, in one thread
    for (int64_t k = i; k < to; ++k) {
      const float v[1] = {tab_get<DT>(row[k])};
      take<FORM>(s, v, c);
    }
  }
  return s;
}

template <int TH>
__device__ __forceinline__ Sums block_sums(Sums v, float c, Sums* part) {
  constexpr int W = TH / 64;
  const auto both = [&](Sums x, Sums y) { return join(x, y, c); };
  v = lanes_reduce(v, both);
  if constexpr (W > 1) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lanes_reduce<W>(part[threadIdx.x & (W - 1)], both);
  }
  return v;
}

// A row's entries in LDS, sized by K: their tokens, shares and the shares' logs, and for the gradient a table of the
// tokens that are named: open addressing, at most half full. Of a token's entries the first one writes its gradient.
// (Each entry compared with each other: 256 entries of 8192 x 500 bf16 took 167 us with the loss, 195 by itself, where
// the table takes 36 and 20; at one entry both take the same.)
struct Entries {
  static constexpr int kNone = 0x7fffffff;   // no token
  int K, mask;
  int* id;
  float *share, *log;
  int *slot, *key, *first;   // of an entry, or -1; of a slot: its token, negative (by 2^31) if several entries name it
  __device__ __forceinline__ Entries(int k, int slots) : K(k), mask(slots - 1) {
    extern __shared__ float entries[];
    id = reinterpret_cast<int*>(entries);
    share = entries + K;
    log = share + K;
    slot = reinterpret_cast<int*>(log + K);
    key = slot + K;
    first = key + slots;
  }
  // By `threads` threads, of which this is the `own`th; then a barrier, where it is not one wave.
  __device__ __forceinline__ void clear(int own, int threads) const {
    for (int i = own; i <= mask; i += threads) key[i] = kNone, first[i] = kNone;
  }
  __device__ __forceinline__ int place(int token) const { return (int)((uint32_t)token * 0x9e3779b1u >> 7) & mask; }
  // Entry j names `token` (-1: none). At the next barrier the table knows.
  __device__ __forceinline__ void name(int j, int token) const {
    int at = token < 0 ? -1 : place(token);
    if (token >= 0) {
      for (;; at = (at + 1) & mask) {
        const int was = atomicCAS(&key[at], kNone, token);
        if (was == kNone || (was & kNone) == token) break;
      }
      if (atomicMin(&first[at], j) != kNone) atomicOr(&key[at], ~kNone);
    }
    slot[j] = at;
  }
  __device__ __forceinline__ bool named(int token) const {
    for (int at = place(token); key[at] != kNone; at = (at + 1) & mask)
      if ((key[at] & kNone) == token) return true;
    return false;
  }
};

struct Teacher {   // maximum and sum of its entries, and whether there are any
  float top, total;
  bool some;
};

// One wave: the teacher's tokens and probabilities (not yet over `total`) into id[] and q[], their logs into lq[].
__device__ __forceinline__ Teacher teacher_of(const Distill& a, int64_t n, int* id, float* q, float* lq) {
  const int lane = threadIdx.x & 63;
  float top = -INFINITY, total = 0.0f;
  bool any = false;
  for (int j = lane; j < a.K; j += 64) {
    float t;
    const int i = entry(a, n, j, t);
    id[j] = i;
    q[j] = t;
    any |= i >= 0;
    if (i >= 0) top = fmaxf(top, t);
  }
  top = wave_reduce(top, [](float x, float y) { return fmaxf(x, y); });
  for (int j = lane; j < a.K; j += 64) {
    const float l = (q[j] - top) * a.inv_t, e = id[j] >= 0 ? expf(l) : 0.0f;
    q[j] = e;
    lq[j] = l;
    total += e;
  }
  total = wave_reduce(total, [](float x, float y) { return x + y; });
  return {top, total, __ballot(any) != 0};
}

// e^r - 1 - r, which is not negative; by its series where the exponential's rounding would be left of it.
__device__ __forceinline__ float past_tangent(float r) {
  if (!(fabsf(r) < 0.5f)) return expf(r) - 1.0f - r;
  float p = 1.0f / 362880.0f;
  p = fmaf(p, r, 1.0f / 40320.0f);
  p = fmaf(p, r, 1.0f / 5040.0f);
  p = fmaf(p, r, 1.0f / 720.0f);
  p = fmaf(p, r, 1.0f / 120.0f);
  p = fmaf(p, r, 1.0f / 24.0f);
  p = fmaf(p, r, 1.0f / 6.0f);
  return r * r * fmaf(p, r, 0.5f);
}

// One wave: sum_j q_j (log q_j - log p[i_j]) where that is small beside its terms. With r_j = log(p[i_j] / q_j) it is
//   sum_j q_j (e^(r_j) - 1 - r_j) + 1 - sum_j p[i_j]:
// no term of the sum is negative, and the rest is what the tokens that no entry names have, here summed in 64 bits of
// the same exponentials as the named ones' (0 where all are named once). An error of both softmaxes' sums then counts by
// its square. False, and nothing, where the entries name half of p or less: the loss is log 2 at least, and its terms'
// own roundings are small beside it.
template <int DT>
__device__ __forceinline__ bool close_loss(const Distill& a, const typename TabType<DT>::t* row, const Sums& s, float rtot, const int* id,
                                           const float* q, const float* lq, float& loss) {
  const int lane = threadIdx.x & 63;
  const auto add = [](double x, double y) { return x + y; };
  const auto mass_of = [&](float x) { return (double)exp2_fast((x - s.m) * (a.inv_t * kLog2e)); };
  const auto mass = [&](int64_t i) { return mass_of(tab_get<DT>(row[i])); };
  double named = 0.0, total = 0.0, all = 0.0;
  for (int j = lane; j < a.K; j += 64)
    if (q[j] != 0.0f) named += mass(id[j]), total += (double)q[j];
  named = wave_reduce(named, add);
  if (!(named > 0.5 * (double)s.z)) return false;
  total = wave_reduce(total, add);
  int64_t i = lane;
  // two loads in flight: with four the forms of 512 threads lose a workgroup a compute unit to registers
  for (; i + 64 < a.V; i += 2 * 64) {
    float v[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) v[k] = tab_get<DT>(row[i + k * 64]);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      __builtin_amdgcn_sched_barrier(0);
      all += mass_of(v[k]);
    }
  }
  for (; i < a.V; i += 64) all += mass(i);
  all = wave_reduce(all, add);
  const float shift = (float)log(all / total);
  float l = 0.0f;
  for (int j = lane; j < a.K; j += 64)
    if (q[j] != 0.0f) l += q[j] * rtot * past_tangent((tab_get<DT>(row[id[j]]) - s.m) * a.inv_t - lq[j] - shift);
  l = wave_reduce(l, [](float x, float y) { return x + y; });
  loss = l + (float)((all - named) / all);
  return true;
}

// One wave: the row's loss from its sums, and what is kept of it.
template <int DT>
__device__ __forceinline__ void finish_row(const Distill& a, int64_t n, const Sums& s, const Teacher& t, const int* id, const float* q,
                                           const float* lq, float* loss, float* kept) {
  const auto* row = static_cast<const typename TabType<DT>::t*>(a.logits) + n * a.ld;
  const int lane = threadIdx.x & 63, y = label_of(a, n);
  const bool alive = s.z != 0.0f;   // a NaN stays
  const float share = soft_share(a);
  const bool soft = t.some && alive && share != 0.0f, hard = y >= 0 && alive && a.alpha != 0.0f;
  const float rtot = 1.0f / t.total, logs = logf(s.z) - logf(t.total);
  float l = 0.0f;
  if (soft && !(a.T > kFarT && close_loss<DT>(a, row, s, rtot, id, q, lq, l))) {
    for (int j = lane; j < a.K; j += 64) {
      const float e = q[j];
      if (e != 0.0f) l += e * rtot * (lq[j] - (tab_get<DT>(row[id[j]]) - s.m) * a.inv_t + logs);
    }
    l = wave_reduce(l, [](float x, float y) { return x + y; });
  }
  if (lane == 0) {
    float v = soft ? share * a.T * a.T * l : 0.0f;
    if (hard) v += a.alpha * (logf(s.z1) - (tab_get<DT>(row[y]) - s.m));
    loss[n] = v;
    if (kept) {
      float4* k = reinterpret_cast<float4*>(kept + n * kKept);
      k[0] = {s.m, 1.0f / s.z, 1.0f / s.z1, t.top};
      k[1] = {rtot, soft ? share * a.T : 0.0f, hard ? a.alpha : 0.0f, t.some || y >= 0 ? 1.0f : 0.0f};
    }
  }
}

// The loss of a row, a workgroup each; with parts > 1 the sums of a part of a row, joined by the next kernel. 108 us
// in fp32, 4.9 TB/s, 65 in bf16 with labels: memory; the vector instructions take about a third of their issue. Of 16
// x 131071 fp16 logits in 63 parts 4.8 us, and 4.1 for the join: latency.
template <int DT, int TH, Form FORM>
__global__ void __launch_bounds__(TH) distill_fwd_kernel(Distill a, int parts, int64_t per, Sums* part_sums, float* loss, float* kept) {
  __shared__ Sums part[TH / 64];
  const Entries e(a.K, 1);
  const uint32_t b = block_id();
  const int64_t n = b / (uint32_t)parts, p = b % (uint32_t)parts;
  if (n >= a.N) return;
  const auto* row = static_cast<const typename TabType<DT>::t*>(a.logits) + n * a.ld;
  const float c = a.inv_t * kLog2e;
  Sums s = sums_of<DT, TH, FORM>(row, p * per, min(a.V, (p + 1) * per), c);
  Teacher t{};
  if (parts == 1 && threadIdx.x < 64) t = teacher_of(a, n, e.id, e.share, e.log);
  s = block_sums<TH>(s, c, part);
  if (FORM == kOne) s.z1 = s.z;
  if (parts > 1) {
    if (threadIdx.x == 0) part_sums[b] = s;
  } else if (threadIdx.x < 64) {
    finish_row<DT>(a, n, s, t, e.id, e.share, e.log, loss, kept);
  }
}
template <int DT>
__global__ void __launch_bounds__(64) distill_join_kernel(Distill a, int parts, const Sums* part_sums, float* loss, float* kept) {
  const Entries e(a.K, 1);
  const int64_t n = blockIdx.x;
  const float c = a.inv_t * kLog2e;
  Sums s{-INFINITY, 0.0f, 0.0f};
  for (int p = threadIdx.x; p < parts; p += 64) s = join(s, part_sums[n * parts + p], c);
  const Teacher t = teacher_of(a, n, e.id, e.share, e.log);
  s = block_sums<64>(s, c, nullptr);
  finish_row<DT>(a, n, s, t, e.id, e.share, e.log, loss, kept);
}

// Rows with an entry or a label, counted by kCounts workgroups of four waves: a lane a row while the label or the first
// entry is there, a wave a row where not.
__global__ void __launch_bounds__(256) distill_count_kernel(Distill a, int* counts) {
  __shared__ int part[4];
  constexpr int64_t kWaves = kCounts * 4;
  const int lane = threadIdx.x & 63;
  const int64_t per = min((int64_t)64, (a.N + kWaves - 1) / kWaves);
  int c = 0;
  for (int64_t first = ((int64_t)blockIdx.x * 4 + wave_id()) * per; first < a.N; first += kWaves * per) {
    const int64_t n = first + lane;
    const bool own = lane < per && n < a.N;
    bool any = false;
    if (own) {
      float t;
      const bool hard = label_of(a, n) >= 0, soft = entry(a, n, 0, t) >= 0;
      any = hard || soft;
    }
    c += __popcll(__ballot(any));
    for (uint64_t left = __ballot(own && !any); left; left &= left - 1) {
      const int64_t row = first + __builtin_ctzll(left);
      bool some = false;
      for (int j = lane; !__ballot(some) && j - lane < a.K; j += 64) {
        float t;
        some = j < a.K && entry(a, row, j, t) >= 0;
      }
      c += __ballot(some) != 0;
    }
  }
  c = block_reduce<256>(lane == 0 ? c : 0, part, [](int x, int y) { return x + y; });
  if (threadIdx.x == 0) counts[blockIdx.x] = c;
}

// Sum of the rows' losses, or their mean over the rows that count (by `counts`, or where that is null by what is
// kept of the rows), and what an upstream gradient is multiplied by. One workgroup, behind another kernel that sums the
// rows in kCounts runs where there are many.
__global__ void __launch_bounds__(256) distill_sum_kernel(const float* loss, const float* kept, int64_t N, double2* sums) {
  __shared__ double part[4];
  const int64_t per = (N + kCounts - 1) / kCounts, from = blockIdx.x * per, to = min(N, from + per);
  double s = 0.0, c = 0.0;
#pragma unroll 4
  for (int64_t n = from + threadIdx.x; n < to; n += 256) {
    s += (double)loss[n];
    if (kept) c += (double)kept[n * kKept + 7];
  }
  const auto add = [](double x, double y) { return x + y; };
  s = block_reduce<256>(s, part, add);
  c = block_reduce<256>(c, part, add);
  if (threadIdx.x == 0) sums[blockIdx.x] = {s, c};
}
__global__ void __launch_bounds__(1024) distill_mean_kernel(const float* loss, const float* kept, const double2* sums, const int* counts,
                                                            int64_t N, int mean, float* out, float* factor) {
  __shared__ double part[16];
  double s = 0.0, c = 0.0;
  if (sums) {
    if (threadIdx.x < kCounts) s = sums[threadIdx.x].x, c = sums[threadIdx.x].y;
  } else {
#pragma unroll 4
    for (int64_t n = threadIdx.x; n < N; n += 1024) {
      s += (double)loss[n];
      if (kept) c += (double)kept[n * kKept + 7];
    }
  }
  if (counts && threadIdx.x < kCounts) c = (double)counts[threadIdx.x];
  const auto add = [](double x, double y) { return x + y; };
  s = block_reduce<1024>(s, part, add);
  if (mean) c = block_reduce<1024>(c, part, add);
  if (threadIdx.x == 0) {
    const double f = mean ? 1.0 / fmax(c, 1.0) : 1.0;
    out[0] = (float)(s * f);
    *factor = (float)f;
  }
}

// A logit's gradient but for the entries that name it.
struct Slope {
  float m, c, w, w1;
  template <Form FORM>
  __device__ __forceinline__ float at(float x) const {
    const float d = x - m, e = exp2_fast(d * c);
    if (FORM == kSquare) return e * fmaf(w1, e, w);
    const float v = w * e;
    return FORM == kTwo ? fmaf(w1, exp2_fast(d * kLog2e), v) : v;
  }
};
// Of a row with shares ws and wh. With one of them 0, or at temperature 1, one softmax is enough.
__device__ __forceinline__ Slope slope_of(const Distill& a, float m, float rz, float rz1, float ws, float wh, Form& form) {
  const float c = a.inv_t * kLog2e;
  form = kOne;
  if (wh == 0.0f) return {m, c, ws * rz, 0.0f};
  if (ws == 0.0f) return {m, kLog2e, wh * rz1, 0.0f};
  if (a.T == 1.0f) return {m, kLog2e, (ws + wh) * rz1, 0.0f};
  form = a.T == 2.0f ? kSquare : kTwo;
  return {m, c, ws * rz, wh * rz1};
}
// f with a row's form, the same in all threads.
template <class F>
__device__ __forceinline__ void by_row_form(Form form, F f) {
  if (form == kOne) f(std::integral_constant<Form, kOne>{});
  else if (form == kSquare) f(std::integral_constant<Form, kSquare>{});
  else f(std::integral_constant<Form, kTwo>{});
}

// A barrier at which all waves' stores have arrived, before other threads write some of the places again.
__device__ __forceinline__ void written() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// The tokens of [from, to) that entries or the label name, written again with their shares taken off; by `threads`
// threads, of which this is the `own`th. weight * share of an entry, label_share of the label (-1: none).
template <int DT, Form FORM>
__device__ __forceinline__ void name_tokens(const typename TabType<DT>::t* row, typename TabType<DT>::t* out, const Entries& e, float weight,
                                            int label, float label_share, int64_t from, int64_t to, const Slope& slope, int own,
                                            int threads) {
  const auto write = [&](int i, float q) { out[i] = Group<DT>::round(slope.at<FORM>(tab_get<DT>(row[i])) - q); };
  for (int j = own; j < e.K; j += threads) {
    const int at = e.slot[j];
    if (at < 0 || e.first[at] != j) continue;
    const int i = e.key[at] & Entries::kNone;
    float q = weight * e.share[j];
    if (e.key[at] < 0)
      for (int o = j + 1; o < e.K; ++o) q += e.slot[o] == at ? weight * e.share[o] : 0.0f;
    write(i, i == label ? q + label_share : q);
  }
  if (own == threads - 1 && label >= from && label < to && !e.named(label)) write(label, label_share);
}

// Gradient of `chunk` logits of a row: all of them from their probabilities, then those that are named. 204 to 217 us
// in fp32, 4.8 to 5.1 TB/s of reads and writes, 113 in bf16 with labels: memory; 16 x 131071 fp16 in 63 parts 6 us.
// The second write of the few named tokens takes the place of a look at the entries by every token.
template <int DT, int TH>
__global__ void __launch_bounds__(TH)
distill_bwd_kernel(Distill a, int slots, const float* kept, const float* upstream, int per_row, const float* factor, float scale,
                   int64_t chunk, int chunks, void* grad) {
  using G = Group<DT>;
  using T = typename TabType<DT>::t;
  const Entries e(a.K, slots);
  const uint32_t b = block_id();
  const int64_t n = b / (uint32_t)chunks, from = b % (uint32_t)chunks * chunk, to = min(a.V, from + chunk);
  if (n >= a.N) return;
  const T* row = static_cast<const T*>(a.logits) + n * a.ld;
  T* out = static_cast<T*>(grad) + n * a.V;
  const float4* k = reinterpret_cast<const float4*>(kept + n * kKept);
  const float4 k0 = k[0], k1 = k[1];
  float g = scale;
  if (upstream) g *= upstream[per_row ? n : 0];
  if (factor) g *= *factor;
  const float a_s = k1.y, a_h = k1.z;
  constexpr int64_t kStep = TH * G::U;
  int64_t i = from + (int64_t)threadIdx.x * G::U;
  if (g == 0.0f || (a_s == 0.0f && a_h == 0.0f)) {
    const float v[G::U] = {};
    for (; i + G::U <= to; i += kStep) G::put(out + i, v);
    for (; i < to && i + G::U > to; ++i) out[i] = G::round(0.0f);
    return;
  }
  Form form;
  const Slope slope = slope_of(a, k0.x, k0.y, k0.z, g * a_s, g * a_h, form);
  e.clear(threadIdx.x, TH);
  __syncthreads();
  for (int j = threadIdx.x; j < a.K; j += TH) {
    float t = -INFINITY;
    const int token = a_s != 0.0f ? entry(a, n, j, t) : -1;
    e.share[j] = g * a_s * expf((t - k0.w) * a.inv_t) * k1.x;
    e.name(j, token >= from && token < to ? token : -1);
  }
  const int label = a_h != 0.0f ? label_of(a, n) : -1;
  by_row_form(form, [&](auto row_form) {
    constexpr Form FORM = decltype(row_form)::value;
    for (; i + 3 * kStep + G::U <= to; i += 4 * kStep) {
      float v[4][G::U];
#pragma unroll
      for (int q = 0; q < 4; ++q) G::get(row + i + q * kStep, v[q]);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
#pragma unroll
        for (int u = 0; u < G::U; ++u) v[q][u] = slope.at<FORM>(v[q][u]);
        G::put(out + i + q * kStep, v[q]);
      }
    }
    for (; i + G::U <= to; i += kStep) {
      float v[G::U];
      G::get(row + i, v);
#pragma unroll
      for (int u = 0; u < G::U; ++u) v[u] = slope.at<FORM>(v[u]);
      G::put(out + i, v);
    }
    for (; i < to; ++i) out[i] = G::round(slope.at<FORM>(tab_get<DT>(row[i])));
    written();
    name_tokens<DT, FORM>(row, out, e, 1.0f, label, g * a_h, from, to, slope, threadIdx.x, TH);
  });
}

// Loss and gradient of a row, a workgroup each, the row's first NV groups of each thread in registers between them.
// In bf16 with labels at T = 2 105 us of a call's 115, 5.0 TB/s: memory, with the vector instructions at some 75% of
// their issue (two passes over the row, an exponential in each). With two workgroups a compute unit one row is read
// while another is summed.
template <int DT, int TH, int NV, Form FORM>
__global__ void __launch_bounds__(TH, TH == 1024 ? 8 : 1)
distill_both_kernel(Distill a, int slots, const int* counts, float scale, float* loss, void* grad) {
  using G = Group<DT>;
  using T = typename TabType<DT>::t;
  constexpr int U = G::U;
  const Entries e(a.K, slots);
  __shared__ float part[2][TH / 64];
  __shared__ int ipart[TH / 64];
  __shared__ Teacher told;
  const int64_t n = block_id();
  if (n >= a.N) return;
  const T* row = static_cast<const T*>(a.logits) + n * a.ld;
  T* out = static_cast<T*>(grad) + n * a.V;
  const int V = (int)a.V, groups = V / U;   // whole ones; the row's last V % U values are one thread's
  const int own = V - groups * U ? (int)threadIdx.x : TH;
  typename G::Vec r[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = j * TH + threadIdx.x;
    if (at < groups) r[j] = *reinterpret_cast<const typename G::Vec*>(row + (int64_t)at * U);
  }
  const int y = label_of(a, n);
  if (threadIdx.x < 64) {
    e.clear(threadIdx.x, 64);
    const Teacher t = teacher_of(a, n, e.id, e.share, e.log);
    if (threadIdx.x == 0) told = t;
    for (int j = threadIdx.x; j < a.K; j += 64) e.name(j, soft_share(a) != 0.0f ? e.id[j] : -1);
  }
  // f(values, first token) of the thread's groups
  const auto each = [&](auto f) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = j * TH + threadIdx.x;
      if (at < groups) {
        float v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = tab_get<DT>(r[j][u]);
        f(v, at * U);
      }
    }
    for (int at = NV * TH + threadIdx.x; at < groups; at += TH) {
      float v[U];
      G::get(row + (int64_t)at * U, v);
      f(v, at * U);
    }
  };
  const auto rest = [&](auto f) {
    if (own == 0)
      for (int i = groups * U; i < V; ++i) f(tab_get<DT>(row[i]), i);
  };
  float m = -INFINITY;
  each([&](const float (&v)[U], int) {
#pragma unroll
    for (int u = 0; u < U; ++u) m = fmaxf(m, v[u]);
  });
  rest([&](float x, int) { m = fmaxf(m, x); });
  m = block_reduce<TH>(m, part[0], [](float x, float y) { return fmaxf(x, y); });
  const float c = a.inv_t * kLog2e, from = m == -INFINITY ? 0.0f : m;
  float z = 0.0f, z1 = 0.0f;
  const auto add = [&](float x) { add_exp<FORM>(x - from, c, z, z1); };
  each([&](const float (&v)[U], int) {
#pragma unroll
    for (int u = 0; u < U; ++u) add(v[u]);
  });
  rest([&](float x, int) { add(x); });
  const auto plus = [](float x, float y) { return x + y; };
  z = block_reduce<TH>(z, part[0], plus);
  z1 = FORM != kOne ? block_reduce<TH>(z1, part[1], plus) : z;
  if (counts) {
    int rows = 0;
    for (int i = threadIdx.x; i < kCounts; i += TH) rows += counts[i];
    rows = block_reduce<TH>(rows, ipart, [](int x, int y) { return x + y; });
    scale *= (float)(1.0 / (double)max(rows, 1));
  }
  if constexpr (TH == 64) __syncthreads();
  const Teacher t = told;
  const bool soft = t.some && z != 0.0f, hard = y >= 0 && z != 0.0f;   // as in finish_row
  const float a_s = soft ? soft_share(a) * a.T : 0.0f, a_h = hard ? a.alpha : 0.0f;
  const bool dead = scale == 0.0f || (a_s == 0.0f && a_h == 0.0f);
  Form form;
  const Slope slope = slope_of(a, m, 1.0f / z, 1.0f / z1, scale * a_s, scale * a_h, form);
  // a row with one share 0 takes one softmax also where the others have two
  const auto by_form_here = [&](auto f) {
    if (FORM == kOne || form == kOne) f(std::integral_constant<Form, kOne>{});
    else f(std::integral_constant<Form, FORM>{});
  };
  if (dead) {
    each([&](const float (&)[U], int i) {
      const float v[U] = {};
      G::put(out + i, v);
    });
    rest([&](float, int i) { out[i] = G::round(0.0f); });
  } else {
    by_form_here([&](auto row_form) {
      each([&](const float (&v)[U], int i) {
        float g[U];
#pragma unroll
        for (int u = 0; u < U; ++u) g[u] = slope.at<decltype(row_form)::value>(v[u]);
        G::put(out + i, g);
      });
      rest([&](float x, int i) { out[i] = G::round(slope.at<decltype(row_form)::value>(x)); });
    });
  }
  written();
  // the first wave sums the loss while the others write the tokens that are named
  if (threadIdx.x < 64) finish_row<DT>(a, n, Sums{m, z, z1}, t, e.id, e.share, e.log, loss, nullptr);
  if (!dead && (TH == 64 || threadIdx.x >= 64))
    by_form_here([&](auto row_form) {
      name_tokens<DT, decltype(row_form)::value>(row, out, e, scale * a_s / t.total, hard ? y : -1, scale * a_h, 0, V, slope,
                                                 TH == 64 ? threadIdx.x : threadIdx.x - 64, TH == 64 ? 64 : TH - 64);
    });
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
// f with the type and the form of the sums. At temperature 2 the second softmax is the first one's square (loss and
// gradient of 4096 x 32000 bf16 with labels by one call: 115 us, with two exponentials 125, as at T = 3 and 4).
template <class F>
void by_form(const Distill& a, int dtype, F f) {
  by_type(dtype, [&](auto dt) {
    if (!a.labels || a.T == 1.0f) f(dt, std::integral_constant<Form, kOne>{});
    else if (a.T == 2.0f) f(dt, std::integral_constant<Form, kSquare>{});
    else f(dt, std::integral_constant<Form, kTwo>{});
  });
}

int check(const Distill& a, int dtype, const char* name) {
  SLG_REQUIRE((a.logits && a.values && a.ids) || a.N == 0, SLG_E_ARG, "%s: null pointer", name);
  SLG_REQUIRE(dtype >= 0 && dtype <= 2 && a.vtype >= 0 && a.vtype <= 2, SLG_E_ARG, "%s: types %d and %d", name, dtype, a.vtype);
  SLG_REQUIRE((a.id_bytes == 4 || a.id_bytes == 8) && (!a.labels || a.label_bytes == 4 || a.label_bytes == 8), SLG_E_ARG,
              "%s: ids of %d bytes, labels of %d", name, a.id_bytes, a.label_bytes);
  SLG_REQUIRE(a.T >= 1e-4f && a.T <= 1e4f, SLG_E_ARG, "%s: temperature %g outside [1e-4, 1e4]", name, (double)a.T);
  SLG_REQUIRE(a.alpha >= 0.0f && a.alpha <= 1.0f, SLG_E_ARG, "%s: alpha %g outside [0, 1]", name, (double)a.alpha);
  SLG_REQUIRE(a.N >= 0 && a.N < (1LL << 31) && a.V >= 1 && a.V < (1LL << 31) - 65536 && a.ld >= 0 && a.K >= 1 && a.K <= kMaxEntries,
              SLG_E_SHAPE, "%s: N %lld, V %lld, K %d", name, (long long)a.N, (long long)a.V, a.K);
  return 0;
}

Distill args(const void* logits, int64_t N, int64_t V, int64_t ld, const void* values, int32_t vtype, const void* ids, int32_t id_bytes,
             int32_t K, const void* labels, int32_t label_bytes, float T, float alpha) {
  return {logits, N, V, ld, values, vtype, ids, id_bytes, K, labels, label_bytes, T, 1.0f / T, alpha};
}

// What `kept` holds: the rows' floats and the factor of an upstream gradient, which the gradient reads; behind them
// the rows' losses, counts and parts' sums.
struct Kept {
  float *rows, *loss, *factor;
  int* counts;
  Sums* parts;
  double2* sums;   // in the parts' place, of which there are none where rows are many
};
Kept layout(float* kept, int64_t N) {
  float *loss = kept + N * kKept + 4, *counts = loss + N, *parts = counts + kCounts;
  return {kept, loss, kept + N * kKept, reinterpret_cast<int*>(counts), reinterpret_cast<Sums*>(parts),
          reinterpret_cast<double2*>(kept + cdiv(parts - kept, 4) * 4)};
}

// The loss of all rows.
void sum_rows(const float* rows, const float* kept, const int* counts, int64_t N, bool mean, float* loss, const Kept& k, hipStream_t st) {
  double2* sums = N > kManyRows ? k.sums : nullptr;
  if (sums) hipLaunchKernelGGL(distill_sum_kernel, dim3(kCounts), dim3(256), 0, st, rows, mean ? kept : nullptr, N, sums);
  hipLaunchKernelGGL(distill_mean_kernel, dim3(1), dim3(1024), 0, st, rows, kept, sums, counts, N, mean, loss, k.factor);
}
// Parts of a row: one where there are rows for every compute unit, else as many as fill them, of 2048 values at least.
int64_t parts_of(int64_t N, int64_t V) { return N >= kParts / 2 ? 1 : std::max<int64_t>(1, std::min<int64_t>(kParts / N, V / 2048)); }

// Slots for the tokens that K entries name, and LDS of the entries with them (0: without).
int slots_of(const Distill& a) {
  int s = 2;
  while (s < 2 * a.K) s *= 2;
  return s;
}
int entry_bytes(const Distill& a, int slots) { return (slots ? 4 * a.K + 2 * slots : 3 * a.K) * 4; }
// A wave a row of few values: with 256 threads the loss of 65536 x 49 fp32 takes 109 us instead of 41, of 65536 x 2000
// 159 instead of 116, the gradient of 65536 x 49 98 instead of 35, of 65536 x 1000 146 instead of 141, but of 65536 x 2000
// 211 where one wave takes 235.
bool loss_by_wave(const Distill& a) { return a.V <= 2048; }
bool grad_by_wave(const Distill& a) { return a.V <= 1024; }

}  // namespace

extern "C" {

int64_t slg_distill_kept(int64_t N) {
  return N < 0 || N >= (1LL << 31) ? -1 : N * (kKept + 1) + 4 + kCounts + 3 * (N + kParts);
}

int slg_distill_fwd(const void* logits, int32_t dtype, int64_t N, int64_t V, int64_t ld, const void* values, int32_t vtype,
                    const void* ids, int32_t id_bytes, int32_t K, const void* labels, int32_t label_bytes, float T, float alpha,
                    int32_t reduction, float* loss, float* kept, slg_stream_t stream) {
  const Distill a = args(logits, N, V, ld, values, vtype, ids, id_bytes, K, labels, label_bytes, T, alpha);
  if (const int rc = check(a, dtype, "distill_fwd")) return rc;
  SLG_REQUIRE(reduction >= 0 && reduction <= 2, SLG_E_ARG, "distill_fwd: reduction %d", reduction);
  SLG_REQUIRE((loss && kept) || (N == 0 && !reduction), SLG_E_ARG, "distill_fwd: null pointer");
  SLG_REQUIRE((uintptr_t)kept % 16 == 0, SLG_E_ARG, "distill_fwd: kept not at a multiple of 16 bytes");
  if (N == 0 && !reduction) return 0;
  hipStream_t st = as_stream(stream);
  const Kept k = layout(kept, N);
  float* rows = reduction ? k.loss : loss;
  if (N) {
    const int64_t parts = parts_of(N, V), per = cdiv(cdiv(V, parts), 8) * 8;
    by_form(a, dtype, [&](auto dt, auto form) {
      constexpr int DT = decltype(dt)::value;
      constexpr Form FORM = decltype(form)::value;
      const int lds = entry_bytes(a, 0);
      if (parts == 1 && loss_by_wave(a))
        hipLaunchKernelGGL((distill_fwd_kernel<DT, 64, FORM>), grid_of(N), dim3(64), lds, st, a, 1, per, k.parts, rows, k.rows);
      else
        hipLaunchKernelGGL((distill_fwd_kernel<DT, 256, FORM>), grid_of(N * parts), dim3(256), lds, st, a, (int)parts, per, k.parts, rows,
                           k.rows);
      if (parts > 1)
        hipLaunchKernelGGL(distill_join_kernel<DT>, dim3((unsigned)N), dim3(64), lds, st, a, (int)parts, k.parts, rows, k.rows);
    });
  }
  if (reduction)
    sum_rows(rows, k.rows, nullptr, N, reduction == 2, loss, k, st);
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
  SLG_REQUIRE((uintptr_t)kept % 16 == 0, SLG_E_ARG, "distill_bwd: kept not at a multiple of 16 bytes");
  if (N == 0) return 0;
  // whole rows where there are enough of them, else chunks that make 2048 workgroups, of 2048 values at least
  const int64_t chunks = std::max<int64_t>(1, std::min<int64_t>(cdiv(2048, N), V / 2048)), chunk = cdiv(cdiv(V, chunks), 8) * 8;
  const int slots = slots_of(a);
  by_type(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const auto go = [&](auto kern, int th) {
      hipLaunchKernelGGL(kern, grid_of(N * chunks), dim3(th), entry_bytes(a, slots), as_stream(stream), a, slots, kept, upstream, reduction == 0,
                         reduction ? layout(const_cast<float*>(kept), N).factor : nullptr, scale, chunk, (int)chunks, grad);
    };
    if (grad_by_wave(a)) go(distill_bwd_kernel<DT, 64>, 64);
    else go(distill_bwd_kernel<DT, 256>, 256);
  });
  SLG_LAUNCH_CHECK("distill_bwd");
  return 0;
}

int slg_distill_loss_grad(const void* logits, int32_t dtype, int64_t N, int64_t V, int64_t ld, const void* values, int32_t vtype,
                          const void* ids, int32_t id_bytes, int32_t K, const void* labels, int32_t label_bytes, float T, float alpha,
                          int32_t reduction, float scale, float* loss, void* grad, float* kept, slg_stream_t stream) {
  SLG_REQUIRE(grad || N == 0, SLG_E_ARG, "distill_loss_grad: null pointer");
  SLG_REQUIRE(isfinite(scale), SLG_E_ARG, "distill_loss_grad: scale %g", (double)scale);
  if (N == 0 || parts_of(N, V) > 1) {   // too few rows for a workgroup each
    if (const int rc = slg_distill_fwd(logits, dtype, N, V, ld, values, vtype, ids, id_bytes, K, labels, label_bytes, T, alpha, reduction,
                                       loss, kept, stream))
      return rc;
    return slg_distill_bwd(logits, dtype, N, V, ld, values, vtype, ids, id_bytes, K, labels, label_bytes, T, alpha, reduction, kept,
                           nullptr, scale, grad, stream);
  }
  const Distill a = args(logits, N, V, ld, values, vtype, ids, id_bytes, K, labels, label_bytes, T, alpha);
  if (const int rc = check(a, dtype, "distill_loss_grad")) return rc;
  SLG_REQUIRE(reduction >= 0 && reduction <= 2, SLG_E_ARG, "distill_loss_grad: reduction %d", reduction);
  SLG_REQUIRE(loss && kept && (uintptr_t)kept % 16 == 0, SLG_E_ARG, "distill_loss_grad: loss or kept null or unaligned");
  hipStream_t st = as_stream(stream);
  const Kept k = layout(kept, N);
  float* rows = reduction ? k.loss : loss;
  int* counts = reduction == 2 ? k.counts : nullptr;
  const int slots = slots_of(a);
  if (counts) hipLaunchKernelGGL(distill_count_kernel, dim3(kCounts), dim3(256), 0, st, a, counts);
  by_form(a, dtype, [&](auto dt, auto form) {
    constexpr int DT = decltype(dt)::value, U = Group<DT>::U;
    constexpr Form FORM = decltype(form)::value;
    const auto go = [&](auto kern, int th) { hipLaunchKernelGGL(kern, grid_of(N), dim3(th), entry_bytes(a, slots), st, a, slots, counts, scale, rows, grad); };
    // the row in as few threads' registers as hold it; 512 threads read what is past 32768 values of 16 bits again (4096 x
    // 50257 bf16 with labels 231 us, x 65536 269; 1024 threads, which would hold it, 218 and 236: not built)
    if (V <= 64 * 4 * U) go(distill_both_kernel<DT, 64, 4, FORM>, 64);
    else if (V <= 256 * 4 * U) go(distill_both_kernel<DT, 256, 4, FORM>, 256);
    else if (DT != kTabF32 || V <= 512 * 8 * U) go(distill_both_kernel<DT, 512, 8, FORM>, 512);
    else if constexpr (DT == kTabF32) go(distill_both_kernel<DT, 1024, 8, FORM>, 1024);
  });
  if (reduction)
    sum_rows(rows, nullptr, counts, N, reduction == 2, loss, k, st);
  SLG_LAUNCH_CHECK("distill_loss_grad");
  return 0;
}

}  // extern "C"
