// The largest logits of a row and tokens drawn from it (gfx950). Both go by one order of the tokens: by value, equal
// values by the lower id. A token's place is a whole number `comp`, its value's bits in rising order above its id
// counted down, so that no two are equal and the order is that of the numbers. Logits that are NaN or -inf, or not
// allowed, are absent.
//
// Drawing (temperature T, limits k, p and m, a random number u in [0, 1)): masses w = exp((s - max) / T), of which
// the first k tokens stay, of these those before which lies less than p of their mass, of these those with w >= m;
// drawn is the first whose running sum passes u times theirs. Masses are held as whole numbers of 2^-F, F = 62 -
// log2 V and at most 52 (45 bits at 131072 tokens, where exp in 64 bits is off by 2^-52): their sums are exact, the
// same in any order, so LDS atomics may make them, and a border between two tokens is where 64-bit sums have it up
// to about V 2^-F.
//
// Finding a place in the order by its running count or mass goes by histogram: 2048 bins of equal width over the
// values (where a logit's mass goes by e^value, bins of equal keys would put most of a row into few bins), a scan,
// then the bin's own tokens, sorted if a thread can hold each, else by bins of their place numbers again until they
// are few.
#include <algorithm>

#include "block_ops.h"
#include "float_types.h"

namespace slg {

constexpr int kBins = 2048;
constexpr int kMaxTop = 1024;

// Rising with x, 0 for absent.
__device__ inline uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);   // -0 and 0 are equal
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ inline float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

template <int TH>
struct SelectLds {
  uint64_t hist[kBins];
  uint64_t list[TH];
  uint64_t part[TH / 64];
  uint64_t at, base;
  int n;
};

// A row of logits, its order, and the masses of its tokens.
template <int DT, int TH>
struct Row {
  using T = typename TabType<DT>::t;
  const T* logits;
  const uint8_t* allowed;   // null: all
  int V, bits;
  uint64_t id_mask;
  SelectLds<TH>* lds;
  // set by masses()
  float top, scale_bins;
  double inv_t, one;
  double least;   // masses under it count nothing
  uint64_t from;  // tokens before it in the numbers count nothing

  __device__ Row(const T* l, const uint8_t* m, int v, SelectLds<TH>* s) : logits(l), allowed(m), V(v), lds(s) {
    bits = 32 - __clz(v);
    id_mask = (1ull << bits) - 1;
    from = 1;
    least = 0.0;
  }
  __device__ uint64_t comp(float x, int i) const { return ((uint64_t)key_of(x) << bits) | (id_mask - (uint64_t)i); }
  __device__ int id_of(uint64_t c) const { return (int)(id_mask - (c & id_mask)); }
  __device__ float of(uint64_t c) const { return value_of((uint32_t)(c >> bits)); }

  // f(comp, x) of the tokens that are there.
  template <class F>
  __device__ void each(F f) const {
    for (int i = threadIdx.x; i < V; i += TH) {
      const float x = tab_get<DT>(logits[i]);
      if (x > -INFINITY && (!allowed || allowed[i])) f(comp(x, i), x);
    }
  }

  __device__ void masses(float max, float min, double t) {
    top = max;
    inv_t = 1.0 / t;
    const int f = min_(52, 62 - bits);
    one = (double)(1ull << f);
    // masses end where they fall under 2^-(F+1), values where the row does
    const float range = fmaxf(fminf((float)((f + 2) * 0.6931472 * t), max - min), 1e-30f);
    scale_bins = (float)kBins / range;
  }
  static __device__ int min_(int a, int b) { return a < b ? a : b; }
  __device__ uint64_t mass(float x) const {
    const double e = exp((x == top ? 0.0 : (double)x - (double)top) * inv_t);
    return e >= least ? (uint64_t)rint(e * one) : 0;   // a NaN (0 times an infinity) is none
  }
  __device__ int bin(float x) const { return (int)fminf((top - x) * scale_bins, (float)(kBins - 1)); }

  __device__ void clear() const {
    for (int i = threadIdx.x; i < kBins; i += TH) lds->hist[i] = 0;
    __syncthreads();
  }
  // The bin in which the running sum passes `target`, and the sum before it; the sum of all bins. None passes: -1.
  __device__ int find(uint64_t target, uint64_t& before, uint64_t& total) const {
    constexpr int B = kBins / TH;
    uint64_t sum = 0;
    for (int b = 0; b < B; ++b) sum += lds->hist[threadIdx.x * B + b];
    uint64_t run = block_scan<TH>(sum, lds->part, total);
    if (target >= total) return -1;
    if (target >= run && target - run < sum) {
      int b = 0;
      for (; b < B - 1; ++b) {
        const uint64_t h = lds->hist[threadIdx.x * B + b];
        if (target - run < h) break;
        run += h;
      }
      lds->at = (uint64_t)(threadIdx.x * B + b);
      lds->base = run;
    }
    __syncthreads();
    const int got = (int)lds->at;
    before = lds->base;
    __syncthreads();
    return got;
  }

  // Sums of weight(x) over the bins of the tokens' values.
  template <class W>
  __device__ void histogram(W weight) const {
    clear();
    each([&](uint64_t c, float x) {
      if (c < from) return;
      const uint64_t w = weight(x);
      if (w) atomicAdd((unsigned long long*)&lds->hist[bin(x)], (unsigned long long)w);
    });
    __syncthreads();
  }

  // The tokens for which in(c, x) holds, in falling order, one a thread (0: none), if there are at most TH; how many.
  template <class P>
  __device__ int collect(P in, uint64_t& mine) const {
    if (threadIdx.x == 0) lds->n = 0;
    lds->list[threadIdx.x] = 0;
    __syncthreads();
    each([&](uint64_t c, float x) {
      if (c >= from && in(c, x)) {
        const int at = atomicAdd(&lds->n, 1);
        if (at < TH) lds->list[at] = c;
      }
    });
    __syncthreads();
    const int n = lds->n;
    mine = lds->list[threadIdx.x];
    __syncthreads();
    if (n <= TH) {
      int size = 2;
      while (size < n) size *= 2;
      mine = block_sort<TH>(mine, size, lds->list);
    }
    return n;
  }

  // The place of the token whose running weight, on from `before` at the first token of bin b, passes `target`.
  // before: the sum before that token.
  template <class W>
  __device__ uint64_t within(int b, uint64_t target, uint64_t& before, W weight) const {
    uint64_t mine, total;
    int n = collect([&](uint64_t, float x) { return bin(x) == b; }, mine);
    if (n > TH) {
      uint64_t lo = ~0ull, hi = 0;
      each([&](uint64_t c, float x) {
        if (c >= from && bin(x) == b) {
          lo = c < lo ? c : lo;
          hi = c > hi ? c : hi;
        }
      });
      lo = block_reduce<TH>(lo, lds->part, [](uint64_t p, uint64_t q) { return p < q ? p : q; });
      hi = block_reduce<TH>(hi, lds->part, [](uint64_t p, uint64_t q) { return p > q ? p : q; });
      while (n > TH) {   // each round at least halves the numbers' range
        int shift = 0;
        while (((hi - lo) >> shift) >= (uint64_t)kBins) ++shift;
        clear();
        each([&](uint64_t c, float x) {
          if (c < lo || c > hi) return;
          const uint64_t w = weight(x);
          if (w) atomicAdd((unsigned long long*)&lds->hist[(hi - c) >> shift], (unsigned long long)w);
        });
        __syncthreads();
        uint64_t run;
        const uint64_t d = (uint64_t)find(target - before, run, total);
        before += run;
        hi -= d << shift;
        const uint64_t width = (1ull << shift) - 1;
        if (hi - lo > width) lo = hi - width;
        n = collect([&](uint64_t c, float) { return c >= lo && c <= hi; }, mine);
      }
    }
    const uint64_t w = mine ? weight(of(mine)) : 0;
    const uint64_t run = before + block_scan<TH>(w, lds->part, total);
    if (w && target >= run && target - run < w) {
      lds->at = mine;
      lds->base = run;
    }
    __syncthreads();
    const uint64_t c = lds->at;
    before = lds->base;
    __syncthreads();
    return c;
  }
};

// Largest and smallest place of the row's tokens; 0 where there is none.
template <int DT, int TH>
__device__ inline void extremes(const Row<DT, TH>& r, uint64_t& first, uint64_t& last) {
  uint64_t hi = 0, lo = ~0ull;
  r.each([&](uint64_t c, float) {
    hi = c > hi ? c : hi;
    lo = c < lo ? c : lo;
  });
  first = block_reduce<TH>(hi, r.lds->part, [](uint64_t p, uint64_t q) { return p > q ? p : q; });
  last = block_reduce<TH>(lo, r.lds->part, [](uint64_t p, uint64_t q) { return p < q ? p : q; });
}

template <int DT, int TH>
__global__ void __launch_bounds__(TH)
top_logits_kernel(const typename TabType<DT>::t* logits, int64_t ld, int V, int K, typename TabType<DT>::t* values, int64_t* ids) {
  __shared__ SelectLds<TH> lds;
  const int64_t n = blockIdx.x;
  Row<DT, TH> r(logits + n * ld, nullptr, V, &lds);
  uint64_t first, last, mine = 0;
  extremes(r, first, last);
  if (first) {
    const auto one = [](float) { return (uint64_t)1; };
    if (V > TH) {
      r.masses(r.of(first), r.of(last), INFINITY);
      r.histogram(one);
      uint64_t before, total;
      const int b = r.find(K - 1, before, total);
      if (b >= 0) r.from = r.within(b, K - 1, before, one);
    }
    r.collect([](uint64_t, float) { return true; }, mine);
  }
  if (threadIdx.x < K) {
    values[n * K + threadIdx.x] = tab_put<DT>(mine ? r.of(mine) : -INFINITY);
    ids[n * K + threadIdx.x] = mine ? r.id_of(mine) : -1;
  }
}

struct Limits {   // of all rows, or with a pointer of each; 64 bits, in which 0.8 of 40 equal masses are 32
  double t, p, m;
  int64_t k;
  const float *ts, *ps, *ms;
  const int64_t* ks;
};

template <int DT, int TH>
__global__ void __launch_bounds__(TH)
sample_kernel(const typename TabType<DT>::t* logits, int64_t ld, int V, const uint8_t* allowed, int64_t allowed_ld, const float* u,
              Limits lim, int64_t* ids) {
  __shared__ SelectLds<TH> lds;
  const int64_t n = blockIdx.x;
  Row<DT, TH> r(logits + n * ld, allowed ? allowed + n * allowed_ld : nullptr, V, &lds);
  uint64_t first, last;
  extremes(r, first, last);
  const double t = lim.ts ? lim.ts[n] : lim.t, p = lim.ps ? lim.ps[n] : lim.p, m = lim.ms ? lim.ms[n] : lim.m;
  const int64_t k = lim.ks ? lim.ks[n] : lim.k;
  if (!first || !(t > 0.0)) {
    if (threadIdx.x == 0) ids[n] = first ? r.id_of(first) : -1;
    return;
  }
  const bool by_p = p < 1.0;
  r.masses(r.of(first), r.of(last), t);
  const double least = m > 0.0 ? fmin(m, 1.0) : 0.0;
  const auto weight = [&](float x) { return r.mass(x); };
  const auto one = [](float) { return (uint64_t)1; };
  uint64_t before, total;
  uint64_t got = first;
  if (k > 0 && k < V) {
    r.histogram(one);
    const int b = r.find(k - 1, before, total);
    if (b >= 0) r.from = r.within(b, k - 1, before, one);
  }
  if (!by_p) r.least = least;
  r.histogram(weight);
  r.find(~0ull, before, total);
  if (by_p) {
    // the last token before which lies less than p of the mass: the one at which the running sum reaches it
    const double mass = p * (double)total;
    const uint64_t reach = mass > 0.0 ? (uint64_t)ceil(mass) - 1 : 0;   // the running sum passes this
    const int b = r.find(min(reach, total - 1), before, total);
    const uint64_t c = r.within(b, min(reach, total - 1), before, weight);
    total = before + r.mass(r.of(c));
    r.from = c;
    r.least = least;
    r.histogram(weight);
    r.find(~0ull, before, total);
  }
  const float v = u[n];
  const uint64_t target = min((uint64_t)(v > 0.0f ? fmin((double)v, 1.0) * (double)total : 0.0), total - 1);
  const int b = r.find(target, before, total);
  got = r.within(b, target, before, weight);
  if (threadIdx.x == 0) ids[n] = r.id_of(got);
}

}  // namespace slg

using namespace slg;

namespace {

// f with the type and the threads of a row: a token a thread where that can be, at most 1024
template <class F>
void dispatch(int dtype, int64_t V, int64_t k, F f) {
  const auto by_threads = [&](auto dt) {
    if (V <= 64) f(dt, std::integral_constant<int, 64>{});
    else if (V <= 4096 && k <= 256) f(dt, std::integral_constant<int, 256>{});
    else f(dt, std::integral_constant<int, 1024>{});
  };
  if (dtype == kTabF32) by_threads(std::integral_constant<int, kTabF32>{});
  else if (dtype == kTabBf16) by_threads(std::integral_constant<int, kTabBf16>{});
  else by_threads(std::integral_constant<int, kTabF16>{});
}

bool sizes(int64_t N, int64_t V, int64_t ld) { return N >= 0 && N < (1LL << 31) && V >= 1 && V <= (1LL << 24) && ld >= 0; }

}  // namespace

extern "C" {

int slg_top_logits(const void* logits, int32_t dtype, int64_t N, int64_t V, int64_t ld, int64_t K, void* values, int64_t* ids,
                   slg_stream_t stream) {
  SLG_REQUIRE((logits && values && ids) || N == 0, SLG_E_ARG, "top_logits: null pointer");
  SLG_REQUIRE(dtype >= 0 && dtype <= 2, SLG_E_ARG, "top_logits: type %d", dtype);
  SLG_REQUIRE(sizes(N, V, ld) && K >= 1 && K <= V && K <= kMaxTop, SLG_E_SHAPE, "top_logits: N %lld, V %lld, K %lld", (long long)N,
              (long long)V, (long long)K);
  if (N == 0) return 0;
  dispatch(dtype, V, K, [&](auto dt, auto th) {
    using T = typename TabType<decltype(dt)::value>::t;
    hipLaunchKernelGGL((top_logits_kernel<decltype(dt)::value, decltype(th)::value>), dim3((unsigned)N), dim3(decltype(th)::value), 0,
                       as_stream(stream), static_cast<const T*>(logits), ld, (int)V, (int)K, static_cast<T*>(values), ids);
  });
  SLG_LAUNCH_CHECK("top_logits");
  return 0;
}

int slg_sample_logits(const void* logits, int32_t dtype, int64_t N, int64_t V, int64_t ld, const uint8_t* allowed, int64_t allowed_ld,
                      const float* u, double temperature, int64_t top_k, double top_p, double min_p, const float* temperatures,
                      const int64_t* top_ks, const float* top_ps, const float* min_ps, int64_t* ids, slg_stream_t stream) {
  SLG_REQUIRE((logits && u && ids) || N == 0, SLG_E_ARG, "sample_logits: null pointer");
  SLG_REQUIRE(dtype >= 0 && dtype <= 2, SLG_E_ARG, "sample_logits: type %d", dtype);
  SLG_REQUIRE(sizes(N, V, ld) && allowed_ld >= 0, SLG_E_SHAPE, "sample_logits: N %lld, V %lld", (long long)N, (long long)V);
  SLG_REQUIRE(temperatures || temperature >= 0.0, SLG_E_ARG, "sample_logits: temperature %g", temperature);
  SLG_REQUIRE(top_ks || top_k >= 0, SLG_E_ARG, "sample_logits: top_k %lld", (long long)top_k);
  SLG_REQUIRE(top_ps || (top_p >= 0.0 && top_p <= 1.0), SLG_E_ARG, "sample_logits: top_p %g outside [0, 1]", top_p);
  SLG_REQUIRE(min_ps || (min_p >= 0.0 && min_p <= 1.0), SLG_E_ARG, "sample_logits: min_p %g outside [0, 1]", min_p);
  if (N == 0) return 0;
  const Limits lim{temperature, top_p, min_p, top_k, temperatures, top_ps, min_ps, top_ks};
  dispatch(dtype, V, 1, [&](auto dt, auto th) {
    using T = typename TabType<decltype(dt)::value>::t;
    hipLaunchKernelGGL((sample_kernel<decltype(dt)::value, decltype(th)::value>), dim3((unsigned)N), dim3(decltype(th)::value), 0,
                       as_stream(stream), static_cast<const T*>(logits), ld, (int)V, allowed, allowed_ld, u, lim, ids);
  });
  SLG_LAUNCH_CHECK("sample_logits");
  return 0;
}

}  // extern "C"
