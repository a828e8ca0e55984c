// The largest logits of a row and tokens drawn from it (gfx950). Both go by one order of the tokens: by value, equal
// values by the lower id. A token's place is a whole number `comp`, its value's bits in rising order above its id
// counted down, so that no two are equal and the order is that of the numbers. Logits that are NaN or -inf, or not
// allowed, are absent.
//
// Drawing (temperature T, limits k, p and m, a random number u in [0, 1)): masses w = exp((s - max) / T), of which
// the first k tokens stay, of these those before which lies less than p of their mass, of these those with w >= m;
// drawn is the first whose running sum passes u times theirs. Masses are held as whole numbers of 2^-F from an
// exponential that is off by 2^-43 of itself, F at most 50 and such that the sum of a row stays under 2^63: 62 - log2 V
// (47 at 32000 tokens), or from 2^18 tokens on 62 less the log of the row's own sum. Their sums are exact, the same in
// any order, so LDS atomics may make them. A mass is off by half a 2^-F, V of them by V 2^-(F+1): a border between two
// tokens is where sums without rounding have it up to 2^-33 of the sum at 32000 tokens and 2^-27 at most, an eighth of
// the steps that u has near 1. (By V alone the 2^24 tokens of a row would be off by 2^-14: a flat tail of masses under
// 2^-38 that hold 6e-5 together would come to 0.)
//
// A workgroup takes a row, in registers where it fits (the only read of it). What the limits keep is found by value
// first: k tokens are at least as large as a threshold that k lanes' own maxima reach, min_p is a threshold by
// itself. If a thread can hold each of the tokens past it, they are sorted and summed in order. Else places in the
// order are found by histogram: bins of equal width over the values (where a logit's mass goes by e^value, bins of
// equal keys would put most of a row into few bins), a scan, then the bin's own tokens, sorted if a thread can hold
// each, else by bins of their place numbers until they are few.
#include <float.h>

#include <algorithm>
#include <type_traits>

#include "block_ops.h"
#include "float_types.h"

#pragma clang fp contract(off)

namespace slg {

constexpr int kMaxTop = 1024;

// Rising with x.
__device__ inline uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);   // -0 and 0 are equal
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ inline float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// Bins of a histogram: enough that a long row's fullest bin seldom holds more tokens than threads, few enough to
// clear and scan.
template <int TH>
constexpr int kBins = TH <= 256 ? 4 * TH : 2048;

template <int TH>
struct SelectLds {
  uint64_t hist[kBins<TH> + 64];   // the last ones take what counts nothing
  uint64_t list[TH];
  uint64_t part[TH / 64];
  uint64_t at, base;
  int n;
};

// 2^f on [-1/2, 1/2] by the polynomial of degree 9 with value 1 at 0 and the least largest relative error, 2^-43
// (fitted by exchange of its extremes). In memory, so that they come to scalar registers: a literal of 64 bits would
// be moved to vector ones before each product.
__constant__ double kExp2[9] = {0x1.62e42fefa08dcp-1,  0x1.ebfbdff823df0p-3,  0x1.c6b08d7a95072p-5,
                                0x1.3b2ab717fb0b6p-7,  0x1.5d87ebe42d79dp-10, 0x1.4308acc67a164p-13,
                                0x1.fffd75179b1a0p-17, 0x1.63d0ec28f10f2p-20, 0x1.89c489e9e3ae4p-24};
__device__ __forceinline__ double exp2_small(double f, double lead) {
  double p = fma(lead, f, kExp2[7]);
#pragma unroll
  for (int i = 6; i >= 0; --i) p = fma(p, f, kExp2[i]);
  return fma(p, f, 1.0);
}

// A row of logits over the threads of a workgroup, group j of thread t the row's (j TH + t)th of 16 bytes: the first NV
// in registers, others read again by each pass (NV = 0: rows shorter than a group too).
template <int DT, int TH, int NV>
struct Row {
  using T = typename TabType<DT>::t;
  static constexpr int VU = 16 / (int)sizeof(T);
  static constexpr int BINS = kBins<TH>;
  static constexpr int SUB = VU == 4 ? 4 : 2;
  static constexpr int AT_A_TIME = 2;   // tokens whose masses are computed side by side
  static constexpr bool MORE = NV == 0 || NV == 8;   // rows may be longer than the registers hold
  using E = std::conditional_t<DT == kTabBf16, __bf16, T>;
  typedef E Vec __attribute__((ext_vector_type(VU), aligned(sizeof(T))));
  typedef uint8_t Bytes __attribute__((ext_vector_type(VU), aligned(1)));
  const T* logits;
  const uint8_t* allowed;   // null: all
  int V, bits;
  uint64_t id_mask;
  SelectLds<TH>* lds;
  mutable Vec r[NV ? NV : 1];
  bool infinite;
  float top, cut, bin_scale, bin_base;   // under `cut` masses are 0
  double lead;   // kExp2's last, in vector registers: an instruction reads one scalar operand
  double top64, slope, shifter, lowest, least;   // slope: log2 e / T; masses under `least` count nothing
  int F;
  uint64_t from;   // tokens whose place number is under it count nothing

  __device__ __forceinline__ Row(const T* l, const uint8_t* m, int v, SelectLds<TH>* s) : logits(l), allowed(m), V(v), lds(s) {
    bits = 32 - __clz(v);
    id_mask = (1ull << bits) - 1;
    infinite = false;
    from = 0;
    least = 0.0;
    lead = kExp2[8];
    asm volatile("" : "+v"(lead));
    if constexpr (NV > 0) {
      const int own = (int)threadIdx.x * VU;
#pragma unroll
      for (int j = 0; j < NV; ++j) r[j] = read(j * TH * VU + own);
      if (allowed) {
        Bytes b[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) b[j] = bytes(j * TH * VU + own);
#pragma unroll
        for (int j = 0; j < NV; ++j) forbid(r[j], b[j]);
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if ((j + 1) * TH * VU > V) bound(r[j], j * TH * VU + own);
    }
  }

  static __device__ __forceinline__ E absent() { return (E)NAN; }
  // The first token of the group that begins at token i: a row's last group is moved back to end with the row, and
  // those past it come to lie there too. Tokens before i in it are another group's.
  __device__ __forceinline__ int base(int i) const { return NV == 0 && V < VU ? i : min(i, V - VU); }
  __device__ __forceinline__ Vec read(int i) const {
    if (NV > 0 || V >= VU) return *reinterpret_cast<const Vec*>(reinterpret_cast<const char*>(logits) + (uint32_t)base(i) * (uint32_t)sizeof(T));
    Vec x;
#pragma unroll
    for (int u = 0; u < VU; ++u) x[u] = reinterpret_cast<const E*>(logits)[min(i + u, V - 1)];
    return x;
  }
  __device__ __forceinline__ Bytes bytes(int i) const {
    if (NV > 0 || V >= VU) return *reinterpret_cast<const Bytes*>(allowed + (uint32_t)base(i));
    Bytes x;
#pragma unroll
    for (int u = 0; u < VU; ++u) x[u] = allowed[min(i + u, V - 1)];
    return x;
  }
  // NaN for tokens that are not allowed; that are another group's, or past the row.
  static __device__ __forceinline__ void forbid(Vec& x, Bytes b) {
#pragma unroll
    for (int u = 0; u < VU; ++u) x[u] = b[u] ? x[u] : absent();
  }
  __device__ __forceinline__ void bound(Vec& x, int i) const {
    const int b = base(i);
#pragma unroll
    for (int u = 0; u < VU; ++u) x[u] = b + u >= i && b + u < V ? x[u] : absent();
  }
  // f(values, first token) of all groups, absent tokens (-inf, NaN) among them, and NaN past the row.
  template <class F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      // a group at a time, and nothing of it kept from an earlier pass: what is computed of all values at once, or
      // kept, does not fit the registers beside them
      int t = threadIdx.x;
      asm volatile("" : "+v"(r[j]), "+v"(t));
      give(f, r[j], base((j * TH + t) * VU));
    }
    if constexpr (MORE) each_again<NV, NV == 0 ? 1 : VU == 4 ? 4 : 2>(f);
  }
  // The same from memory, from group FIRST TH on: for what the registers do not hold, and passes that few rows need.
  // AT_ONCE groups of a thread in flight; those past the row are the last one, struck out.
  template <int FIRST, int AT_ONCE = 1, class F>
  __device__ __forceinline__ void each_again(F f) const {
#pragma unroll 1
    for (int g = FIRST * TH * VU; g < V; g += AT_ONCE * TH * VU) {
      int own = g + (int)threadIdx.x * VU;
      Vec x[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) x[k] = read(own + k * TH * VU);
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int i = own + k * TH * VU;
        if (infinite) only_infinite(x[k]);
        if (allowed) forbid(x[k], bytes(i));
        if (g + (k + 1) * TH * VU > V) bound(x[k], i);
        give(f, x[k], base(i));
      }
    }
  }
  template <class F>
  static __device__ __forceinline__ void give(F f, const Vec& x, int i) {
    float v[VU];
#pragma unroll
    for (int u = 0; u < VU; ++u) v[u] = (float)x[u];
    f(v, i);
    __builtin_amdgcn_sched_barrier(0);
  }
  // f(x, token) of the tokens for which in(x) holds; a branch for SUB of them, and for each where one does.
  template <bool AGAIN, class P, class F>
  __device__ __forceinline__ void each_in(P in, F f) const {
    const auto some = [&](const float (&x)[VU], int i) {
#pragma unroll
      for (int s = 0; s < VU; s += SUB) {
        bool any = false;
#pragma unroll
        for (int u = s; u < s + SUB; ++u) any |= in(x[u]);
        if (__ballot(any) != 0) {
#pragma unroll
          for (int u = s; u < s + SUB; ++u)
            if (in(x[u])) f(x[u], i + u);
        }
        if (SUB < VU) __builtin_amdgcn_sched_barrier(0);
      }
    };
    if constexpr (AGAIN) each_again<0>(some);
    else each(some);
  }
  // The largest is +inf: those that are count as 0, the others are absent.
  static __device__ __forceinline__ void only_infinite(Vec& x) {
#pragma unroll
    for (int u = 0; u < VU; ++u) x[u] = (float)x[u] == INFINITY ? (E)0.0f : absent();
  }
  __device__ __forceinline__ void set_infinite() {
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) only_infinite(r[j]);
    }
    infinite = true;
  }
  __device__ __forceinline__ uint64_t comp(float x, int i) const { return ((uint64_t)key_of(x) << bits) | (id_mask - (uint64_t)i); }
  __device__ __forceinline__ int id_of(uint64_t c) const { return (int)(id_mask - (c & id_mask)); }
  __device__ __forceinline__ float of(uint64_t c) const { return value_of((uint32_t)(c >> bits)); }

  __device__ __forceinline__ void masses(float max, float min, double t) {
    top = max;
    top64 = uniform((double)max);
    slope = uniform(fmax(fmin(1.4426950408889634 / t, 1e300), 1e-300));
    F = bits > 12 ? 62 - bits : 50;
    if constexpr (NV == 8 && TH >= 512) {
      if (bits > 18) F = bits_of_mass();
    }
    shifter = uniform(0x1.8p52 + (double)F);
    lowest = uniform(-100.0 / slope);   // far enough down for a mass of 0
    // bins end where masses fall under 2^-(F+2), or where the row does
    const float reach = (float)((F + 2) * 0.6931472 * t), range = fmaxf(fminf(reach, max - min), 1e-30f);
    cut = uniform(fmaxf(min, max - reach));
    // where the sums of bin_at round by more than a bin's part (large logits, close together) all is one bin
    const float scale = ((float)BINS - 1.0f) / range;
    bin_scale = uniform(fabsf(max) * scale < 4194304.0f ? scale : 0.0f);
    bin_base = uniform(max * bin_scale);
  }
  // F of a long row: by its sum in 32 bits, which chains of at most 2^16 additions leave within 2^-8 of itself.
  __device__ __forceinline__ int bits_of_mass() const {
    float sum = 0.0f;
    each([&](const float (&x)[VU], int) {
#pragma unroll
      for (int u = 0; u < VU; ++u) {
        const float z = (float)(fmax((double)x[u] - top64, -100.0 / slope) * slope);
        sum += x[u] > -INFINITY ? __builtin_amdgcn_exp2f(z) : 0.0f;
      }
    });
    sum = block_reduce<TH>(sum, reinterpret_cast<float*>(lds->part), [](float p, float q) { return p + q; });
    return min(50, 62 - __builtin_amdgcn_frexp_expf(sum));   // the sum is 1 at least
  }
  // 2^F exp(d / T) to a whole number. The products are of single roundings in every place that this comes to: sums over
  // the same tokens have to be the same.
  __device__ __forceinline__ uint64_t mass_at(double d) const {
    // where 1.5 2^52 is added the sum's low bits are the nearest whole number, here of log2 plus F
    const double z = fma(d, slope, shifter), p = exp2_small(fma(d, slope, shifter - z), lead);
    const double e = __hiloint2double(__double2hiint(p) + (__double2loint(z) << 20), __double2loint(p));
    // at most 2^50: rounded to a whole number where 2^52 is added, whose bits it then leaves
    const double w = e + 0x1p52;
    return ((uint64_t)(__double2hiint(w) & 0xfffff) << 32) | (uint32_t)__double2loint(w);
  }
  // The mass of a token, 0 if it is under `least`.
  __device__ __forceinline__ uint64_t mass(float x) const {
    const uint64_t w = mass_at(fmax((double)x - top64, lowest));
    return (double)w >= least ? w : 0;
  }
  // Falling with x.
  __device__ __forceinline__ float bin_at(float x) const { return fmaf(x, -bin_scale, bin_base); }
  __device__ __forceinline__ int bin(float x) const { return min((int)bin_at(x), BINS - 1); }

  // What the threads know of a histogram: the sum before a thread's own bins, of its own, of all.
  struct Prefix {
    uint64_t run, sum, total;
  };
  __device__ __forceinline__ Prefix prefix() const {
    constexpr int B = BINS / TH;
    Prefix p;
    p.sum = 0;
#pragma unroll
    for (int b = 0; b < B; ++b) p.sum += lds->hist[threadIdx.x * B + b];
    p.run = block_scan<TH>(p.sum, lds->part, p.total);
    return p;
  }
  // The bin in which the running sum passes `target` (less than the total), and the sum before it.
  __device__ __forceinline__ int find(const Prefix& p, uint64_t target, uint64_t& before) const {
    constexpr int B = BINS / TH;
    if (target >= p.run && target - p.run < p.sum) {
      uint64_t run = p.run;
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
    const int got = (int)uniform(lds->at);
    before = uniform(lds->base);
    __syncthreads();
    return got;
  }
  __device__ __forceinline__ void clear() const {
    for (int i = threadIdx.x; i < BINS; i += TH) lds->hist[i] = 0;
    __syncthreads();
  }
  // Masses over the bins of the tokens' values; AGAIN: from memory, of the tokens from `from` on, and not under `least`.
  template <bool AGAIN>
  __device__ __forceinline__ Prefix histogram() const {
    clear();
    if constexpr (AGAIN) {
      each_in<true>([&](float x) { return x >= cut; }, [&](float x, int i) {
        if (comp(x, i) >= from) atomicAdd((unsigned long long*)&lds->hist[bin(x)], (unsigned long long)mass(x));
      });
    } else {
      // no branch for a token: those under the cut, or absent, add 0, past the bins to a place of their own lane's
      const uint32_t last = BINS + (threadIdx.x & 63);
      each([&](const float (&x)[VU], int) {
#pragma unroll
        for (int u = 0; u < VU; ++u) {
          const float v = x[u] >= cut ? x[u] : -INFINITY;
          const uint64_t w = mass_at(fmax((double)v - top64, lowest));
          uint32_t b;
          asm("v_cvt_u32_f32 %0, %1" : "=v"(b) : "v"(bin_at(v)));   // 0 for a NaN and under 0, the largest past it
          atomicAdd((unsigned long long*)&lds->hist[min(b, last)], (unsigned long long)w);
          if (u % AT_A_TIME == AT_A_TIME - 1) __builtin_amdgcn_sched_barrier(0);
        }
      });
    }
    __syncthreads();
    return prefix();
  }

  // The tokens for which in(x) holds, in falling order, one a thread (0: none), if there are at most TH; how many. AGAIN:
  // from memory, of those with place numbers in [lo, hi].
  template <bool AGAIN, class P>
  __device__ __forceinline__ int collect(P in, uint64_t& mine, uint64_t lo = 0, uint64_t hi = ~0ull) const {
    if (threadIdx.x == 0) lds->n = 0;
    lds->list[threadIdx.x] = 0;
    __syncthreads();
    each_in<AGAIN>(in, [&](float x, int i) {
      const uint64_t c = comp(x, i);
      if (!AGAIN || (c >= lo && c <= hi)) {
        const int at = atomicAdd(&lds->n, 1);
        if (at < TH) lds->list[at] = c;
      }
    });
    __syncthreads();
    const int n = uniform(lds->n);
    mine = lds->list[threadIdx.x];
    __syncthreads();
    if (n <= TH) mine = block_sort<TH>(mine, n, lds->list);
    return n;
  }

  // Of the tokens with place numbers in [lo, hi], the one whose running weight, on from `before` at the first of them,
  // passes `target`, and the sum before it. By bins of the place numbers until a thread can hold each token of one.
  template <class W>
  __device__ __forceinline__ uint64_t descend(uint64_t lo, uint64_t hi, uint64_t target, uint64_t& before, W weight) const {
    const auto there = [](float x) { return x > -INFINITY; };
    uint64_t mine;
    int n = TH + 1;
    for (int round = 0; round < 16 && n > TH; ++round) {   // each cuts the numbers' range to a 128th at most, or to one number
      int shift = 0;
      while (((hi - lo) >> shift) >= (uint64_t)BINS) ++shift;
      clear();
      each_in<true>(there, [&](float x, int i) {
        const uint64_t c = comp(x, i);
        if (c < lo || c > hi) return;
        const uint64_t w = weight(x);
        if (w) atomicAdd((unsigned long long*)&lds->hist[(hi - c) >> shift], (unsigned long long)w);
      });
      __syncthreads();
      uint64_t run;
      const uint64_t d = (uint64_t)find(prefix(), target - before, run);
      before += run;
      hi -= d << shift;
      const uint64_t width = (1ull << shift) - 1;
      if (hi - lo > width) lo = hi - width;
      n = collect<true>(there, mine, lo, hi);
    }
    return among(mine, target, before, weight);
  }
  // The same of tokens in order, one a thread.
  template <class W>
  __device__ __forceinline__ uint64_t among(uint64_t mine, uint64_t target, uint64_t& before, W weight) const {
    const uint64_t w = mine ? weight(of(mine)) : 0;
    uint64_t total;
    const uint64_t run = before + block_scan<TH>(w, lds->part, total);
    if (w && target >= run && target - run < w) {
      lds->at = mine;
      lds->base = run;
    }
    __syncthreads();
    const uint64_t c = uniform(lds->at);
    before = uniform(lds->base);
    __syncthreads();
    return c;
  }
  // c: the token of bin b at which the running mass, on from `before` at the bin's first, passes `target`. False if
  // the bin holds more tokens than there are threads: then nothing is found, or with AGAIN it is, and the bins of the
  // values are overwritten.
  template <bool AGAIN>
  __device__ __forceinline__ bool within(int b, uint64_t target, uint64_t& before, uint64_t& c) const {
    const float lo = b ? (float)b : -INFINITY, hi = b < BINS - 1 ? (float)(b + 1) : bin_at(cut) + 1.0f;
    const auto in = [&](float x) {
      const float at = bin_at(x);
      return at >= lo && at < hi;
    };
    const auto weight = [&](float x) { return mass(x); };
    uint64_t mine;
    if (collect<AGAIN>(in, mine, from) <= TH) {
      c = among(mine, target, before, weight);
      return true;
    }
    if constexpr (AGAIN) {
      uint64_t first = ~0ull, last = 0;
      each_in<true>(in, [&](float x, int i) {
        const uint64_t at = comp(x, i);
        if (at < from) return;
        first = at < first ? at : first;
        last = at > last ? at : last;
      });
      first = block_reduce<TH>(first, lds->part, [](uint64_t p, uint64_t q) { return p < q ? p : q; });
      last = block_reduce<TH>(last, lds->part, [](uint64_t p, uint64_t q) { return p > q ? p : q; });
      c = descend(first, last, target, before, weight);
    }
    return false;
  }
  // The kth token in order, one at least as large as `least_value`; there are more than k such.
  __device__ __forceinline__ uint64_t kth(int64_t k, float least_value) const {
    uint64_t before = 0;
    return descend((uint64_t)key_of(least_value) << bits, ~0ull >> (32 - bits), (uint64_t)(k - 1), before,
                   [](float) { return (uint64_t)1; });
  }
  // A value that at least k tokens (at most TH) reach, if there are as many: in each wave as many lanes as make k of
  // all waves have a token of that size, own: each lane's largest.
  __device__ __forceinline__ float reached(float own, int k) const {
    constexpr int W = TH / 64;
    const int place = (k + W - 1) / W - 1;
    own = read_lane(wave_sort(own, true), place);
    return block_reduce<TH>(own, reinterpret_cast<float*>(lds->part), [](float p, float q) { return fminf(p, q); });
  }
  // Largest and smallest of the tokens that are there, and a thread's own largest.
  __device__ __forceinline__ void extremes(float& max, float& min, float& own) const {
    own = -INFINITY;
    min = INFINITY;
    each([&](const float (&x)[VU], int) {   // both pass over a NaN
#pragma unroll
      for (int u = 0; u < VU; ++u) {
        own = fmaxf(own, x[u]);
        min = fminf(min, x[u]);
      }
    });
    const auto smaller = [](float p, float q) { return fminf(p, q); };
    max = block_reduce<TH>(own, reinterpret_cast<float*>(lds->part), [](float p, float q) { return fmaxf(p, q); });
    min = block_reduce<TH>(min, reinterpret_cast<float*>(lds->part), smaller);
    if (min == -INFINITY) {
      min = INFINITY;
      each_in<true>([](float x) { return x > -INFINITY; }, [&](float x, int) { min = fminf(min, x); });
      min = block_reduce<TH>(min, reinterpret_cast<float*>(lds->part), smaller);
    }
  }
};

// The K largest of a row, a workgroup each. 64 of 4096 x 32000 bf16: 52 to 55 us, 4.8 to 5.0 TB/s, where 512 threads
// hold the row in 64 registers each and two passes look at it (lanes' maxima, then what is past the threshold, some
// 190 tokens): memory, with the vector instructions at 80% of their issue; in fp32 96 us, 5.5 TB/s. 100 of 33 x
// 131071 fp32: 18 to 20 us, on 33 compute units.
template <int DT, int TH, int NV>
__global__ void __launch_bounds__(TH)
top_logits_kernel(const typename TabType<DT>::t* logits, int64_t N, int64_t ld, int V, int K, typename TabType<DT>::t* values,
                  int64_t* ids) {
  __shared__ SelectLds<TH> lds;
  const int64_t n = block_id();
  if (n >= N) return;
  Row<DT, TH, NV> r(logits + n * ld, nullptr, V, &lds);
  float least = -FLT_MAX;
  if (V > TH) {
    float own = -FLT_MAX;
    r.each([&](const auto& x, int) {
#pragma unroll
      for (int u = 0; u < Row<DT, TH, NV>::VU; ++u) own = fmaxf(own, x[u]);
    });
    least = r.reached(own, K);
  }
  uint64_t mine;
  const auto listed = [&](float x) { return x >= least; };
  if (r.template collect<false>(listed, mine) > TH) r.template collect<true>(listed, mine, r.kth(K, least));
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

// The running sum that is passed by the last token before which lies less than p of `total`.
__device__ inline uint64_t reach_of(double p, uint64_t total) {
  const double mass = p * (double)total;
  const uint64_t reach = mass > 0.0 ? (uint64_t)ceil(mass) - 1 : 0;
  return reach < total ? reach : total - 1;
}
__device__ inline uint64_t target_of(float u, uint64_t total) {
  const uint64_t t = u > 0.0f ? (uint64_t)(fmin((double)u, 1.0) * (double)total) : 0;
  return t < total ? t : total - 1;
}

// A token of a row, a workgroup each. 4096 x 32000 fp32, in a captured graph over three sets of inputs: 113 us by
// min_p, 125 by the first 40, 203 without a limit and 219 by top_p, where each token's mass (24 vector instructions,
// most in 64 bits) and its place in a histogram (an LDS atomic of 64 bits, 15 cycles a wave) are what bounds it:
// vector instructions 73% of their issue. Half of such a row fits the registers at two workgroups a compute unit; a
// form of 1024 threads or 16 groups a thread, which hold all of it with one, was slower, as was one of 256 threads
// for short lists (64 rows of 32000: 28 us instead of 21). Masses of 32 bits for the histogram, with exact ones where
// a border is near, came to 185 us without a limit (exact ones alone then to 202) but 252 by top_p (234).
template <int DT, int TH, int NV>
__global__ void __launch_bounds__(TH, 4)
sample_kernel(const typename TabType<DT>::t* logits, int64_t N, int64_t ld, int V, const uint8_t* allowed, int64_t allowed_ld,
              const float* us, Limits lim, int64_t* ids) {
  __shared__ SelectLds<TH> lds;
  const int64_t n = block_id();
  if (n >= N) return;
  Row<DT, TH, NV> r(logits + n * ld, allowed ? allowed + n * allowed_ld : nullptr, V, &lds);
  const double t = lim.ts ? lim.ts[n] : lim.t, p = lim.ps ? lim.ps[n] : lim.p, m = lim.ms ? lim.ms[n] : lim.m;
  const int64_t k = lim.ks ? lim.ks[n] : lim.k;
  const float u = us[n];
  float max, min, own;
  r.extremes(max, min, own);
  if (max == -INFINITY || !(t > 0.0)) {
    int first = V;
    r.template each_in<true>([&](float x) { return x == max && max > -INFINITY; }, [&](float, int i) { first = i < first ? i : first; });
    first = block_reduce<TH>(first, reinterpret_cast<int*>(lds.part), [](int a, int b) { return a < b ? a : b; });
    if (threadIdx.x == 0) ids[n] = first < V ? first : -1;
    return;
  }
  if (max == INFINITY) {
    r.set_infinite();
    max = min = 0.0f;
    own = own == INFINITY ? 0.0f : -INFINITY;
  }
  r.masses(max, min, t);
  const bool by_p = p < 1.0, by_m = m > 0.0, by_k = k > 0 && k < V;
  const double least = by_m ? fmin(m, 1.0) : 0.0;
  float lower = -FLT_MAX;
  if (by_k && k <= TH && V > TH) lower = fmaxf(lower, r.reached(own, (int)k));
  if (by_m && !by_p) {
    // under the border by more than its rounding and the bound's own
    const double b = (double)max + t * log(least);
    lower = fmaxf(lower, (float)(b - 1e-6 * (fabs(b) + t) - 1e-37));
  }
  uint64_t mine = 0, total;
  int many = TH + 1;
  if (V <= TH || (by_k && k <= TH) || (by_m && !by_p))
    many = r.template collect<false>([&](float x) { return x >= lower; }, mine);
  if (many <= TH) {   // a token a thread, in order
    if (by_k && threadIdx.x >= k) mine = 0;
    uint64_t w = mine ? r.mass(r.of(mine)) : 0;
    const uint64_t run = block_scan<TH>(w, lds.part, total);
    if (by_p || by_m) {
      if (by_p && run > reach_of(p, total)) w = 0;
      r.least = ldexp(least, r.F);
      if (by_m && mine && w) w = r.mass(r.of(mine));
      total = block_reduce<TH>(w ? run + w : 0, lds.part, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
    }
    const uint64_t target = target_of(u, total);
    if (w && target >= run && target - run < w) ids[n] = r.id_of(mine);
    return;
  }
  if (by_k) {
    // without a threshold the kth may not be there
    int there = 0;
    r.template each_in<true>([](float x) { return x > -INFINITY; }, [&](float, int) { ++there; });
    there = block_reduce<TH>(there, reinterpret_cast<int*>(lds.part), [](int a, int b) { return a + b; });
    if (there > k) r.from = r.kth(k, k <= TH && V > TH ? lower : min);
  }
  uint64_t before = 0, c = 0;
  if (!r.from && (by_p || !by_m)) {
    const auto hist = r.template histogram<false>();
    total = hist.total;
    bool found = true;
#pragma unroll 1
    for (int step = by_p ? 0 : 1; step < 2 && found; ++step) {   // the last token that top_p keeps, the token drawn
      const uint64_t target = step ? target_of(u, total) : reach_of(p, total);
      const int b = r.find(hist, target, before);
      found = r.template within<false>(b, target, before, c);
      if (step == 0 && found) {
        const uint64_t w = r.mass(r.of(c));
        total = before + w;
        found = !by_m || (double)w >= ldexp(least, r.F) + 1.0;   // min_p keeps them all
      }
    }
    if (found) {
      if (threadIdx.x == 0) ids[n] = r.id_of(c);
      return;
    }
  }
  if (!by_p) r.least = ldexp(least, r.F);
  auto hist = r.template histogram<true>();
  total = hist.total;
#pragma unroll 1
  for (int step = by_p ? 0 : 1; step < 2; ++step) {
    const uint64_t target = step ? target_of(u, total) : reach_of(p, total);
    const int b = r.find(hist, target, before);
    r.template within<true>(b, target, before, c);
    if (step == 0) {
      r.from = c;
      r.least = ldexp(least, r.F);
      hist = r.template histogram<true>();
      total = hist.total;
    }
  }
  if (threadIdx.x == 0) ids[n] = r.id_of(c);
}

}  // namespace slg

using namespace slg;

namespace {

// f with the type, the threads and the groups of 16 bytes a thread of N rows of V logits. Listing up to k tokens takes
// as many threads. (Draws pass k = 1 whatever their limit, which may be each row's own: where fewer lanes hold tokens
// than their top_k asks for, there is no threshold, and the list overflows into the histograms. 4096 x 257 by the first
// 50 take 17 us in fp32 and 24 in bf16, by top_p 12 and 14.)
template <bool LIST, class F>
void dispatch(int dtype, int64_t N, int64_t V, int64_t k, F f) {
  using std::integral_constant;
  const auto by_size = [&](auto dt) {
    constexpr int VU = 16 / (int)sizeof(typename TabType<decltype(dt)::value>::t);
    const auto go = [&](auto th, auto nv) { f(dt, th, nv); };
    const int64_t groups = cdiv(V, VU);
    // a row that fills no group is read token by token
    if (V < VU) return go(integral_constant<int, 64>{}, integral_constant<int, 0>{});
    // as few threads as hold the row: more rows are under way side by side, and their barriers are of fewer waves (8192
    // rows of 2000 fp32 by top_p take 42 us with 128 threads, 214 with 512 of eight groups; of 8000 113 with 256, 223 with
    // 512); but about three times k tokens reach a list's threshold where the row fills the lanes, and 40 of 64 rows of 500
    // take 5 us with 128 threads, 11 with 64
    if (groups <= 128 && k <= 24) return go(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    if (groups <= 256 && k <= 48) return go(integral_constant<int, 128>{}, integral_constant<int, 2>{});
    if (groups <= 512 && k <= 48) return go(integral_constant<int, 128>{}, integral_constant<int, 4>{});
    if (groups <= 1024 && k <= 48) return go(integral_constant<int, 128>{}, integral_constant<int, 8>{});
    if (groups <= 2048 && k <= 96) return go(integral_constant<int, 256>{}, integral_constant<int, 8>{});
    if constexpr (LIST) {
      if (groups <= 4096 && k <= 160) return go(integral_constant<int, 512>{}, integral_constant<int, 8>{});
      if (groups <= 4096) return go(integral_constant<int, 1024>{}, integral_constant<int, 4>{});
      go(integral_constant<int, 1024>{}, integral_constant<int, 8>{});
    } else {
      // a compute unit holds one workgroup of 1024 threads, or two of 512: fp32 by top_p, 64 rows of 130000 take 53 us with
      // the former and 65 with the latter, 300 of 50257 62 and 53, 4096 of 32000 307 and 219
      if (groups > 4096 && N <= 256) return go(integral_constant<int, 1024>{}, integral_constant<int, 8>{});
      go(integral_constant<int, 512>{}, integral_constant<int, 8>{});
    }
  };
  if (dtype == kTabF32) by_size(integral_constant<int, kTabF32>{});
  else if (dtype == kTabBf16) by_size(integral_constant<int, kTabBf16>{});
  else by_size(integral_constant<int, kTabF16>{});
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
  dispatch<true>(dtype, N, V, K, [&](auto dt, auto th, auto nv) {
    using T = typename TabType<decltype(dt)::value>::t;
    hipLaunchKernelGGL((top_logits_kernel<decltype(dt)::value, decltype(th)::value, decltype(nv)::value>), grid_of(N), dim3(decltype(th)::value), 0,
                       as_stream(stream), static_cast<const T*>(logits), N, ld, (int)V, (int)K, static_cast<T*>(values), ids);
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
  dispatch<false>(dtype, N, V, 1, [&](auto dt, auto th, auto nv) {
    using T = typename TabType<decltype(dt)::value>::t;
    hipLaunchKernelGGL((sample_kernel<decltype(dt)::value, decltype(th)::value, decltype(nv)::value>), grid_of(N), dim3(decltype(th)::value), 0,
                       as_stream(stream), static_cast<const T*>(logits), N, ld, (int)V, allowed, allowed_ld, u, lim, ids);
  });
  SLG_LAUNCH_CHECK("sample_logits");
  return 0;
}

}  // extern "C"
