// Bucket table of references (see ref_table.h): the references sorted by key
// (radix_sort.h: stable, so a bucket's references ascend), then each key's
// first place by a search (ref_start). The time does not depend on how the
// references fall on the keys: 160000 references over 20000 keys take 37 us in
// five launches. Buckets filled through counters and then ranked, the larger
// ones sorted by one lane, took 41 us in six, but 4.9 ms at 3718 references over
// 2 keys.
#include "ref_table.h"

#include "radix_sort.h"

namespace slg {

struct RefKeys {
  const int* keys;
  __device__ int key(int64_t i) const { return keys[i]; }
};

// start[k] = entries of keys below k (threads 0..nkeys), sorted[j] = entry j's
// reference (the threads after them).
__global__ void __launch_bounds__(256) ref_start_kernel(const int2* __restrict__ ent, int R, int nkeys,
                                                        int start_blocks, int* __restrict__ start,
                                                        int* __restrict__ sorted) {
  const int64_t b = blockIdx.x;
  if (b >= start_blocks) {
    const int64_t j = (b - start_blocks) * 256 + threadIdx.x;
    if (j < R) sorted[j] = ent[j].y;
    return;
  }
  const int64_t k = b * 256 + threadIdx.x;
  if (k > nkeys) return;
  start[k] = ref_start(ent, R, k);
}

static inline int64_t round4i(int64_t n) { return (n + 3) & ~int64_t(3); }

void ref_starts(const int2* ent, int64_t R, int64_t nkeys, int* start, int* sorted, hipStream_t st) {
  const int64_t sb = cdiv(nkeys + 1, 256);
  hipLaunchKernelGGL(ref_start_kernel, dim3((unsigned)(sb + (sorted ? cdiv(R, 256) : 0))), dim3(256), 0, st, ent,
                     (int)R, (int)nkeys, (int)sb, start, sorted);
}

int64_t ref_table_ints(int64_t R, int64_t nkeys) {
  return round4i(nkeys + 1) + round4i(R) + radix_plan(R, nkeys).words();
}

int build_ref_table(const int* keys, int64_t R, int64_t nkeys, int* ws, hipStream_t st,
                    RefTable* out) {
  SLG_REQUIRE(R >= 0 && R < (1LL << 31) && nkeys > 0 && nkeys < (1LL << 31), SLG_E_SHAPE,
              "reference table: %lld references over %lld keys", (long long)R,
              (long long)nkeys);
  int* start = ws;
  int* sorted = start + round4i(nkeys + 1);
  int* sort_ws = sorted + round4i(R);
  const int2* ent = reinterpret_cast<const int2*>(sort_ws);
  if (R > 0)
    ent = radix_sort(RefKeys{keys}, radix_plan(R, nkeys), sort_ws, RadixClear{}, st);
  ref_starts(ent, R, nkeys, start, sorted, st);
  SLG_LAUNCH_CHECK("reference table");
  out->start = start;
  out->sorted = sorted;
  return 0;
}

}  // namespace slg
