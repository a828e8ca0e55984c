// Buckets of references for the gather form of a scatter (the input
// gradients of the soft backward): given keys[r] in [0, nkeys) for r < R,
// build start[0..nkeys] (exclusive prefix of the bucket sizes) and sorted[]
// where sorted[start[k] .. start[k+1]) lists the r with key k in ascending
// order. The order is fixed, so sums over a bucket are the same on every call.
#pragma once

#include "slg_common.h"

namespace slg {

struct RefTable {
  int* start;   // [nkeys + 1]
  int* sorted;  // [R]
};

// Workspace ints for R references over nkeys buckets (16-byte multiples).
int64_t ref_table_ints(int64_t R, int64_t nkeys);

// Enqueue the build on st; R < 2^31, nkeys < 2^31. Returns 0 or an error.
int build_ref_table(const int* keys, int64_t R, int64_t nkeys, int* ws, hipStream_t st,
                    RefTable* out);

// How many of R entries sorted by key (x) lie below key k: three reads a step
// leave a quarter of the range (by halves, twice as many reads one after the
// other).
__device__ inline int ref_start(const int2* __restrict__ ent, int R, int64_t k) {
  int lo = 0, n = R;  // between lo and lo + n
  while (n > 0) {
    const int a = lo + (n >> 2), b = lo + (n >> 1), c = b + (n >> 2), end = lo + n;
    const bool pa = ent[a].x < k, pb = ent[b].x < k, pc = ent[c].x < k;
    lo = pc ? c + 1 : pb ? b + 1 : pa ? a + 1 : lo;
    n = (pc ? end : pb ? c : pa ? b : a) - lo;
  }
  return lo;
}

// start[k] = ref_start of every key k in [0, nkeys]; with sorted, also the
// entries' references (y) alone.
void ref_starts(const int2* ent, int64_t R, int64_t nkeys, int* start, int* sorted, hipStream_t st);

}  // namespace slg
