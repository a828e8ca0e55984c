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

// How many of R entries sorted by key (x) lie below key k.
__device__ inline int ref_start(const int2* __restrict__ ent, int R, int64_t k) {
  int lo = 0, hi = R;
  while (lo < hi) {
    const int mid = lo + ((hi - lo) >> 1);
    if (ent[mid].x < k) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// start[k] = ref_start of every key k in [0, nkeys]; with sorted, also the
// entries' references (y) alone.
void ref_starts(const int2* ent, int64_t R, int64_t nkeys, int* start, int* sorted, hipStream_t st);

}  // namespace slg
