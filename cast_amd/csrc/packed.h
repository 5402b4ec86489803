// Sequences of different lengths behind each other: offsets[b] .. offsets[b + 1] are the rows
// of request b.
#pragma once
#include "rcsa_common.h"

namespace rcsa {

// The last request b of B with first(b) <= item, -1 if there is none, for a first() that does
// not decrease: 64 requests are looked at together, so that the loads of a search are one
// behind the other only ceil(log64 B) times.  The wavefront calls it together; the
// result is uniform.
template <typename First>
__device__ __forceinline__ int request_at(int B, int64_t item, int lane, First&& first) {
  int lo = 0, n = B;
  while (true) {
    const int step = (n + kWave - 1) / kWave;
    const int b = lo + lane * step;
    const bool below = lane * step < n && first(b) <= item;
    const uint64_t at = __ballot(below);
    if (at == 0) return -1;
    const int last = 63 - __builtin_clzll(at);
    lo += last * step;
    n = n - last * step < step ? n - last * step : step;
    if (step == 1) return lo;
  }
}

// Rows [first, first + count) of request b, within [0, rows): whatever the offsets hold.
struct RowsOf {
  int first, count;
};
__device__ __forceinline__ RowsOf rows_of(const int32_t* offsets, int b, int rows) {
  int lo = offsets[b], hi = offsets[b + 1];
  lo = lo < 0 ? 0 : (lo > rows ? rows : lo);
  hi = hi < lo ? lo : (hi > rows ? rows : hi);
  return {lo, hi - lo};
}

}  // namespace rcsa
