// Device helpers shared by the append and the attention over the paged 8-bit cache.
#pragma once
#include "common.cuh"
#include "held8.cuh"
#include "kv8.h"

namespace ib200 {

// The sequence whose new tokens include token t, its first new token and their number; false for a token behind (or before) all of them.
__device__ __forceinline__ bool find_sequence(const int* cu, int batch, int each, int t, int& b, int& first, int& count) {
  if (!cu) {
    b = t / each;
    first = b * each;
    count = each;
    return b < batch;
  }
  int lo = 0, hi = batch;  // the largest b with cu[b] <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  b = lo;
  first = cu[b];
  const int end = cu[b + 1];
  count = end - first;
  return batch > 0 && first >= 0 && first <= t && t < end;
}

}  // namespace ib200
