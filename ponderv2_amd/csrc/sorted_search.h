// Search in sorted keys.  Host and device code alike: nothing in it is the device's own.
#pragma once

namespace pv2 {

// first position of a key >= v among n < 2^31 sorted ones; keys: anything that has [int]
template <typename Keys>
__host__ __device__ inline int lower_bound(const Keys& keys, int n, int v) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = lo + ((hi - lo) >> 1);   // (lo + hi passes the largest int where n is above 2^30)
    if (keys[mid] < v) lo = mid + 1; else hi = mid;
  }
  return lo;
}

}  // namespace pv2
