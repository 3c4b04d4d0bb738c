// Relative positions: what the bias's own kernels and the attention kernels share.
//
// Distances of one side fall into `side` buckets by their starts; beyond far = start[side - 1] all
// share the last. A head's bias is therefore a function of rel = j - i - shift that is constant
// outside (-far, far): kernels expand it to one value per rel in [-far, far]. far is 1 at least, so
// that the two sides stay apart.
#pragma once
#include "common.cuh"

namespace b200 {
namespace relative {

__host__ __device__ __forceinline__ int buckets_of(const b200_relative& r) { return r.bidirectional ? 2 * r.side : r.side; }
__host__ __device__ __forceinline__ int far_of(const b200_relative& r) { return r.start[r.side - 1] > 1 ? r.start[r.side - 1] : 1; }

// the bucket of a relative position, |rel| clamped to far by the caller or not
__device__ __forceinline__ int bucket_of(const b200_relative& r, int rel) {
  int n = r.bidirectional ? abs(rel) : max(0, -rel), lo = 0, hi = r.side;
  while (hi - lo > 1) {  // the last start <= n
    const int mid = (lo + hi) >> 1;
    if (r.start[mid] <= n) lo = mid;
    else hi = mid;
  }
  return lo + (r.bidirectional && rel > 0 ? r.side : 0);
}

// the sum of a bucket's positions from the sums by rel (rel + far; the ends hold all beyond them): neighbours on each side, in order
__device__ __forceinline__ float bucket_sum(const b200_relative& r, int far, const float* by_rel, int bucket) {
  const int side = bucket % r.side;
  const int lo = r.start[side], hi = side + 1 < r.side ? r.start[side + 1] : far + 1;  // distances lo .. hi - 1
  float s = 0.f;
  if (r.bidirectional && bucket >= r.side) {
    for (int n = max(lo, 1); n < hi; ++n) s += by_rel[far + n];
    return s;
  }
  for (int n = lo; n < hi; ++n) s += by_rel[far - n];
  if (!r.bidirectional && lo == 0 && hi > 0)
    for (int n = 1; n <= far; ++n) s += by_rel[far + n];  // later keys share the first bucket
  return s;
}

inline int check(const char* what, const b200_relative* r) {
  B200_REQUIRE(r, "%s: no buckets", what);
  B200_REQUIRE(r->side >= 1 && r->side <= B200_RELATIVE_MAX_SIDE, "%s: %d buckets a side (1 to %d)", what, r->side, B200_RELATIVE_MAX_SIDE);
  B200_REQUIRE(r->start[0] == 0, "%s: the first bucket starts at %d, not 0", what, r->start[0]);
  for (int i = 1; i < r->side; ++i)
    B200_REQUIRE(r->start[i] >= r->start[i - 1] && r->start[i] <= B200_RELATIVE_MAX_FAR, "%s: bucket %d starts at %d after %d (at most %d)",
                 what, i, r->start[i], r->start[i - 1], B200_RELATIVE_MAX_FAR);
  return B200_OK;
}

}  // namespace relative
}  // namespace b200
