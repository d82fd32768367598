// Which keys a query sees, for the cache and window attention kernels.
//
// The query at position i sees key j iff j < len, (not causal or j <= i) and
// (no window or j > i - window or j < sinks): at most two ranges,
// [0, lo_end) and [lo, hi).
#pragma once
#include "common.cuh"

namespace vcb {

struct Visibility {
  int64_t window;   // 0: unlimited
  int64_t sinks;
  int causal;
};

struct KeyRanges {
  int64_t sink_end;   // keys [0, sink_end) ...
  int64_t lo, hi;     // ... and [lo, hi) are visible; sink_end <= lo, and 0 = sink_end where one range suffices
};

// The keys that the query at position i of a sequence of len keys sees.
__host__ __device__ __forceinline__ KeyRanges visible_keys(const Visibility& v, int64_t i, int64_t len) {
  KeyRanges r;
  r.hi = v.causal ? min64(len, i + 1) : len;
  if (r.hi < 0) r.hi = 0;
  r.lo = 0;
  r.sink_end = 0;
  if (v.window > 0) {
    r.lo = i - v.window + 1;
    if (r.lo < 0) r.lo = 0;
    if (r.lo > r.hi) r.lo = r.hi;
    r.sink_end = min64(v.sinks, r.hi);
    if (r.sink_end >= r.lo) {   // the ranges touch: one range
      r.lo = 0;
      r.sink_end = 0;
    }
  }
  return r;
}

}  // namespace vcb
