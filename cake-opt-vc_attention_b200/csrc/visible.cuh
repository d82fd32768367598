// Which keys a query sees, for the cache and window attention kernels.
//
// The query at position i sees key j iff j < len, (not causal or j <= i) and
// (no window or j > i - window or j < sinks): at most two ranges,
// [0, lo_end) and [lo, hi).
#pragma once
#include "common.cuh"

namespace vcb {

// Positions and token counts stay below 2^30 and a window or sink count is
// clamped to 2^30 (which is then no limit), so 32-bit arithmetic holds.
constexpr int64_t kMostTokens = int64_t(1) << 30;

inline int64_t max64(int64_t a, int64_t b) { return a > b ? a : b; }

struct Visibility {
  int window;   // 0: unlimited
  int sinks;
  int causal;
};

inline Visibility visibility(int64_t window, int64_t sinks, int causal) {
  return Visibility{static_cast<int>(min64(window, kMostTokens)), static_cast<int>(min64(sinks, kMostTokens)), causal};
}

struct KeyRanges {
  int sink_end;   // keys [0, sink_end) ...
  int lo, hi;     // ... and [lo, hi) are visible; sink_end <= lo, and 0 = sink_end where one range suffices
};

// The keys that the query at position i of a sequence of len keys sees.
__host__ __device__ __forceinline__ KeyRanges visible_keys(const Visibility& v, int i, int len) {
  KeyRanges r;
  r.hi = v.causal && i + 1 < len ? i + 1 : len;
  if (r.hi < 0) r.hi = 0;
  r.lo = 0;
  r.sink_end = 0;
  if (v.window > 0) {
    r.lo = i - v.window + 1;
    if (r.lo < 0) r.lo = 0;
    if (r.lo > r.hi) r.lo = r.hi;
    r.sink_end = v.sinks < r.hi ? v.sinks : r.hi;
    if (r.sink_end >= r.lo) {   // the ranges touch: one range
      r.lo = 0;
      r.sink_end = 0;
    }
  }
  return r;
}

}  // namespace vcb
