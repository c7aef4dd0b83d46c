// Sequences packed one after another: which of them a block or wave works on, found from their starts alone.
#pragma once
#include "fw_common.h"

namespace fw {

// The last sequence s with start(s) <= slot, for starts that ascend with s, or -1; every lane of the wave asks with the
// same slot. 64 sequences at a time: one round of loads up to 64 sequences, two up to 4096. Of starts that do not
// ascend some sequence below n is found.
template <class F>
__device__ __forceinline__ int last_started(int n, int64_t slot, F start) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = n;
  for (;;) {
    const int step = (hi - lo + 63) / 64, s = lo + lane * step;
    const int found = __popcll(__builtin_amdgcn_ballot_w64(s < hi && start(min(s, n - 1)) <= slot));
    if (found == 0) return -1;
    lo += (found - 1) * step;
    if (step == 1) return lo;
    hi = min(hi, lo + step);
  }
}

// Whether a launch of so many blocks stays within the 2^32 - 1 threads of a grid's axis.
inline bool grid_ok(int64_t blocks, int threads) { return blocks <= 0xFFFFFFFFll / threads; }

// A start or end within the rows there are.
__device__ __forceinline__ int64_t within(int64_t x, int64_t low, int64_t rows) { return min(max(x, low), rows); }

}  // namespace fw
