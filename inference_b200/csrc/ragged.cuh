// Finding one's sequence in a packed batch, by a warp.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace ib200 {

// The last i of [0, n) with key(i) <= t in a nondecreasing list, -1 if there is none; the whole warp calls it.  32 places per
// step.  (What a list in another order gives is some index in range.)
template <typename F>
__device__ __forceinline__ int last_at_or_below(int64_t t, int n, F key) {
  const int lane = threadIdx.x & 31;
  int lo = 0, count = n;
  while (true) {
    const int step = (count + 31) / 32;
    const int at = lo + lane * step;
    const bool in = lane * step < count && key(at) <= t;
    const int c = __popc(__ballot_sync(0xFFFFFFFFu, in));
    if (c == 0) return -1;
    lo += (c - 1) * step;
    if (step == 1) return lo;
    count = min(step, count - (c - 1) * step);
  }
}

}  // namespace ib200
