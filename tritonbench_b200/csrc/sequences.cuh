// Which sequence of a packed batch an index belongs to, found on the device from the batch's bounds.
#pragma once

#include <cuda_runtime.h>

namespace b200fp8 {

// The largest b in [0, batch) with key(b) <= at, by all lanes of a warp, 32 candidates a step.  key does not decrease,
// key(0) <= at; with other keys the answer is any b of the range.
template <typename Key>
__device__ __forceinline__ int search_sequence(int batch, long long at, const Key& key) {
  const int lane = static_cast<int>(threadIdx.x) & 31;
  int lo = 0, n = batch;  // the answer is in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int b = lo + lane * step;
    const bool below = lane * step < n && key(b) <= at;
    const int last = 31 - __clz(__ballot_sync(0xffffffffu, below) | 1);
    n = min(step, n - last * step);
    lo += last * step;
  }
  return lo;
}

}  // namespace b200fp8
