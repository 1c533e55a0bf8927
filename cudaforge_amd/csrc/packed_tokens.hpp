// packed_tokens.hpp -- batches whose sequences' tokens lie one after another.
#pragma once

#include <hip/hip_runtime.h>

namespace cfa {

// The sequence b and the place j in it of token t, for a whole wave at once; false
// where t belongs to none (in front of the first, or behind the last).  a.cu
// [B + 1], rising, or null: a.n tokens a sequence.
template <class A>
__device__ __forceinline__ bool place_token(const A &a, int t, int lane, int &b, int &j) {
  if (!a.cu) {
    b = t / a.n;
    j = t - b * a.n;
    return true;
  }
  b = 0;  // ends at or before t
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const bool ended = b0 + lane < a.B && a.cu[b0 + lane + 1] <= t;
    b += __popcll(__ballot(ended));
  }
  if (b >= a.B) return false;
  j = t - a.cu[b];
  return j >= 0;
}

}  // namespace cfa
