// Where the parts of an output tile lie in the scratch of the block-scaled attention: plain C++, so that
// its bounds are also checked on the host.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define LQ_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define LQ_HOST_DEVICE inline
#endif

namespace lq {

// The first of run `run`'s rows (of `tile` each) that belong to (sequence, head) `bh` of row tile rt. A run
// that goes from one (sequence, head) on into the next moves on by one slot.
LQ_HOST_DEVICE int64_t part_slot(int rt, int runs, int heads, int run, int bh, int tile) {
  return ((int64_t)rt * ((int64_t)runs + heads) + run + bh) * tile;
}

// The runs that begin and end a (sequence, head) are words that the attention kernel leaves in the scratch:
// the number of its parts, or 0 where they name no runs of the launch (a CTA that gave up a wait marks
// what it did not begin with -1).
LQ_HOST_DEVICE int parts_between(int first, int last, int runs) {
  return first >= 0 && first <= last && last < runs ? last - first + 1 : 0;
}

}  // namespace lq
