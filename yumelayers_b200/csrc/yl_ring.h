// yl_ring.h -- how a role takes the stages of a shared-memory ring (host and
// device, so that the order of its waits can be run on the CPU).
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define YL_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define YL_HOST_DEVICE inline
#endif

namespace yl {

// A role's way through the stages of a tile, from ring number `it` on: `products`
// that it works on, then `others` that another role reads and frees.  next() waits
// with `landed(it)` for a stage's copies and says whether there is a product to do;
// the loop's increment passes on to the next.
//
//   for (StageWalk w{products, others}; w.next(it, landed); w.pass(it)) ...
//
// The stages of the others are waited for as well.  A barrier's parity tells a
// stage's present fill from the one before only to a role that has seen every
// fill: past one that was skipped, the wait for the next lets this role into a
// stage that still holds, or still receives, the skipped one.  For the same reason
// the other role must not free its stages, and so have them filled again, before
// this walk has seen them: what lets it begin (the last accumulator of a tile) is
// handed over behind the walk.
struct StageWalk {
  int products, others;
  int at = 0;
  bool lost = false;  // a wait ran out

  template <class Landed>
  YL_HOST_DEVICE bool next(uint32_t& it, Landed landed) {
    for (; at < products + others; pass(it)) {
      lost = !landed(it);
      if (lost) return false;
      if (at < products) return true;
    }
    return false;
  }
  YL_HOST_DEVICE void pass(uint32_t& it) {
    ++at;
    ++it;
  }
};

}  // namespace yl
