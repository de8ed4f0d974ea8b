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

// Passes `others` stages of a tile, from ring number `it` on, that another role
// reads and frees; `landed(it)` waits for a stage's copies.
//
// A role has to wait for those as for its own.  A barrier's parity tells a stage's
// present fill from the one before only to a role that has seen every fill: past one
// that was skipped, the wait for the next lets the role into a stage that still
// holds, or still receives, the skipped one.  For the same reason the other role must
// not free its stages, and so have them filled again, before this one has seen them:
// it is told so on a barrier.  (One of two barriers in turn is enough for that with a
// ring of three: the tile after the next cannot be seen before the stages of this
// one are free.)
template <class Landed>
YL_HOST_DEVICE bool pass_stages(uint32_t& it, int others, Landed landed) {
  for (int e = 0; e < others; ++e, ++it)
    if (!landed(it)) return false;
  return true;
}

}  // namespace yl
