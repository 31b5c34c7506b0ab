// The sums of a page plan: pages that requests need, and which of them are granted.
// Host and device.
#pragma once

#include <cstdint>

#if defined(__HIPCC__)
#define TQ_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define TQ_HOST_DEVICE inline
#endif

namespace tq {

// Of needs, also within one scan: 1,024 sequences of up to 2^26 pages each, 2^20 in all.
using PlanSum = int64_t;

// Pages needed before a request, as far as they matter: more than a pool has is one more.
TQ_HOST_DEVICE int plan_before(PlanSum needed, int num_pages) {
  return static_cast<int>(needed <= num_pages ? needed : static_cast<PlanSum>(num_pages) + 1);
}

// Whether a request for `need` pages (-1: refused already) is granted, with `found` free
// ones (at most num_pages) and `before` of them spoken for.
TQ_HOST_DEVICE bool plan_grants(int need, int before, int found) {
  return need == 0 || (need > 0 && before <= found && need <= found - before);
}

}  // namespace tq
