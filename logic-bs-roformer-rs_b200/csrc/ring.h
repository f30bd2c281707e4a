// The end of a ring of stages (plain C++, so that the host can check it too).
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define LBRR_HD __host__ __device__ __forceinline__
#else
#define LBRR_HD inline
#endif

namespace lbrr {

// Use u of a ring fills stage u % STAGES, and the consumer's arrival that frees
// it completes phase u / STAGES of the stage's barrier.  A producer waits for that
// arrival before it fills the stage again, so after `uses` of them nobody has
// waited for the last STAGES arrivals.  This waits for those, oldest first;
// wait(stage, parity) returns false to give up.
template <int STAGES, class Wait>
LBRR_HD bool drain_ring(uint32_t uses, Wait wait) {
  for (uint32_t u = uses > STAGES ? uses - STAGES : 0; u < uses; ++u)
    if (!wait(static_cast<int>(u % STAGES), (u / STAGES) & 1u)) return false;
  return true;
}

}  // namespace lbrr
