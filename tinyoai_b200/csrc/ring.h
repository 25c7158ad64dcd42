// Phases of a ring of mbarriers, one a stage: copy i goes to stage i % stages
// and completes phase i / stages of its barrier.
#pragma once

#ifdef __CUDACC__
#define TCU_RING_FN __host__ __device__ inline
#else
#define TCU_RING_FN inline
#endif

namespace tcu {

// Parity of the phase that the last of `sent` copies to go to `stage`
// completes; -1: none of them did.
TCU_RING_FN int ring_last_parity(int sent, int stage, int stages) {
  return stage < sent ? ((sent - 1 - stage) / stages) & 1 : -1;
}

}  // namespace tcu
