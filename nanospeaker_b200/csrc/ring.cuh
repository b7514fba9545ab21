// A ring of stages in shared memory, filled by copies that a barrier per stage waits for. (No CUDA in here: the
// tests compile it for the host too.)
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define MOE_RING_FN __host__ __device__ __forceinline__
#else
#define MOE_RING_FN inline
#endif

namespace moe {

// wait(stage, parity) for the uses whose copies may be in flight when the reader gives up at use `first`: a ring's
// worth from there on, as it frees no stage any more. With waits that have a limit, for some may never be started;
// but what landed behind a kernel's end would land in the shared memory of the next one.
template <typename Wait>
MOE_RING_FN void unseen_uses(uint32_t first, uint32_t stages, Wait wait) {
  for (uint32_t i = first; i < first + stages; ++i) wait(i % stages, (i / stages) & 1);
}

}  // namespace moe
