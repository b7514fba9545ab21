// The status word's codes (0 = fine), and which of them concern a kernel that runs. (The choice has no CUDA in it:
// the tests compile it for the host too.)
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define MOE_STATUS_FN __host__ __device__ __forceinline__
#else
#define MOE_STATUS_FN inline
#endif

namespace moe {

enum DevStatus { ST_OK = 0, ST_WAIT_TIMEOUT = 1, ST_BAD_EXPERT = 2, ST_BAD_OFFSETS = 3 };

// Whether waits give up at this code: at a wait that ran out, whose data will not come. The other codes report an
// input that the kernels have already taken into range, this call's or an earlier one's: nobody stops for them.
MOE_STATUS_FN bool status_ends_waits(int32_t status) { return status == ST_WAIT_TIMEOUT; }

#ifdef __CUDACC__
// Reports an input. A code that is there stays: an earlier report, or a wait that ran out, which is worse.
__device__ __forceinline__ void report_input(int32_t* status, DevStatus code) { atomicCAS(status, ST_OK, code); }
#endif

}  // namespace moe
