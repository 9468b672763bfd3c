// How a kernel whose bounded wait ran out waits, again with a limit, for the copies
// that it still has on their way.  Apart from the kernels, and free of device
// code, so that the host can check it against their order of issue.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define RT_LANDING __host__ __device__ __forceinline__
#else
#define RT_LANDING inline
#endif

namespace rt {

// A ring of `depth` barriers: `count` phases in order, from `phase` of `slot` on.
template <typename Wait>
RT_LANDING void land_ring(int depth, int count, int slot, uint32_t phase, Wait wait) {
    for (int i = 0; i < count; ++i) {
        wait(slot, phase);
        if (++slot == depth) {
            slot = 0;
            phase ^= 1;
        }
    }
}

}  // namespace rt
