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

// The stages of a pair of CTAs whose copies both report to the leader's barriers,
// `slots` of them.  The leader issued `own` stages, its peer `peer`; a stage is
// issued once the one `slots` before it has been read, so the last `slots` hold every
// copy on its way.  The leader's issue announces the bytes of both: of a stage that
// the peer alone issued its bytes are announced here, of one that the leader alone
// issued the peer's are made up for.
template <typename Expect, typename Complete, typename Wait>
RT_LANDING void land_pair(int slots, int own, int peer, Expect expect, Complete complete, Wait wait) {
    const int last = own > peer ? own : peer;
    for (int i = last > slots ? last - slots : 0; i < last; ++i) {
        if (i >= own)
            expect(i % slots);
        else if (i >= peer)
            complete(i % slots);
        wait(i % slots, (uint32_t)(i / slots) & 1u);
    }
}

}  // namespace rt
