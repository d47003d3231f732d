// ark_ring.h -- a reader's place among barriers that complete in turn.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define ARK_HD __host__ __device__ __forceinline__
#else
#define ARK_HD inline
#endif

namespace ark {

// N barriers, waited for by their phase's parity.
template <uint32_t N>
struct Ring {
    uint32_t at = 0, parity = 0;
    ARK_HD void next() {
        if (++at == N) at = 0, parity ^= 1u;
    }
};

// Items first, first + step, ... below end: done(i) as long as it says true, and lost(i)
// for the one where it did not and for all that follow.  A wait that ran out is final:
// the barrier is then stuck in the phase that was waited for, and a later wait for the
// other parity would be answered at once by the phase before it, whose results are
// long gone.
template <class Done, class Lost>
ARK_HD void until_lost(uint32_t first, uint32_t end, uint32_t step, Done done, Lost lost) {
    uint32_t i = first;
    while (i < end && done(i)) i += step;
    for (; i < end; i += step) lost(i);
}

}  // namespace ark
