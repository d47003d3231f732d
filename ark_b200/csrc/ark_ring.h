// ark_ring.h -- a reader's place among barriers that complete in turn.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define ARK_HD __host__ __device__ __forceinline__
#else
#define ARK_HD inline
#endif

namespace ark {

// N barriers, waited for by their phase's parity.  A wait that ran out is final:
// the barrier is then stuck in the phase that was waited for, and a later wait
// for the other parity would be answered at once by the phase before it, whose
// results are long gone.  So nothing is waited for after that.
template <uint32_t N>
struct Ring {
    uint32_t at = 0, parity = 0;
    // lost(): whether a wait has run out; waited(barrier, parity): whether the phase has
    // completed, and if not, lost() from then on
    template <class L, class F>
    ARK_HD bool wait(L lost, F waited) const {
        return !lost() && waited(at, parity);
    }
    ARK_HD void next() {
        if (++at == N) at = 0, parity ^= 1u;
    }
};

}  // namespace ark
