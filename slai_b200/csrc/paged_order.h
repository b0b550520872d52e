// Orders of work inside the paged chunk kernels, apart from what does the work: plain C++, which the kernels and the host's tests both compile.
#pragma once
#include <stdint.h>

#ifndef PAGED_HD
#ifdef __CUDACC__
#define PAGED_HD __host__ __device__ __forceinline__
#else
#define PAGED_HD inline
#endif
#endif

namespace paged {

// Products of a part of `n` units whose first has number `u`, with two stages of tensor memory that hold a unit's scores and then, in their place, its weights
// (paged_prompt32.cu).  scores(i): QK of unit i, into stage i % 2.  outputs(i): PV of unit i, once the weights stand in stage i % 2.  Products of
// different shapes and accumulators have no order of their own: before scores(i) overwrites the weights of unit i - 2, done(i - 2) waits for the PV that reads them.
template <class Done, class Scores, class Outputs>
PAGED_HD void chunk_products(uint32_t u, int n, Done done, Scores scores, Outputs outputs) {
    auto next = [&](uint32_t i) {
        if (i >= 2) done(i - 2);
        scores(i);
    };
    next(u);
    for (int j = 0; j < n; j++) {
        if (j + 1 < n) next(u + j + 1);
        outputs(u + j);
    }
}

// One slot of a ring, as its filler sees it (paged_prompt.cu).  Fill i completes phase i of the slot's "full" barrier; its reader completes phase i of "empty".
// A wait that gives up returns false: nothing is filled then, nor counted, so that settle() waits for the last fill that was asked for, whatever was left out behind it.
// (A phase is told by its parity alone: a wait for one that nobody begins would be over at once, or never.)
struct SlotFills {
    uint32_t sent = 0;
    template <class Empty>  // empty(i): waits for phase i
    PAGED_HD bool may_fill(Empty empty) const { return sent == 0 || empty(sent - 1); }
    PAGED_HD void filled() { sent++; }
    template <class Full>  // full(i): waits for phase i
    PAGED_HD void settle(Full full) const {
        if (sent > 0) full(sent - 1);
    }
};

}  // namespace paged
