// A warp's ring of asynchronous copies into shared memory: which stage the next copy goes to, which is waited for
// next and with which parity, and, where a wait gives up, which copies are still in flight and have to land before
// the block may end.
//
// Plain counters of copies, not ring positions: a full ring and an empty one have the same positions.
#pragma once

#include "fastdiv.h"

namespace mfb {

template <unsigned DEPTH>
struct CopyRing {
    static_assert(DEPTH != 0 && (DEPTH & (DEPTH - 1)) == 0, "the counters may wrap");
    unsigned issued = 0, consumed = 0;

    MFB_HD unsigned next() const { return issued % DEPTH; }  // stage of the next copy
    // The oldest copy that is not consumed, and those behind it.
    MFB_HD unsigned stage(unsigned behind = 0) const { return (consumed + behind) % DEPTH; }
    MFB_HD unsigned parity(unsigned behind = 0) const { return (consumed + behind) / DEPTH & 1; }

    // Waits, by wait(stage, parity), for every copy in flight; false if one of the waits gave up.
    template <typename Wait>
    MFB_HD bool drain(Wait&& wait) {
        bool landed = true;
        for (; consumed != issued; ++consumed) landed = wait(stage(), parity()) && landed;
        return landed;
    }
};

}  // namespace mfb
