// sequence_rules.h -- rules that the sequence operators' kernels follow, as
// constexpr functions without HIP: the kernels call them, and so do checks on the
// CPU, which see the orders of events and the accesses that a run on the GPU hides.
#pragma once

namespace seera {

// A sum over a block's waves with one barrier: each wave writes its part, all wait,
// each reads every part. A wave that is past the barrier may come to the next sum
// and write before another has read this one's parts, so consecutive sums of a block
// use different halves of the parts, whichever sums they are. Two halves are
// enough: the barrier of the sum between orders the reads of one before the
// writes of the next but one.
struct Halves {
    int now = 0;
    constexpr int next() {
        const int half = now;
        now ^= 1;
        return half;
    }
};

}  // namespace seera
