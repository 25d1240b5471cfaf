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

// A block's walk over the steps begin <= t < end of a sequence that has n of them:
// step u of the walk, from 0, is time_of(u). Its rows of memory are those of steps
// t < n alone: steps lo <= u < hi.
struct Walk {
    bool back;
    int begin, end, n, lo, hi;
    constexpr int length() const { return end - begin; }
    constexpr int time_of(int u) const { return back ? end - 1 - u : begin + u; }
    constexpr bool live(int u) const { return u >= lo && u < hi; }
    // whether any of `steps` steps from u on is live
    constexpr bool any(int u, int steps) const { return (u > lo ? u : lo) < (u + steps < hi ? u + steps : hi); }
    // whether all of them are and, backward, have a step before them (by the walk's end and n: by
    // lo and hi the scan's forward is 4 % slower)
    constexpr bool whole(int u, int steps) const {
        if (u + steps > length()) return false;
        return back ? end - u <= n && end - u - steps > 0 : begin + u + steps <= n;
    }
    // the live step next to u (where there is one)
    constexpr int nearest(int u) const { return u < lo ? lo : u >= hi ? hi - 1 : u; }
};
constexpr Walk walk_of(bool back, int begin, int end, int n) {
    const int length = end - begin, inside = n < begin ? 0 : n > end ? length : n - begin;
    return Walk{back, begin, end, n, back ? length - inside : 0, back ? length : inside};
}

}  // namespace seera
