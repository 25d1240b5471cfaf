// The rules of sequence_rules.h against what they are for, host code only.
#include <cstdio>
#include <vector>

#include "sequence_rules.h"

using namespace seera;

static int bad = 0;

// A block's sums over `waves` waves, `sums` of them, in the order of events that is
// worst for one barrier a sum: `fast` runs alone until the barrier holds it, again
// and again, and the others read as late as they may. Returns the number of parts
// that a wave read of another sum than its own.
template <class NextHalf>
static int stale_reads(int waves, int sums, int fast, NextHalf&& next_half) {
    std::vector<int> part(2 * waves, -1);
    std::vector<int> half(sums);
    for (int k = 0; k < sums; ++k) half[k] = next_half(k);
    int stale = 0;
    auto write = [&](int wave, int k) { part[half[k] * waves + wave] = k; };
    auto read = [&](int k) {
        for (int w = 0; w < waves; ++w) stale += part[half[k] * waves + w] != k;
    };
    // the barrier of sum k opens when all have written k; then `fast` reads k and
    // writes k + 1, before the others read k and write k + 1
    for (int w = 0; w < waves; ++w) write(w, 0);
    for (int k = 0; k < sums; ++k) {
        read(k);
        if (k + 1 < sums) write(fast, k + 1);
        for (int w = 0; w < waves; ++w)
            if (w != fast) read(k);
        for (int w = 0; w < waves; ++w)
            if (w != fast && k + 1 < sums) write(w, k + 1);
    }
    return stale;
}

static void sums_of_a_row() {
    for (int waves : {2, 4, 16})
        for (int fast = 0; fast < waves; ++fast) {
            Halves halves;
            if (stale_reads(waves, 9, fast, [&](int) { return halves.next(); })) ++bad, std::printf("Halves: %d waves, wave %d ahead\n", waves, fast);
            // planted: one half for each kind of sum. Two kinds in turn are right, one alone is not
            if (stale_reads(waves, 9, fast, [](int k) { return k & 1; })) ++bad, std::printf("two kinds in turn\n");
            if (!stale_reads(waves, 9, fast, [](int) { return 0; })) ++bad, std::printf("a planted fixed half is not seen\n");
        }
}

int main() {
    sums_of_a_row();
    if (!bad) std::puts("all checks passed");
    return bad != 0;
}
