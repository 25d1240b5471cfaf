// f8_routes.h -- which way a product of operands in 8 bits is computed (matmul_f8.hip).
// Host code without HIP, so that the rule is checked on the CPU: tests/cpp/test_f8_routes.cpp
// pins the ways of the sizes that the GPU tests run each of them at.
#pragma once

#include <algorithm>
#include <cstdint>

namespace seera {

// The ways to compute a product: tiles of rows x cols, `at_once` workgroups a compute unit. A
// launch takes `start` us (3.3 of them an empty one) and, for each slice of 128 along K, `few` where most
// compute units have nothing to do, `full` where each has its workgroup, `pair` where each has two. Fitted
// to times of each way at 16 to 512 rows with K = 1024, 4096 and 16384 (bf16; fp32 below: 32 to 777 rows, K = 1024 and
// 4096). Of the chosen way's times at 1024 to 8192 rows it was within 15 % (bf16), and 25 % too low at fp32
// 5501 x 1300 x 1500; memory's rate is not in it (64 x 131072 x 4096 takes 138 us, not 66).
enum F8Way { kSplit, kStream16x64, kStream32x32, kStream32x64, kStream64x64, kTiles128, kTiles128x256, kTiles256, kF8Ways };
struct F8Cost {
    int rows, cols, at_once;
    double start, few, full, pair;
};
constexpr F8Cost kF8Costs16[kF8Ways] = {{16, 16, 1, 1.9, 0, 0, 0}, {16, 64, 1, 3.0, .20, .23, 0}, {32, 32, 1, 3.4, .18, .19, 0}, {32, 64, 1, 3.2, .22, .23, 0},
                                  {64, 64, 2, 3.2, .38, .39, .49}, {128, 128, 1, 4.6, .49, .66, 0}, {128, 256, 1, 6.0, .68, .96, 0}, {256, 256, 1, 9.0, 1.15, 1.63, 0}};
// (fp32 results: twice the matrix instructions' time, which binds the larger tiles)
constexpr F8Cost kF8Costs32[kF8Ways] = {{16, 16, 1, 1.9, 0, 0, 0}, {16, 64, 1, 3.2, .27, .28, 0}, {32, 32, 1, 3.6, .26, .26, 0}, {32, 64, 1, 3.4, .34, .34, 0},
                                  {64, 64, 2, 3.4, .46, .48, .76}, {128, 128, 1, 4.6, 1.40, 1.45, 0}, {128, 256, 1, 6.0, 1.65, 1.95, 0}, {256, 256, 0, 0, 0, 0, 0}};

inline double f8_time(const F8Cost& c, int64_t m, int64_t n, int64_t slices, int64_t cus) {
    const int64_t tiles = ((m + c.rows - 1) / c.rows) * ((n + c.cols - 1) / c.cols);
    // the way from registers reads a row of A and of W for each of its 16 (where there are as many)
    const double full = c.rows == 16 && c.cols == 16 ? .10 + .003 * std::min<int64_t>(m, 16) : c.full, few = c.few > 0 ? c.few : full;
    const int64_t round = cus * c.at_once, rounds = tiles / round, rest = tiles % round;
    double slice = rounds * (c.at_once == 2 ? c.pair : full);
    if (rest) slice += c.at_once == 2 && rest > cus ? c.pair : few + (full - few) * std::min<int64_t>(rest, cus) / cus;
    return c.start + slices * slice;
}

// The way that the table expects to take least time for m x n over `slices` (one at least) of 128 along K.
// The one without tiles in LDS is for up to 16 rows.
inline F8Way f8_way(bool f32, int64_t m, int64_t n, int64_t slices, int64_t cus) {
    const F8Cost* costs = f32 ? kF8Costs32 : kF8Costs16;
    F8Way best = kSplit;
    double least = m <= 16 ? f8_time(costs[kSplit], m, n, slices, cus) : 1e300;
    for (int way = kSplit + 1; way < kF8Ways; ++way) {
        if (!costs[way].at_once) continue;
        const double t = f8_time(costs[way], m, n, slices, cus);
        if (t < least) least = t, best = (F8Way)way;
    }
    return best;
}

}  // namespace seera
