// The way that f8_routes.h chooses for each line "fp32 m n k way" of stdin, on 256
// compute units: the sizes at which the GPU tests run the ways.
#include <cstdio>

#include "f8_routes.h"

using namespace seera;

int main() {
    int f32, way, bad = 0, seen[2][kF8Ways] = {};
    long m, n, k;
    while (std::scanf("%d %ld %ld %ld %d", &f32, &m, &n, &k, &way) == 5) {
        const int got = f8_way(f32, m, n, (k + 127) / 128, 256);
        if (got != way) ++bad, std::printf("fp32 %d, %ld x %ld x %ld: way %d, not %d\n", f32, m, n, k, got, way);
        seen[f32 != 0][got] = 1;
        const F8Cost& c = (f32 ? kF8Costs32 : kF8Costs16)[got];
        if (got >= kTiles128 && ((m + c.rows - 1) / c.rows) * ((n + c.cols - 1) / c.cols) <= 256)
            ++bad, std::printf("fp32 %d, %ld x %ld x %ld: no workgroup has a second tile\n", f32, m, n, k);
    }
    for (int w = 0; w < kF8Ways; ++w)
        for (int f = 0; f < 2; ++f)
            if (!seen[f][w] && !(f && !kF8Costs32[w].at_once)) ++bad, std::printf("fp32 %d: no size takes way %d\n", f, w);
    if (!bad) std::puts("all checks passed");
    return bad != 0;
}
