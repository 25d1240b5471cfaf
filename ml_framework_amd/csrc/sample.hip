// sample.hip -- a token for each row of logits (seera_hip_sample).
//
// With d = l - max l, a token's weight is exp(d / T), held as a whole number of
// 2^-40: sums of weights are then the same in whatever order they are taken, and a
// border between two tokens, or of a cut, lies where the formulas have it but for
// 2^-41 of a weight. Tokens are ranked by l, ties by index. The cuts keep a beginning
// of that order: top-k its first k, top-p the fewest whose weights reach p of those
// that top-k kept, min-p those of at least min_p of the first one's weight. The token
// drawn is the first, by index, where the sum of kept weights passes u of their total.
//
// No order is made. A cut is found as (value, how many of the tokens that have it):
// a histogram over distances from the largest (monotone in l, so a bin is a stretch
// of the order), then the bin that holds the cut by the digits of its tokens' values.
#include <algorithm>

#include "inference.h"
#include "io_types.h"
#include "runtime.h"

namespace seera {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr float kBinsPerBit = 48.f;  // 42.67 bits in all: weights behind them are 0
constexpr int kBits = 40;
constexpr int kSegments = 1024;

// The order of values as unsigned numbers (-0 counts as 0).
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t b = __float_as_uint(l + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct Row {
    float largest;
    float bins;     // bins for each unit of distance
    double scale;   // log2(e) / T
    // The token's weight. -infinity and NaN have none; of infinities each has 1.
    __device__ uint64_t weight(float l) const {
        if (l == largest) return 1ull << kBits;
        const double z = ((double)l - (double)largest) * scale;
        return z > -42.0 ? (uint64_t)rint(exp2(z) * (double)(1ull << kBits)) : 0ull;
    }
    __device__ int bin(float l) const {
        if (l == largest) return 0;
        return (int)fminf((largest - l) * bins, (float)(kBins - 1));
    }
};

// The part of a row of logits that a step walks: `f(l, index)` for N values of each
// lane at a time, in tiles of 64 N from `begin` on; -infinity past the end and in
// place of NaN.
template <class T, class F>
__device__ __forceinline__ void tile_values(const T* row, int vocab, int tile, int lane, F f) {
    constexpr int N = 16 / sizeof(T);
    const int at = (tile * 64 + lane) * N;
    T v[N];
    const bool whole = at + N <= vocab;
    if (whole) __builtin_memcpy(v, row + at, 16);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float l = whole ? to_f32(v[i]) : at + i < vocab ? to_f32(row[at + i]) : -__builtin_huge_valf();
        if (l != l) l = -__builtin_huge_valf();
        f(i, l, at + i);
    }
}

struct Shared {
    uint32_t counts[kBins];
    uint64_t masses[kBins];
    uint64_t wave_mass[kWaves];
    uint32_t wave_count[kWaves];
    float best[kWaves];
    int best_at[kWaves];
    uint64_t above_mass, found_mass;
    uint32_t above_count, found_count;
    int found;
};

// Inclusive sums over the block's threads of (count, mass).
struct Sums {
    uint32_t count;
    uint64_t mass;
};
__device__ __forceinline__ uint64_t up64(uint64_t v, int by) {
    return (uint64_t)(uint32_t)__shfl_up((int)(uint32_t)(v >> 32), by) << 32 | (uint32_t)__shfl_up((int)(uint32_t)v, by);
}
__device__ __forceinline__ Sums wave_scan(Sums s) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int by = 1; by < 64; by <<= 1) {
        const uint32_t c = (uint32_t)__shfl_up((int)s.count, by);
        const uint64_t m = up64(s.mass, by);
        if (lane >= by) s.count += c, s.mass += m;
    }
    return s;
}
__device__ __forceinline__ Sums block_scan(Sums s, Shared& sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    s = wave_scan(s);
    __syncthreads();
    if (lane == 63) sh.wave_count[wave] = s.count, sh.wave_mass[wave] = s.mass;
    __syncthreads();
    for (int w = 0; w < wave; ++w) s.count += sh.wave_count[w], s.mass += sh.wave_mass[w];
    return s;
}

// A cut: tokens above `value` are kept, and the first `ties` of those that have it.
struct Cut {
    uint32_t key;
    uint32_t ties;
    uint64_t mass;  // what is kept
};

// In sh.counts / sh.masses [0, n), in rank's order, the entry that holds the cut:
// the one where the count reaches `count` (BY_COUNT), or the mass `mass`. Sets
// sh.found (-1: none) and what lies above it and in it.
template <bool BY_COUNT>
__device__ __forceinline__ void find(int n, uint32_t count, uint64_t mass, Shared& sh) {
    if (threadIdx.x == 0) sh.found = -1;
    const int per = (n + kThreads - 1) / kThreads, first = threadIdx.x * per;
    Sums own = {0, 0};
    for (int i = first; i < min(first + per, n); ++i) own.count += sh.counts[i], own.mass += sh.masses[i];
    const Sums all = block_scan(own, sh);
    uint32_t c = all.count - own.count;
    uint64_t m = all.mass - own.mass;
    for (int i = first; i < min(first + per, n); ++i) {
        const uint32_t c2 = c + sh.counts[i];
        const uint64_t m2 = m + sh.masses[i];
        if (BY_COUNT ? c < count && c2 >= count : m < mass && m2 >= mass) {
            sh.found = i;
            sh.above_count = c, sh.above_mass = m;
            sh.found_count = sh.counts[i], sh.found_mass = sh.masses[i];
        }
        c = c2, m = m2;
    }
    __syncthreads();
}

// The cut inside bin `bin`, above which lie `above_count` and `above_mass`.
template <bool BY_COUNT, class T>
__device__ Cut cut_in_bin(const T* row, int vocab, int tiles, const Row& r, int bin, uint32_t count, uint64_t mass, uint32_t above_count,
                          uint64_t above_mass, Shared& sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t prefix = 0;
    uint32_t in = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (threadIdx.x < 256) sh.counts[threadIdx.x] = 0, sh.masses[threadIdx.x] = 0;
        __syncthreads();
        for (int t = wave; t < tiles; t += kWaves)
            tile_values(row, vocab, t, lane, [&](int, float l, int) {
                if (l == -__builtin_huge_valf() || r.bin(l) != bin) return;
                const uint32_t key = key_of(l);
                if (shift < 24 && key >> (shift + 8) != prefix) return;
                const uint32_t digit = 255 - (key >> shift & 255);  // larger values first
                atomicAdd(&sh.counts[digit], 1u);
                atomicAdd((unsigned long long*)&sh.masses[digit], (unsigned long long)r.weight(l));
            });
        __syncthreads();
        find<BY_COUNT>(256, count - above_count, mass - above_mass, sh);
        prefix = prefix << 8 | (uint32_t)(255 - sh.found);
        above_count += sh.above_count;
        above_mass += sh.above_mass;
        in = sh.found_count;
    }
    const uint64_t each = sh.found_mass / in;  // tokens of one value have one weight
    __syncthreads();
    uint32_t ties = count - above_count;
    if (!BY_COUNT) ties = (uint32_t)min((uint64_t)in, (mass - above_mass + each - 1) / each);
    return Cut{prefix, ties, above_mass + ties * each};
}

template <class T>
__global__ __launch_bounds__(kThreads) void sample_rows(Sample a) {
    constexpr int N = 16 / sizeof(T);
    __shared__ Shared sh;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t at = blockIdx.x;
    const T* row = (const T*)a.logits + at * a.ld;
    const int tiles = (a.vocab + 64 * N - 1) / (64 * N);
    const float lowest = -__builtin_huge_valf();

    // the largest, and where it is first
    float best = lowest;
    int best_at = 0x7fffffff;
    for (int t = wave; t < tiles; t += kWaves)
        tile_values(row, a.vocab, t, lane, [&](int, float l, int i) {
            if (l > best) best = l, best_at = i;
        });
    auto join = [&](float l, int i) {
        if (l > best || (l == best && i < best_at)) best = l, best_at = i;
    };
#pragma unroll
    for (int m = 32; m; m >>= 1) join(__shfl_xor(best, m), __shfl_xor(best_at, m));
    if (lane == 0) sh.best[wave] = best, sh.best_at[wave] = best_at;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) join(sh.best[w], sh.best_at[w]);
    const float temperature = a.temperature ? a.temperature[at] : 1.f;
    if (best == lowest || !(temperature > 0.f)) {
        if (threadIdx.x == 0) {
            a.tokens[at] = best == lowest ? -1 : best_at;
            if (a.logp) a.logp[at] = best == lowest ? lowest : 0.f;
        }
        return;
    }

    Row r;
    r.largest = best;
    r.scale = 1.4426950408889634 / (double)temperature;
    r.bins = (float)min(r.scale * (double)kBinsPerBit, 3e38);
    const int k = a.top_k ? a.top_k[at] : 0;
    const float p = a.top_p ? a.top_p[at] : 1.f;
    const bool by_count = k > 0 && k < a.vocab, by_mass = p < 1.f;
    Cut cut = {0, 0, 0};  // all values are above
    if (by_count || by_mass) {
        for (int i = threadIdx.x; i < kBins; i += kThreads) sh.counts[i] = 0, sh.masses[i] = 0;
        __syncthreads();
        for (int t = wave; t < tiles; t += kWaves)
            tile_values(row, a.vocab, t, lane, [&](int, float l, int) {
                if (l == lowest) return;
                const int b = r.bin(l);
                atomicAdd(&sh.counts[b], 1u);
                atomicAdd((unsigned long long*)&sh.masses[b], (unsigned long long)r.weight(l));
            });
        __syncthreads();
        uint64_t all = 0;
        if (by_mass) {
            // the cut by mass needs what top-k keeps
            uint64_t own = 0;
            for (int i = threadIdx.x; i < kBins; i += kThreads) own += sh.masses[i];
            const Sums s = block_scan(Sums{0, own}, sh);
            __syncthreads();
            if (threadIdx.x == kThreads - 1) sh.above_mass = s.mass;
            __syncthreads();
            all = sh.above_mass;
            __syncthreads();
        }
        int bin_k = -1, bin_p = -1;
        uint32_t count_k = 0, count_p = 0;
        uint64_t mass_k = 0, mass_p = 0;
        if (by_count) {
            find<true>(kBins, (uint32_t)k, 0, sh);
            bin_k = sh.found, count_k = sh.above_count, mass_k = sh.above_mass;
            __syncthreads();
        }
        const bool within = bin_k >= 0;
        // (the histogram is made anew by the cut inside a bin, and once more for the other)
        if (within) {
            cut = cut_in_bin<true>(row, a.vocab, tiles, r, bin_k, (uint32_t)k, 0, count_k, mass_k, sh);
            all = cut.mass;
        }
        if (by_mass) {
            const double share = p > 0.f ? (double)p * (double)all : 0.0;
            const uint64_t target = max((uint64_t)1, (uint64_t)ceil(share));
            if (within) {
                for (int i = threadIdx.x; i < kBins; i += kThreads) sh.counts[i] = 0, sh.masses[i] = 0;
                __syncthreads();
                for (int t = wave; t < tiles; t += kWaves)
                    tile_values(row, a.vocab, t, lane, [&](int, float l, int) {
                        if (l == lowest) return;
                        const int b = r.bin(l);
                        atomicAdd(&sh.counts[b], 1u);
                        atomicAdd((unsigned long long*)&sh.masses[b], (unsigned long long)r.weight(l));
                    });
                __syncthreads();
            }
            find<false>(kBins, 0, target, sh);
            bin_p = sh.found, count_p = sh.above_count, mass_p = sh.above_mass;
            __syncthreads();
            if (bin_p >= 0) {
                const Cut c = cut_in_bin<false>(row, a.vocab, tiles, r, bin_p, 0, target, count_p, mass_p, sh);
                if (!within || c.key > cut.key || (c.key == cut.key && c.ties < cut.ties)) cut = c;
            }
        }
    }
    const float min_p = a.min_p ? a.min_p[at] : 0.f;
    const double z_least = min_p > 0.f ? log2((double)fminf(min_p, 1.f)) : -1e300;

    // What each segment of the row keeps: the mass above the cut's value, and how many have it.
    // 0: not kept, 1: kept, 2: kept if among the first ties
    auto kept = [&](float l) {
        if (l == lowest) return 0;
        const uint32_t key = key_of(l);
        if (key < cut.key) return 0;
        if (l != r.largest && ((double)l - (double)r.largest) * r.scale < z_least) return 0;
        return key > cut.key ? 1 : 2;
    };
    const int per = (tiles + kSegments - 1) / kSegments, segments = (tiles + per - 1) / per;
    __syncthreads();
    for (int s = wave; s < segments; s += kWaves) {
        uint64_t mass = 0;
        uint32_t ties = 0;
        for (int t = s * per; t < min((s + 1) * per, tiles); ++t)
            tile_values(row, a.vocab, t, lane, [&](int, float l, int) {
                const int how = kept(l);
                if (how == 1) mass += r.weight(l);
                ties += how == 2;
            });
        const Sums all = wave_scan(Sums{ties, mass});
        if (lane == 63) sh.counts[s] = all.count, sh.masses[s] = all.mass;
    }
    __syncthreads();
    // the weight of the cut's own value (its ties all have it)
    float cut_value = __uint_as_float(cut.key & 0x80000000u ? cut.key & 0x7fffffffu : ~cut.key);
    const uint64_t each = cut.ties ? r.weight(cut_value) : 0;
    Sums own = {0, 0};
    if ((int)threadIdx.x < segments) own = Sums{sh.counts[threadIdx.x], sh.masses[threadIdx.x]};
    const uint32_t ties_before = block_scan(Sums{own.count, 0}, sh).count - own.count;
    auto among = [&](uint32_t before, uint32_t n) { return before >= cut.ties ? 0u : min(n, cut.ties - before); };
    const uint64_t own_mass = own.mass + among(ties_before, own.count) * each;
    const uint64_t upto = block_scan(Sums{0, own_mass}, sh).mass;
    __syncthreads();
    if (threadIdx.x == kThreads - 1) sh.above_mass = upto;
    __syncthreads();
    const uint64_t total = sh.above_mass;
    const float u = a.uniform[at];
    const uint64_t target = min(total - 1, (uint64_t)((u > 0.f ? (double)fminf(u, 1.f) : 0.0) * (double)total));
    if (upto > target && upto - own_mass <= target) {
        sh.found = threadIdx.x;
        sh.found_mass = upto - own_mass;
        sh.found_count = ties_before;
    }
    __syncthreads();
    if (wave) return;
    // one wave walks the segment
    uint64_t before = sh.found_mass;
    uint32_t ties = sh.found_count;
    for (int t = sh.found * per; t < min((sh.found + 1) * per, tiles); ++t) {
        uint64_t w[N];
        uint32_t tie[N];
        int index = 0;
        Sums mine = {0, 0};
        tile_values(row, a.vocab, t, lane, [&](int i, float l, int where) {
            const int how = kept(l);
            w[i] = how == 1 ? r.weight(l) : 0;
            tie[i] = how == 2;
            mine.count += tie[i];
            if (i == 0) index = where;
        });
        const Sums upto_ties = wave_scan(Sums{mine.count, 0});
        uint32_t rank = ties + upto_ties.count - mine.count;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (tie[i] && rank++ < cut.ties) w[i] = each;
            mine.mass += w[i];
        }
        const Sums s = wave_scan(Sums{0, mine.mass});
        uint64_t m = before + s.mass - mine.mass;
        if (m <= target && m + mine.mass > target) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (m <= target && m + w[i] > target) {
                    a.tokens[at] = index + i;
                    if (a.logp) {
                        const float l = to_f32(row[index + i]);
                        const double d = l == r.largest ? 0.0 : ((double)l - (double)r.largest) / (double)temperature;
                        a.logp[at] = (float)(d - log((double)total * 0x1p-40));
                    }
                }
                m += w[i];
            }
        }
        before += __shfl((unsigned long long)s.mass, 63);
        ties += (uint32_t)__shfl((int)upto_ties.count, 63);
        if (before > target) break;
    }
}

template <class T>
int launch(Sample a, hipStream_t st) {
    constexpr int kMost = (int)(kMaxThreads / kThreads / 2);
    for (int left = a.rows; left > 0; left -= kMost) {
        a.rows = std::min(left, kMost);
        hipLaunchKernelGGL((sample_rows<T>), dim3(a.rows), dim3(kThreads), 0, st, a);
        SEERA_HIP_TRY(hipGetLastError());
        auto on = [&](auto& p, int64_t bytes) {
            if (p) p = (std::decay_t<decltype(p)>)((char*)p + a.rows * bytes);
        };
        on(a.logits, a.ld * sizeof(T));
        on(a.uniform, 4), on(a.temperature, 4), on(a.top_k, 4), on(a.top_p, 4), on(a.min_p, 4), on(a.tokens, 4), on(a.logp, 4);
    }
    return SEERA_OK;
}

}  // namespace

int sample(const Sample& a, hipStream_t st) {
    return a.dtype == SEERA_DTYPE_F32 ? launch<float>(a, st) : a.dtype == SEERA_DTYPE_F16 ? launch<f16_t>(a, st) : launch<bf16_t>(a, st);
}

}  // namespace seera
