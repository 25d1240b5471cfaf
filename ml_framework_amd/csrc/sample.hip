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
// No order is made. A cut is found as (value, how many of the tokens that have it).
// 16-bit logits are counted value by value, two counters a word, in 128 KB of shared
// memory; sums over 128 values next to each other, then the values of the 128 that hold
// the cut, end the search. Others (and rows where a counter runs over: 65536
// tokens of one value) have a histogram over distances from the largest (monotone in l, so a
// bin is a stretch of the order); the tokens of the bin that holds the cut are listed and
// compared with each other, after a histogram of that bin alone if they are too many for
// it, or told apart digit by digit of their values if that is not enough. Tokens too
// far below the largest to have a weight take no part, and the largest are counted apart where
// many threads have met them: in rows masked by the type's lowest value or of equal logits,
// all would meet at one counter.
//
// One workgroup has a row and reads it three to six times, mostly from the caches. 64 x 131072
// bf16 with top-p 61 us (32 values a histogram bin and every token's weight summed there: 132),
// 256 x 50001 fp16 with top-k and top-p 44 (64), 1 x 32768 fp32 with all cuts 33. Instructions
// bind it, about 100 a token of the last (35 of them a weight, 12 of these on 64 bits), and with
// 16-bit logits the random accesses to shared memory as well: an atomic and a read a token.
#include <algorithm>
#include <type_traits>

#include "inference.h"
#include "io_types.h"
#include "runtime.h"

namespace seera {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048;
// The bins cover 42.67 bits of weight, behind which weights are 0.
constexpr float kBinsPerBit = 48.f;
constexpr int kBits = 40;
// 2^-42 of the largest's weight and less is no weight
constexpr double kNone = -42.0;
constexpr int kSegments = 1024;
constexpr int kListed = 512;
// counters of 16-bit values, two a word, and the chunks of them that are summed up. Weights of
// values take the same memory when the cuts are found.
constexpr int kValueWords = 32768, kChunk = 128, kChunks = 2 * kValueWords / kChunk;
constexpr int kTabled = kValueWords / 2;

// The order of values as unsigned numbers (-0 counts as 0).
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t b = __float_as_uint(l + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// 2^(i / 256), times 2^40.
constexpr int kPowers = 256;

struct Row {
    float largest;
    bool many;    // many tokens are the largest: they are counted apart
    float least;  // tokens below it have no weight
    float bins;   // for each unit of distance
    int top;      // the largest's place among the type's values (16 bits)
    int reach;    // and how far below it the last place is that may have a weight
    double scale;   // 256 log2(e) / T
    double lowest;  // of the exponent's 256 parts: no weight, or where the largest is infinite (z is none) 1
    const double* powers;
    // The weight of a token that is not below `least`. Of infinities each has 1. 2^(z / 256) with z = 256 a + i + f is
    // 2^a, a value of the table and three terms of 2^(f / 256)'s series: within 2^-42 of itself.
    // (No branch: the table's values of several tokens are asked for at once.)
    __device__ __forceinline__ uint64_t weight(float l) const {
        const double z = fmax(((double)l - (double)largest) * scale, lowest), n = rint(z), f = z - n;
        const int whole = (int)n;
        constexpr double c1 = 0.6931471805599453 / kPowers, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3;
        const double w = powers[whole & (kPowers - 1)] * fma(f, fma(f, fma(f, c3, c2), c1), 1.0);
        const double power = __hiloint2double(((whole >> 8) + 1023) << 20, 0);
        // rounded to a whole number by the addition of 2^52
        return (uint64_t)(__double_as_longlong(fma(w, power, 0x1p52)) - __double_as_longlong(0x1p52));
    }
    // The bin of a token, and its place in the finer bins that `outer` is divided into.
    // (Infinities, whose difference is none, share a bin too.)
    __device__ __forceinline__ int bin(float l) const { return (int)fminf((largest - l) * bins, kBins - 1.f); }
    __device__ __forceinline__ int inner(float l, int outer) const { return (int)fminf(fmaxf(((largest - l) * bins - outer) * kBins, 0.f), kBins - 1.f); }
    // the order of 16-bit values as whole numbers (-0 counts as 0), and the value at a place
    template <class T>
    static __device__ __forceinline__ int place(T v) {
        const int b = __builtin_bit_cast(uint16_t, v);
        return b & 0x8000 ? 0x8000 - (b & 0x7fff) : b | 0x8000;
    }
    template <class T>
    static __device__ __forceinline__ T value_at(int place) {
        return __builtin_bit_cast(T, (uint16_t)(place & 0x8000 ? place & 0x7fff : 0x8000 | (0x8000 - place)));
    }
};

// A row of logits as a thread sees it: tiles of 64 N tokens for each wave in turn, a tile's
// lane having N next to each other, -infinity past the end. (NaN passes no comparison below.)
template <class T>
struct Logits {
    typedef T Type;
    static constexpr int N = 16 / sizeof(T);
    struct alignas(16) Values {
        T v[N];
    };
    const T* row;
    int vocab, tiles, lane, wave;

    __device__ __forceinline__ Values load(int tile) const {
        const int at = (tile * 64 + lane) * N;
        Values x;
        const bool whole = at + N <= vocab;
        if (whole) __builtin_memcpy(&x, row + at, 16);
        else
#pragma unroll
            for (int i = 0; i < N; ++i) x.v[i] = at + i < vocab ? row[at + i] : from_f32<T>(-__builtin_huge_valf());
        return x;
    }
    __device__ __forceinline__ Logits(const T* logits, int n) : row(logits), vocab(n), tiles((n + 64 * N - 1) / (64 * N)) {
        lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    }
    // How far below the place `top` each of 16-bit values lies (two a register). NaN comes out farther than
    // the type's lowest value.
    typedef uint16_t Steps __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ Steps below(const Values& x, int top) {
        typedef int16_t Signed __attribute__((ext_vector_type(8)));
        const Signed v = __builtin_bit_cast(Signed, x), sign = v >> 15;
        return __builtin_bit_cast(Steps, (Signed)((int16_t)(top - 0x8000) - ((v ^ (sign & (int16_t)0x7fff)) - sign)));
    }
    // f(values, tile) for each of the wave's tiles, the next one being loaded meanwhile
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        if (wave >= tiles) return;
        Values now = load(wave);
        for (int t = wave; t < tiles; t += kWaves) {
            const Values next = load(min(t + kWaves, tiles - 1));
            f(now, t);
            now = next;
        }
    }
    // f(l) for each token
    template <class F>
    __device__ __forceinline__ void tokens(F f) const {
        each([&](const Values& x, int) {
#pragma unroll
            for (int i = 0; i < N; ++i) f(to_f32(x.v[i]));
        });
    }
};

struct Shared {
    double powers[kPowers];
    uint64_t masses[kBins];
    uint64_t wave_mass[kWaves];
    uint64_t above_mass, found_mass, cut_mass;
    uint32_t counts[kBins];
    uint32_t wave_count[kWaves];
    float best[kWaves];
    int best_at[kWaves];
    uint32_t above_count, found_count, listed_count, tops;
    uint32_t cut_key, cut_ties;
    int found;
};

// Shared memory of which a row has one use after the other.
union Scratch {
    uint32_t words[kValueWords];  // 16-bit logits only, as `table` is
    uint64_t table[kTabled];
    struct {
        uint64_t weights[kListed];
        float values[kListed];
    } list;
};
__device__ __forceinline__ Scratch& scratch() {
    extern __shared__ uint64_t memory[];
    return *(Scratch*)memory;
}

// Inclusive sums over the block's threads of (count, mass).
struct Sums {
    uint32_t count;
    uint64_t mass;
};
// Lanes are added in rows of 16, then over the four rows; a lane that nothing comes to adds 0.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ void scan_step(Sums& s) {
    const uint32_t lo = moved<CTRL, ROWS>((uint32_t)s.mass), hi = moved<CTRL, ROWS>((uint32_t)(s.mass >> 32));
    s.count += moved<CTRL, ROWS>(s.count);
    s.mass += (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ Sums wave_scan(Sums s) {
    scan_step<0x111, 0xf>(s);  // row_shr:1
    scan_step<0x112, 0xf>(s);
    scan_step<0x114, 0xf>(s);
    scan_step<0x118, 0xf>(s);
    scan_step<0x142, 0xa>(s);  // row_bcast:15
    scan_step<0x143, 0xc>(s);  // row_bcast:31
    return s;
}
__device__ __forceinline__ Sums block_scan(Sums s, Shared& sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    s = wave_scan(s);
    __syncthreads();
    if (lane == 63) sh.wave_count[wave] = s.count, sh.wave_mass[wave] = s.mass;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        s.count += w < wave ? sh.wave_count[w] : 0;
        s.mass += w < wave ? sh.wave_mass[w] : 0;
    }
    return s;
}

// A cut: tokens above `value` are kept, and the first `ties` of those that have it.
struct Cut {
    uint32_t key;
    uint32_t ties;
    uint64_t mass;  // what is kept
};

// In n entries of sh.counts / sh.masses from `base` on, in rank's order, the one that holds
// the cut: where the count reaches `count` (BY_COUNT), or the mass `mass`. Sets
// sh.found (-1: none) and what lies above it and in it.
template <bool BY_COUNT>
__device__ __forceinline__ void find(int n, uint32_t count, uint64_t mass, Shared& sh, int base = 0) {
    if (threadIdx.x == 0) sh.found = -1;
    const int per = (n + kThreads - 1) / kThreads, first = threadIdx.x * per;
    Sums own = {0, 0};
    for (int i = first; i < min(first + per, n); ++i) own.count += sh.counts[base + i], own.mass += sh.masses[base + i];
    const Sums all = block_scan(own, sh);
    uint32_t c = all.count - own.count;
    uint64_t m = all.mass - own.mass;
    for (int i = first; i < min(first + per, n); ++i) {
        const uint32_t c2 = c + sh.counts[base + i];
        const uint64_t m2 = m + sh.masses[base + i];
        if (BY_COUNT ? c < count && c2 >= count : m < mass && m2 >= mass) {
            sh.found = i;
            sh.above_count = c, sh.above_mass = m;
            sh.found_count = sh.counts[base + i], sh.found_mass = sh.masses[base + i];
        }
        c = c2, m = m2;
    }
    __syncthreads();
}

// The sum over the block's threads, in all of them.
__device__ __forceinline__ uint64_t block_total(uint64_t mass, Shared& sh) {
#pragma unroll
    for (int m = 32; m; m >>= 1) mass += __shfl_xor((unsigned long long)mass, m);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave_mass[threadIdx.x >> 6] = mass;
    __syncthreads();
    mass = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) mass += sh.wave_mass[w];
    return mass;
}

// The cut among the tokens that `in(l)` says are there, above which lie `above_count` and
// `above_mass`, if they are not too many to be listed: where the count reaches `count` (BY_COUNT), or the
// mass `mass`.
template <bool BY_COUNT, class L, class In>
__device__ __forceinline__ bool cut_in_list(const L& logits, const Row& r, In in, uint32_t count, uint64_t mass, uint32_t above_count, uint64_t above_mass,
                                            Shared& sh, Cut& cut) {
    auto& list = scratch().list;
    __syncthreads();
    if (threadIdx.x == 0) sh.listed_count = 0;
    __syncthreads();
    logits.tokens([&](float l) {
        if (!in(l)) return;
        const uint32_t at = atomicAdd(&sh.listed_count, 1u);
        if (at >= kListed) return;
        list.values[at] = l;
        list.weights[at] = r.weight(l);
    });
    __syncthreads();
    const uint32_t n = sh.listed_count;
    if (n > kListed) return false;
    // each token against all others: one of those that have the cut's value writes it down
    if (threadIdx.x < n) {
        const float l = list.values[threadIdx.x];
        const uint64_t w = list.weights[threadIdx.x];
        uint32_t c = above_count, same = 0;
        uint64_t m = above_mass;
        for (uint32_t k = 0; k < n; ++k) {
            const float other = list.values[k];
            const uint64_t ow = list.weights[k];
            c += other > l;
            m += other > l ? ow : 0;
            same += other == l;
        }
        if (BY_COUNT ? c < count && c + same >= count : m < mass && m + same * w >= mass) {
            const uint32_t ties = BY_COUNT ? count - c : (uint32_t)((mass - m + w - 1) / w);
            sh.cut_key = key_of(l), sh.cut_ties = ties, sh.cut_mass = m + ties * w;  // the same from each of them
        }
    }
    __syncthreads();
    cut = Cut{sh.cut_key, sh.cut_ties, sh.cut_mass};
    __syncthreads();
    return true;
}

// The cut inside bin `bin`, above which lie `above_count` and `above_mass`. The histogram's memory is used.
template <bool BY_COUNT, class L>
__device__ __forceinline__ Cut cut_in_bin(const L& logits, const Row& r, int bin, uint32_t count, uint64_t mass, uint32_t above_count, uint64_t above_mass,
                                          Shared& sh) {
    Cut cut;
    auto in_bin = [&](float l) { return l >= r.least && !(r.many && l == r.largest) && r.bin(l) == bin; };
    if (cut_in_list<BY_COUNT>(logits, r, in_bin, count, mass, above_count, above_mass, sh, cut)) return cut;
    // the bin's own histogram
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.counts[i] = 0, sh.masses[i] = 0;
    __syncthreads();
    logits.tokens([&](float l) {
        if (!in_bin(l)) return;
        const int at = r.inner(l, bin);
        if (BY_COUNT) atomicAdd(&sh.counts[at], 1u);
        atomicAdd((unsigned long long*)&sh.masses[at], (unsigned long long)r.weight(l));
    });
    __syncthreads();
    find<BY_COUNT>(kBins, count - above_count, mass - above_mass, sh);
    const int fine = sh.found;
    above_count += sh.above_count, above_mass += sh.above_mass;
    auto in_fine = [&](float l) { return in_bin(l) && r.inner(l, bin) == fine; };
    if (cut_in_list<BY_COUNT>(logits, r, in_fine, count, mass, above_count, above_mass, sh, cut)) return cut;
    uint32_t prefix = 0, in = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (threadIdx.x < 256) sh.counts[threadIdx.x] = 0, sh.masses[threadIdx.x] = 0;
        __syncthreads();
        logits.tokens([&](float l) {
            if (!in_fine(l)) return;
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

// The histogram of the row's tokens; with TOPS of all but the largest ones, whose number is sh.tops: in
// rows of equal logits all would meet at one counter (64 x 131072 1.3 ms; 0.05 without them).
template <bool TOPS, class L>
__device__ __forceinline__ void histogram(const L& logits, const Row& r, bool counts, bool masses, Shared& sh) {
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.counts[i] = 0, sh.masses[i] = 0;
    if (threadIdx.x == 0) sh.tops = 0;
    __syncthreads();
    uint32_t tops = 0;
    logits.each([&](const typename L::Values& x, int) {
#pragma unroll
        for (int from = 0; from < L::N; from += 4) {  // four at a time: registers
            int bin[4];
            uint64_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float l = to_f32(x.v[from + i]);
                if (TOPS) tops += l == r.largest;
                bin[i] = l >= r.least && (!TOPS || l != r.largest) ? r.bin(l) : -1;
                w[i] = masses ? r.weight(l) : 0;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (bin[i] < 0) continue;
                if (counts) atomicAdd(&sh.counts[bin[i]], 1u);
                if (masses) atomicAdd((unsigned long long*)&sh.masses[bin[i]], (unsigned long long)w[i]);
            }
        }
    });
    if (TOPS && tops) atomicAdd(&sh.tops, tops);
    __syncthreads();
}

// 16-bit logits: the tokens of each value (but the largest, as above); of kChunk values their sums.
// False if a counter ran over, which leaves fewer than there are.
template <bool TOPS, class L>
__device__ __forceinline__ bool count_values(const L& logits, const Row& r, bool masses, Shared& sh) {
    typedef typename L::Type T;
    uint32_t* words = scratch().words;
    const int chunks = r.reach / kChunk + 1;
    __syncthreads();
    for (int i = threadIdx.x; i < chunks * (kChunk / 8); i += kThreads) ((uint4*)words)[i] = make_uint4(0, 0, 0, 0);
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.counts[i] = 0, sh.masses[i] = 0;
    if (threadIdx.x == 0) sh.tops = 0;
    __syncthreads();
    uint32_t counted = 0, tops = 0;
    logits.each([&](const typename L::Values& x, int) {
        const typename L::Steps steps = L::below(x, r.top);
#pragma unroll
        for (int i = 0; i < L::N; ++i) {
            const uint32_t at = steps[i];
            if (TOPS) tops += at == 0;
            if (TOPS ? at - 1 >= (uint32_t)r.reach : at > (uint32_t)r.reach) continue;
            atomicAdd(&words[at >> 1], at & 1 ? 65536u : 1u);
            ++counted;
        }
    });
    if (TOPS && tops) atomicAdd(&sh.tops, tops);
    __syncthreads();
    for (int c = logits.wave; c < chunks; c += kWaves) {
        const uint32_t word = words[c * 64 + logits.lane];
        if (!__any(word != 0)) continue;
        Sums s = {0, 0};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t n = i ? word >> 16 : word & 0xffffu;
            s.count += n;
            if (masses && __any(n != 0)) s.mass += n * r.weight(to_f32(Row::value_at<T>(r.top - (c * kChunk + 2 * logits.lane + i))));
        }
        s = wave_scan(s);
        if (logits.lane == 63) sh.counts[c] = s.count, sh.masses[c] = s.mass;
    }
    __syncthreads();
    if (logits.vocab < 65536) return true;
    return block_total((uint64_t)counted - (threadIdx.x < kChunks ? sh.counts[threadIdx.x] : 0u), sh) == 0;
}

// The cut among the values of one chunk.
template <bool BY_COUNT, class L>
__device__ __forceinline__ Cut cut_in_chunk(const L&, const Row& r, int chunk, uint32_t count, uint64_t mass, uint32_t above_count, uint64_t above_mass,
                                            Shared& sh) {
    auto value = [&](int at) { return to_f32(Row::value_at<typename L::Type>(r.top - (chunk * kChunk + at))); };
    __syncthreads();
    if (threadIdx.x < kChunk) {
        const uint32_t n = scratch().words[chunk * (kChunk / 2) + threadIdx.x / 2] >> (threadIdx.x & 1) * 16 & 0xffffu;
        sh.counts[kChunks + threadIdx.x] = n, sh.masses[kChunks + threadIdx.x] = n * r.weight(value(threadIdx.x));
    }
    __syncthreads();
    find<BY_COUNT>(kChunk, count - above_count, mass - above_mass, sh, kChunks);
    above_count += sh.above_count, above_mass += sh.above_mass;
    const float l = value(sh.found);
    const uint64_t w = r.weight(l);
    const uint32_t ties = BY_COUNT ? count - above_count : (uint32_t)min((uint64_t)sh.found_count, (mass - above_mass + w - 1) / w);
    __syncthreads();
    return Cut{key_of(l), ties, above_mass + ties * w};
}

// What top-k and top-p keep.
template <class L>
__device__ __forceinline__ Cut find_cut(const L& logits, const Row& r, uint32_t k, float p, Shared& sh) {
    Cut cut = {0, 0, 0};  // all values are above
    const bool by_mass = p < 1.f;
    if (!k && !by_mass) return cut;
    bool counted = false;
    if constexpr (L::N == 8) counted = r.many ? count_values<true>(logits, r, by_mass, sh) : count_values<false>(logits, r, by_mass, sh);
    if (!counted) {
        if (r.many) histogram<true>(logits, r, k != 0, by_mass, sh);
        else histogram<false>(logits, r, k != 0, by_mass, sh);
    }
    const uint32_t tops = sh.tops;
    const uint64_t top_mass = (uint64_t)tops << kBits;
    auto cut_in = [&](auto by_count, uint32_t count, uint64_t mass) {
        constexpr bool BY_COUNT = decltype(by_count)::value;
        if (BY_COUNT ? count <= tops : mass <= top_mass) {
            const uint32_t ties = BY_COUNT ? count : (uint32_t)((mass + (1ull << kBits) - 1) >> kBits);
            return Cut{key_of(r.largest), ties, (uint64_t)ties << kBits};
        }
        find<BY_COUNT>(counted ? kChunks : kBins, count - tops, mass - top_mass, sh);
        const int found = sh.found;
        if (found < 0) return Cut{0, 0, 0};
        const uint32_t above_count = BY_COUNT ? sh.above_count + tops : 0;
        const uint64_t above_mass = sh.above_mass + top_mass;
        if constexpr (L::N == 8)
            if (counted) return cut_in_chunk<BY_COUNT>(logits, r, found, count, mass, above_count, above_mass, sh);
        return cut_in_bin<BY_COUNT>(logits, r, found, count, mass, above_count, above_mass, sh);
    };
    // the bins of the masses stay where they are wanted after the first cut has used their memory
    uint64_t kept[kBins / kThreads], all = 0;
    if (by_mass) {
#pragma unroll
        for (int i = 0; i < kBins / kThreads; ++i) all += kept[i] = sh.masses[threadIdx.x + i * kThreads];
        all = block_total(all, sh) + top_mass;
    }
    if (k) cut = cut_in(std::true_type(), k, 0);  // none if there are not so many
    if (cut.key) all = cut.mass;
    if (!by_mass) return cut;
    const uint64_t target = max((uint64_t)1, (uint64_t)ceil(p > 0.f ? (double)p * (double)all : 0.0));
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBins / kThreads; ++i) sh.masses[threadIdx.x + i * kThreads] = kept[i];
    __syncthreads();
    const Cut c = cut_in(std::false_type(), 0, target);
    if (c.key && (!cut.key || c.key > cut.key || (c.key == cut.key && c.ties < cut.ties))) cut = c;
    return cut;
}

template <class T>
__global__ __launch_bounds__(kThreads) void sample_rows(Sample a) {
    constexpr int N = 16 / sizeof(T);
    __shared__ Shared sh;
    const int64_t at = blockIdx.x;
    const Logits<T> logits((const T*)a.logits + at * a.ld, a.vocab);
    const int lane = logits.lane, wave = logits.wave, tiles = logits.tiles;
    const float lowest = -__builtin_huge_valf();
    if (threadIdx.x < kPowers) sh.powers[threadIdx.x] = exp2((double)threadIdx.x / kPowers) * (double)(1ull << kBits);

    // the largest, and where it is first
    float best = lowest;
    logits.tokens([&](float l) { best = l > best ? l : best; });
    const float own_best = best;
#pragma unroll
    for (int m = 32; m; m >>= 1) best = fmaxf(best, __shfl_xor(best, m));
    const int alike = __popcll(__ballot(own_best == best));
    if (lane == 0) sh.best[wave] = best, sh.wave_count[wave] = alike;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) best = fmaxf(best, sh.best[w]);
    int many = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) many += sh.best[w] == best ? (int)sh.wave_count[w] : 0;
    const float temperature = a.temperature ? a.temperature[at] : 1.f;
    if (best == lowest || !(temperature > 0.f)) {
        int first = 0x7fffffff;
        if (best != lowest) {
            logits.each([&](const typename Logits<T>::Values& x, int tile) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (to_f32(x.v[i]) == best) first = min(first, (tile * 64 + lane) * N + i);
            });
        }
#pragma unroll
        for (int m = 32; m; m >>= 1) first = min(first, __shfl_xor(first, m));
        if (lane == 0) sh.best_at[wave] = first;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 0; w < kWaves; ++w) first = min(first, sh.best_at[w]);
            a.tokens[at] = best == lowest ? -1 : first;
            if (a.logp) a.logp[at] = best == lowest ? lowest : 0.f;
        }
        return;
    }

    Row r;
    r.largest = best;
    r.many = many >= kThreads / 16;  // as many threads have met it
    r.powers = sh.powers;
    r.bins = (float)min(1.4426950408889634 / (double)temperature * (double)kBinsPerBit, 3e38);
    r.scale = kPowers * 1.4426950408889634 / (double)temperature;
    r.lowest = best < __builtin_huge_valf() ? kNone * kPowers : 0.0;
    // (rounding it does not carry it past a value)
    r.least = best < __builtin_huge_valf() ? fmaxf((float)((double)best + kNone * kPowers / r.scale), -3.4028235e38f) : best;
    if constexpr (N == 8) {
        r.top = Row::place(from_f32<T>(best));
        const T least = from_f32<T>(r.least);  // may be rounded down past it
        r.reach = r.top - Row::place(least) - (to_f32(least) < r.least);
    }
    const int k = a.top_k ? a.top_k[at] : 0;
    const float p = a.top_p ? a.top_p[at] : 1.f;
    const Cut cut = find_cut(logits, r, k > 0 && k < a.vocab ? (uint32_t)k : 0u, p, sh);
    const float min_p = a.min_p ? a.min_p[at] : 0.f;
    const double z_least = min_p > 0.f ? kPowers * log2((double)fminf(min_p, 1.f)) : -1e300;

    // What each segment of the row keeps: the mass above the cut's value, and how many have it.
    // 0: not kept, 1: kept, 2: kept if among the first ties
    const float cut_value = cut.key ? __uint_as_float(cut.key & 0x80000000u ? cut.key & 0x7fffffffu : ~cut.key) : lowest;
    const float last = fmaxf(cut_value, r.least);
    const bool by_weight = min_p > 0.f;
    auto kept = [&](float l) {
        if (!(l >= last)) return 0;
        if (by_weight && l != r.largest && ((double)l - (double)r.largest) * r.scale < z_least) return 0;
        return l > cut_value ? 1 : 2;
    };
    const int per = (tiles + kSegments - 1) / kSegments, segments = (tiles + per - 1) / per;
    __syncthreads();
    // The kept weights of 16-bit values, from the largest's to the last that is kept, are tabled: 12
    // instructions a token, not 40. Values around zero (below 2^-12 of the farthest, more if the table has no
    // room) would take most of the table and few tokens have them: they share an entry, and their tokens' weights
    // are their own.
    bool tabled = false;
    int values = 0, gap_at = -1;
    constexpr int kTies = 48, kGap = 56;  // a tie and a value of the gap are counted in these bits of a weight
    uint16_t gap_from = 0, gap_less = 0;
    if constexpr (N == 8) {
        values = (cut.key ? r.top - Row::place(from_f32<T>(cut_value)) : r.reach) + 1;
        const int above = r.top - 0x8000;  // the largest's places above zero
        const float far = fmaxf(fabsf(r.largest), fabsf(to_f32(Row::value_at<T>(r.top - values + 1))));
        const int half = max(Row::place(from_f32<T>(far * 0x1p-12f)) - 0x8000, (values - kTabled) / 2 + 2);
        const int from = min(max(above - half, 0), values), to = min(max(above + half + 1, 0), values);
        if (to > from) gap_at = gap_from = from, gap_less = to - from - 1;
        const int entries = values - gap_less;
        tabled = entries < kTabled && entries <= a.vocab;
        auto value = [&](int i) { return to_f32(Row::value_at<T>(r.top - i)); };
        if (tabled) {
            for (int i = threadIdx.x; i <= entries; i += kThreads) {
                const float l = value(i > gap_from ? i + gap_less : i);
                const int how = i < entries ? kept(l) : 0;
                scratch().table[i] = i == gap_at ? 1ull << kGap : how == 1 ? r.weight(l) : how == 2 ? 1ull << kTies : 0;
            }
        }
        __syncthreads();
    }
    auto sum_tile = [&](const typename Logits<T>::Values& x, uint64_t& mass, uint32_t& ties) {
        if constexpr (N == 8) {
            if (tabled) {
                typedef typename Logits<T>::Steps Steps;
                const Steps steps = __builtin_elementwise_min(logits.below(x, r.top), (Steps)(uint16_t)values);
                const Steps at = steps - __builtin_elementwise_min(__builtin_elementwise_max(steps, (Steps)gap_from) - gap_from, (Steps)gap_less);
                uint64_t all = 0;
#pragma unroll
                for (int i = 0; i < N; ++i) all += scratch().table[at[i]];
                mass += all & ((1ull << kTies) - 1);
                ties += (uint32_t)(all >> kTies) & 0xff;
                if (!__any(all >> kGap != 0)) return;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    if (at[i] != gap_at) continue;
                    const float l = to_f32(x.v[i]);
                    const int how = kept(l);
                    mass += how == 1 ? r.weight(l) : 0;
                    ties += how == 2;
                }
                return;
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float l = to_f32(x.v[i]);
            if (!__any(l >= last)) continue;  // most tokens of a row are not kept
            const int how = kept(l);
            const uint64_t w = r.weight(l);
            mass += how == 1 ? w : 0;
            ties += how == 2;
        }
    };
    auto segment_done = [&](int s, uint64_t mass, uint32_t ties) {
        const bool some = __any(ties != 0 || mass != 0);
        Sums all = {0, 0};
        if (some) all = wave_scan(Sums{ties, mass});
        if (lane == 63) sh.counts[s] = all.count, sh.masses[s] = all.mass;
    };
    if (per == 1) {
        logits.each([&](const typename Logits<T>::Values& x, int tile) {
            uint64_t mass = 0;
            uint32_t ties = 0;
            sum_tile(x, mass, ties);
            segment_done(tile, mass, ties);
        });
    } else {
        for (int s = wave; s < segments; s += kWaves) {
            uint64_t mass = 0;
            uint32_t ties = 0;
            for (int t = s * per; t < min((s + 1) * per, tiles); ++t) sum_tile(logits.load(t), mass, ties);
            segment_done(s, mass, ties);
        }
    }
    __syncthreads();
    // the weight of the cut's own value (its ties all have it)
    const uint64_t each = cut.ties ? r.weight(cut_value) : 0;
    Sums own = {0, 0};
    if ((int)threadIdx.x < segments) own = Sums{sh.counts[threadIdx.x], sh.masses[threadIdx.x]};
    const Sums above = block_scan(own, sh);
    const uint32_t ties_before = above.count - own.count;
    // the first `ties` of the ties: those of the segments before, and of the segment
    const uint64_t upto = above.mass + min(above.count, cut.ties) * each, own_mass = upto - (above.mass - own.mass) - min(ties_before, cut.ties) * each;
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
        const auto x = logits.load(t);
        uint64_t w[N];
        uint32_t tie[N];
        Sums mine = {0, 0};
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int how = kept(to_f32(x.v[i]));
            w[i] = how == 1 ? r.weight(to_f32(x.v[i])) : 0;
            tie[i] = how == 2;
            mine.count += tie[i];
        }
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
                    a.tokens[at] = (t * 64 + lane) * N + i;
                    if (a.logp) {
                        const float l = to_f32(x.v[i]);
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
    constexpr size_t memory = sizeof(T) == 2 ? sizeof(Scratch) : sizeof(Scratch::list);
    if (memory > 65536) SEERA_HIP_TRY(hipFuncSetAttribute((const void*)sample_rows<T>, hipFuncAttributeMaxDynamicSharedMemorySize, memory));
    for (int left = a.rows; left > 0; left -= kMost) {
        a.rows = std::min(left, kMost);
        hipLaunchKernelGGL((sample_rows<T>), dim3(a.rows), dim3(kThreads), memory, st, a);
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
