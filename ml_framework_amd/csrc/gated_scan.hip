// gated_scan.hip -- the gated linear recurrence over time, forward and
// backward (seera_hip_gated_scan_fwd / _bwd).
//
//   h_t = a_t h_{t-1} + b_t,   b = x (LINEAR) or (1 - a) x (SIGMOID)
//   c_t = a_t (dh_t + c_{t+1}),  g_t = dh_t + c_{t+1}   (backward; dh0 = c_0)
//
// Both are chains of affine maps c -> A c + B, one chain per (sequence,
// channel). The forward reads x, f and writes h (3 values an element, about 25
// vector instructions of a lane); the backward reads x, f, h, dh and writes dx,
// df (6 values): bytes bound both, and the problem is to have enough of them in
// flight while a chain is serial. Measured (bf16, sigmoid, x and f slices of one
// matrix; floors at 5.35 TB/s, a large copy's rate): 8 x 2048 x 1024 forward 27
// us (floor 19), backward 52 (38); 16 x 2048 x 1024 44 and 88 (38, 75).
//
// df could be had from h_{t-1} - h_t without reading x, but that difference
// cancels for a near 1, with a 16-bit h altogether.
#include <algorithm>
#include <type_traits>

#include "io_types.h"
#include "runtime.h"
#include "sequence.h"
#include "sequence_rules.h"

namespace seera {
namespace {

// A gate's small side: min(a, 1 - a) of a sigmoid, from e^-|f|, so that neither
// side cancels; the other one is 1 minus it, rounded without a bias.
__device__ __forceinline__ float small_side(float f) {
    const float e = __expf(-fabsf(f));
    return e * __builtin_amdgcn_rcpf(1.f + e);
}
// a and 1 - a from f and the small side (LINEAR: a = f and a factor of 1).
template <int GATE>
__device__ __forceinline__ void sides(float f, float small, float& a, float& rest) {
    if (GATE == SEERA_GATE_LINEAR) {
        a = f;
        rest = 1.f;
    } else {
        const float large = 1.f - small;
        a = f >= 0.f ? large : small;
        rest = f >= 0.f ? small : large;
    }
}
template <int GATE>
__device__ __forceinline__ void gates(float f, float& a, float& rest) {
    sides<GATE>(f, GATE == SEERA_GATE_LINEAR ? 0.f : small_side(f), a, rest);
}

__device__ __forceinline__ int steps_of(const int* lengths, int b, int time) {
    return lengths ? min(max(lengths[b], 0), time) : time;
}

// One thread per sequence and V channels, step by step: a generation's single
// token (64 x 1024 channels in 3 us, of which the launch is most), and the calls
// that the tiles do not reach.
template <class T, int V, int GATE>
__global__ __launch_bounds__(256) void scan_fwd_steps(ScanFwd p, ScanShape s, int64_t items) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= items) return;
    const int packs = s.channels / V;
    const int b = (int)(i / packs), c = (int)(i % packs) * V;
    const int n = steps_of(p.lengths, b, s.time);
    const int64_t step = s.time_major ? s.batch : 1;
    int64_t row = s.time_major ? b : (int64_t)b * s.time;
    const int64_t state = (int64_t)b * s.channels + c;
    typedef Pack<T, V> P;
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = p.h0 ? p.h0[state + v] : 0.f;
    for (int t = 0; t < s.time; ++t, row += step) {
        P out;
        if (t < n) {
            const P x = *(const P*)((const T*)p.x + row * p.ldx + c), f = *(const P*)((const T*)p.f + row * p.ldf + c);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float a, rest;
                gates<GATE>(to_f32(f.v[v]), a, rest);
                h[v] = fmaf(a, h[v], rest * to_f32(x.v[v]));
                out.v[v] = from_f32<T>(h[v]);
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) out.v[v] = from_f32<T>(0.f);
        }
        *(P*)((T*)p.h + row * s.channels + c) = out;
    }
    if (p.hT)
#pragma unroll
        for (int v = 0; v < V; ++v) p.hT[state + v] = h[v];
}

template <class T, int V, int GATE>
__global__ __launch_bounds__(256) void scan_bwd_steps(ScanBwd p, ScanShape s, int64_t items) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= items) return;
    const int packs = s.channels / V;
    const int b = (int)(i / packs), c = (int)(i % packs) * V;
    const int n = steps_of(p.lengths, b, s.time);
    const int64_t step = s.time_major ? s.batch : 1;
    const int64_t row0 = s.time_major ? b : (int64_t)b * s.time;
    const int64_t state = (int64_t)b * s.channels + c;
    typedef Pack<T, V> P;
    float carry[V];
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = p.dhT ? p.dhT[state + v] : 0.f;
    for (int t = s.time - 1; t >= 0; --t) {
        const int64_t row = row0 + t * step;
        P ox, of;
        if (t < n) {
            const P f = *(const P*)((const T*)p.f + row * p.ldf + c), dh = *(const P*)((const T*)p.dh + row * s.channels + c);
            P x, h;
            if (GATE == SEERA_GATE_SIGMOID) x = *(const P*)((const T*)p.x + row * p.ldx + c);
            if (t > 0) h = *(const P*)((const T*)p.h + (row - step) * s.channels + c);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float a, rest;
                gates<GATE>(to_f32(f.v[v]), a, rest);
                const float before = t > 0 ? to_f32(h.v[v]) : p.h0 ? p.h0[state + v] : 0.f;
                const float g = to_f32(dh.v[v]) + carry[v], one = g * rest;
                carry[v] = a * g;
                ox.v[v] = from_f32<T>(one);
                of.v[v] = from_f32<T>(GATE == SEERA_GATE_SIGMOID ? one * (before - to_f32(x.v[v])) * a : g * before);
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) ox.v[v] = of.v[v] = from_f32<T>(0.f);
        }
        *(P*)((T*)p.dx + row * p.lddx + c) = ox;
        *(P*)((T*)p.df + row * p.lddf + c) = of;
    }
    if (p.dh0)
#pragma unroll
        for (int v = 0; v < V; ++v) p.dh0[state + v] = carry[v];
}

// ---- tiles: long sequences ----
//
// A block of NT threads owns CL * V channels of one sequence and walks its time
// segment in tiles. Each thread holds L consecutive steps of V channels in
// registers and composes them to one affine map; the maps are composed over a
// wave's slots (shuffles), then over the waves (shared memory), always in the
// order of time, so a result does not depend on timing. With its carry each
// thread then runs its steps again from registers: x, f (dh, h) are read once.
// The next tile's loads are issued before the present one is computed, and pass
// the cache by (non-temporal: backward 8 x 2048 x 1024 57 -> 53 us). Two tiles
// ahead, or more waves, gained nothing: with 256 blocks the pattern of memory (64
// bytes of each row a block) holds the forward at 3.7 TB/s; the same bytes in 512
// blocks of 128 (32 x 512 x 1024) take 24 us, 4.2 TB/s.
//
// DIR 0 runs forward (maps a, b), 1 backward in time (maps a, a dh). A step's
// place in the walk is u, from 0 at the segment's first step of the walk.

struct Segments {
    int count, steps;       // of the time axis; steps is a multiple of the tile
    float2* maps;           // [count][batch * channels]: a segment's composed map
    float* start;           // [batch * channels]: h0 or dhT, kept apart from hT or dh0, which may be the same memory
};

struct ScanPtrs {
    const void *x, *f, *h, *dh;
    void *out, *out2;       // h; or dx, df
    const float *h0, *init; // init: h0 or dhT
    float* last;            // hT or dh0
    const int* lengths;
    int64_t ldx, ldf, ldo, ldo2;
};

template <class T, int V, int L>
struct Steps {
    Pack<T, V> v[L];
};

template <class T, int V, int CL, int NT, int L, int GATE, int DIR, bool MAPS>
__global__ __launch_bounds__(NT) void scan_tiles(ScanPtrs p, ScanShape s, Segments seg, unsigned groups, unsigned blocks) {
    constexpr int W = NT / 64, SL = 64 / CL, kSteps = W * SL * L;
    typedef Pack<T, V> P;
    typedef Steps<T, V, L> S;
    typedef std::conditional_t<sizeof(P) == 8, uint64_t, std::conditional_t<sizeof(P) == 4, uint32_t, uint16_t>> Bits __attribute__((may_alias));
    __shared__ float2 totals[2][W][CL][V];
    // neighbouring channel groups on one die: they share lines of memory
    const unsigned chunk = (blocks + 7) / 8, id = (blockIdx.x & 7) * chunk + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= chunk || id >= blocks) return;
    const unsigned rest_id = id / groups, group = id - rest_id * groups, order = rest_id / (unsigned)s.batch, b = rest_id - order * (unsigned)s.batch;
    // `part` of the walk; the second launch begins with the parts that the first one read last, which are in the cache
    const unsigned part = MAPS || seg.count == 1 ? order : seg.count - 1 - order;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, cl = lane % CL, slot = lane / CL;
    const int segment = DIR == 0 ? (int)part : seg.count - 1 - (int)part;
    const int begin = segment * seg.steps, end = min(begin + seg.steps, s.time), length = end - begin;
    const Walk walk = walk_of(DIR == 1, begin, end, steps_of(p.lengths, b, s.time));
    const int channel = (group * CL + cl) * V;
    const bool active = channel < s.channels;
    // lanes past the last channel do that channel's work again: same loads, same values, same stores
    const int c = active ? channel : s.channels - V;
    const int64_t step = s.time_major ? s.batch : 1, row0 = s.time_major ? b : (int64_t)b * s.time;
    const int64_t state = (int64_t)b * s.channels + c, states = (int64_t)s.batch * s.channels;
    const int first = (wave * SL + slot) * L;  // of the thread's steps in a tile

    // Addresses: the row of a tile's step i is uniform but for the thread's first
    // step, whose distance is 32 bits (far_apart sees to it). In a tile that is not
    // whole, a thread's steps outside of the sequence repeat its live one next to them,
    // and a thread without a live step loads nothing.
    const int64_t dir = DIR == 0 ? 1 : -1;
    auto low_row = [&](int u0) { return row0 + (int64_t)(DIR == 0 ? begin + u0 : end - u0 - kSteps) * step; };
    const unsigned from_low = DIR == 0 ? first : kSteps - 1 - first;
    auto load = [&](const void* base, int64_t ld, int u0, int shift, bool whole, S& to) {
        if (whole) {
            const int64_t stride = dir * step * ld * (int64_t)sizeof(T);
            const char* q = (const char*)base + (low_row(u0) - shift * step) * ld * (int64_t)sizeof(T);
            const unsigned mine = from_low * (unsigned)(step * ld * (int64_t)sizeof(T)) + c * (unsigned)sizeof(T);
#pragma unroll
            for (int i = 0; i < L; ++i, q += stride) {
                const Bits w = __builtin_nontemporal_load((const Bits*)(q + mine));
                __builtin_memcpy(&to.v[i], &w, sizeof(w));
            }
        } else {
#pragma unroll
            for (int i = 0; i < L; ++i) to.v[i] = P{};
            if (!walk.any(u0 + first, L)) return;
#pragma unroll
            for (int i = 0; i < L; ++i) {
                const int t = max(walk.time_of(walk.nearest(u0 + first + i)) - shift, 0);
                to.v[i] = *(const P*)((const char*)base + ((row0 + t * step) * ld + c) * (int64_t)sizeof(T));
            }
        }
    };
    constexpr bool kNeedX = DIR == 0 || (!MAPS && GATE == SEERA_GATE_SIGMOID), kNeedH = DIR == 1 && !MAPS;
    auto load_tile = [&](int u0, S& x, S& f, S& d, S& h) {
        const bool whole = walk.whole(u0, kSteps);
        load(p.f, p.ldf, u0, 0, whole, f);
        if (kNeedX) load(p.x, p.ldx, u0, 0, whole, x);
        if (DIR == 1) load(p.dh, s.channels, u0, 0, whole, d);
        if (kNeedH) load(p.h, s.channels, u0, 1, whole, h);
    };

    float carry[V], h0[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const float* init = MAPS || seg.count == 1 ? p.init : seg.start;
        carry[v] = init ? init[state + v] : 0.f;
        h0[v] = kNeedH && p.h0 ? p.h0[state + v] : 0.f;
        if (MAPS && part == 0 && active && wave == 0 && slot == 0) seg.start[state + v] = carry[v];
        if (MAPS) carry[v] = 0.f;
    }
    float product[V];  // MAPS: of the segment's a
#pragma unroll
    for (int v = 0; v < V; ++v) product[v] = 1.f;

    int parity = 0;
    // From the maps of all slots: z, the state before this one; `carry` moves behind the last.
    auto compose = [&](float (&A)[V], float (&B)[V], float (&z)[V]) {
#pragma unroll
        for (int d = 1; d < SL; d *= 2) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float pa = __shfl_up(A[v], d * CL, 64), pb = __shfl_up(B[v], d * CL, 64);
                if (slot >= d) {
                    B[v] = fmaf(A[v], pb, B[v]);
                    A[v] *= pa;
                }
            }
        }
        if (slot == SL - 1)
#pragma unroll
            for (int v = 0; v < V; ++v) totals[parity][wave][cl][v] = make_float2(A[v], B[v]);
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) z[v] = carry[v];
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float2 t = totals[parity][w][cl][v];
                carry[v] = fmaf(t.x, carry[v], t.y);
                if (MAPS) product[v] *= t.x;
                if (!MAPS && w + 1 == wave) z[v] = carry[v];
            }
        parity ^= 1;
        if (SL > 1 && !MAPS)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float pa = __shfl_up(A[v], CL, 64), pb = __shfl_up(B[v], CL, 64);
                if (slot > 0) z[v] = fmaf(pa, z[v], pb);
            }
    };
    S rx, rf, rd, rh, nx, nf, nd, nh;
    auto compute = [&](int u0) {
        const bool cut = !walk.whole(u0, kSteps);
        if (cut) {
            // steps outside: a = 1 and nothing added
#pragma unroll
            for (int i = 0; i < L; ++i) {
                if (walk.live(u0 + first + i)) continue;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    rf.v[i].v[v] = from_f32<T>(GATE == SEERA_GATE_LINEAR ? 1.f : __builtin_inff());
                    (DIR == 0 ? rx : rd).v[i].v[v] = from_f32<T>(0.f);
                }
            }
        }
        // kept for the second run: a and b; backward the gates' small sides (f and dh
        // are in registers as they came)
        float a[DIR == 0 ? L : 1][V], m[L][V];
        float A[V], B[V];
#pragma unroll
        for (int v = 0; v < V; ++v) A[v] = 1.f, B[v] = 0.f;
#pragma unroll
        for (int i = 0; i < L; ++i) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float f = to_f32(rf.v[i].v[v]), small = GATE == SEERA_GATE_LINEAR ? 0.f : small_side(f);
                float ai, rest;
                sides<GATE>(f, small, ai, rest);
                if (DIR == 0) {
                    a[i][v] = ai;
                    m[i][v] = rest * to_f32(rx.v[i].v[v]);
                    B[v] = fmaf(ai, B[v], m[i][v]);
                } else {
                    m[i][v] = small;
                    B[v] = ai * (to_f32(rd.v[i].v[v]) + B[v]);
                }
                A[v] *= ai;
            }
        }
        float z[V];
        compose(A, B, z);
        if (MAPS) return;
        const int64_t stride = dir * step * p.ldo * (int64_t)sizeof(T), stride2 = dir * step * p.ldo2 * (int64_t)sizeof(T);
        char* q = (char*)p.out + low_row(u0) * p.ldo * (int64_t)sizeof(T);
        char* q2 = (char*)p.out2 + low_row(u0) * p.ldo2 * (int64_t)sizeof(T);
        const unsigned mine = from_low * (unsigned)(step * p.ldo * (int64_t)sizeof(T)) + c * (unsigned)sizeof(T);
        const unsigned mine2 = from_low * (unsigned)(step * p.ldo2 * (int64_t)sizeof(T)) + c * (unsigned)sizeof(T);
        auto second = [&](auto whole_tile) {
            constexpr bool kWhole = decltype(whole_tile)::value;
#pragma unroll
            for (int i = 0; i < L; ++i, q += stride, q2 += stride2) {
                const int u = u0 + first + i;
                P o, o2;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    float one, two = 0.f;
                    if (DIR == 0) {
                        one = z[v] = fmaf(a[i][v], z[v], m[i][v]);
                    } else {
                        float ai, rest;
                        sides<GATE>(to_f32(rf.v[i].v[v]), m[i][v], ai, rest);
                        const float g = to_f32(rd.v[i].v[v]) + z[v];
                        z[v] = ai * g;
                        const float before = kWhole || walk.time_of(u) > 0 ? to_f32(rh.v[i].v[v]) : h0[v];
                        one = g * rest;
                        two = GATE == SEERA_GATE_SIGMOID ? one * (before - to_f32(rx.v[i].v[v])) * ai : g * before;
                    }
                    o.v[v] = from_f32<T>(kWhole || walk.live(u) ? one : 0.f);
                    o2.v[v] = from_f32<T>(kWhole || walk.live(u) ? two : 0.f);
                }
                if (kWhole || u < length) {
                    *(P*)(q + mine) = o;
                    if (DIR == 1) *(P*)(q2 + mine2) = o2;
                }
            }
        };
        // two copies: with the tests in one, its steps are blocks of code too small to overlap
        // (backward 8 x 2048 x 1024 52 -> 68 us)
        if (cut) second(std::false_type{});
        else second(std::true_type{});
    };
    load_tile(0, rx, rf, rd, rh);
    if (!MAPS && part > 0) {
        // the segments before this one: each slot composes its share of their maps
        constexpr int kSlots = W * SL;
        const int per = ((int)part + kSlots - 1) / kSlots, from = (wave * SL + slot) * per;
        float A[V], B[V], z[V];
#pragma unroll
        for (int v = 0; v < V; ++v) A[v] = 1.f, B[v] = 0.f;
        for (int k = from; k < min(from + per, (int)part); ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float2 m = seg.maps[(DIR == 0 ? k : seg.count - 1 - k) * states + state + v];
                B[v] = fmaf(m.x, B[v], m.y);
                A[v] *= m.x;
            }
        compose(A, B, z);
    }
    // The values loaded before the loop are waited for here: in it, a wait for them
    // would be one for the next tile's loads too.
#pragma unroll
    for (int v = 0; v < V; ++v) asm volatile("" : "+v"(carry[v]), "+v"(h0[v]));
    for (int u0 = 0; u0 < length; u0 += kSteps) {
        if (u0 + kSteps < length) load_tile(u0 + kSteps, nx, nf, nd, nh);
        compute(u0);
        rx = nx, rf = nf, rd = nd, rh = nh;
    }
    if (!active || wave || slot) return;
    if (MAPS) {
#pragma unroll
        for (int v = 0; v < V; ++v) seg.maps[segment * states + state + v] = make_float2(product[v], carry[v]);
    } else if ((int)part == seg.count - 1 && p.last) {
#pragma unroll
        for (int v = 0; v < V; ++v) p.last[state + v] = carry[v];
    }
}

constexpr int kLongestTile = 1024;  // steps

// Launches the tiles; parts > 1 splits time (where it is long enough) for a second
// pass over x, f (f, dh), in exchange for that many times the blocks.
template <class T, int V, int CL, int NT, int L, int GATE, int DIR>
int launch_tiles(const ScanShape& s, const ScanPtrs& p, int64_t parts, hipStream_t st) {
    constexpr int kSteps = NT / CL * L;
    static_assert(kSteps <= kLongestTile, "far_apart() counts on it");
    const unsigned groups = (s.channels + CL * V - 1) / (CL * V);
    const int64_t chains = (int64_t)groups * s.batch, states = (int64_t)s.batch * s.channels;
    const int tiles = (s.time + kSteps - 1) / kSteps;
    Segments seg{1, s.time, nullptr, nullptr};
    if (parts > 1 && tiles > 1) {
        const int per = (int)std::max<int64_t>(1, (tiles + parts - 1) / parts);
        seg.count = (tiles + per - 1) / per;
        seg.steps = per * kSteps;
    }
    const int64_t blocks = chains * seg.count;
    if (blocks > kMaxThreads / NT - 8) return fail(SEERA_ERR_INVALID_ARGUMENT, "gated_scan: batch * channels is too large");
    // a whole number of blocks for each of the eight dies
    auto grid = [](int64_t n) { return dim3((unsigned)((n + 7) / 8 * 8)); };
    if (seg.count > 1) {
        void* ws = nullptr;
        const size_t n = (size_t)seg.count * states;
        SEERA_TRY(workspace(n * sizeof(float2) + states * sizeof(float), &ws, st));
        seg.maps = (float2*)ws;
        seg.start = (float*)(seg.maps + n);
        hipLaunchKernelGGL((scan_tiles<T, V, CL, NT, L, GATE, DIR, true>), grid(blocks - chains), dim3(NT), 0, st, p, s, seg, groups, (unsigned)(blocks - chains));
        SEERA_HIP_TRY(hipGetLastError());
    }
    hipLaunchKernelGGL((scan_tiles<T, V, CL, NT, L, GATE, DIR, false>), grid(blocks), dim3(NT), 0, st, p, s, seg, groups, (unsigned)blocks);
    SEERA_HIP_TRY(hipGetLastError());
    return SEERA_OK;
}

// Which tiles a call gets. V: values that may be moved as one in a narrow tile (4
// bytes, or one value where nothing is aligned to that), WV: in a wide one.
//
//   time <= 32, 128  small blocks: 64 x 32 x 1024 forward 5.1 us, with 512 threads 11.3;
//                    64 x 128 x 1024 12.5, with 128 threads 13.9
//   else, by the number of blocks that whole chains give:
//   128 bytes of channels a block from 3 blocks on 4 compute units: fp32 8 x 2048 x 1024
//                    40 us, with 64 bytes 56; below that 64 bytes: bf16 8 x 2048 x 1024 27
//                    us, with 128 bytes (128 blocks) 39
//   64 bytes from 5 blocks on 8, and for short chains: bf16 5 x 4096 x 1024 46 and 92 us,
//                    split 56 and 97; 4 x 300 x 1024 7.8 and 9.4, split 10.4 and 11.7
//   else time is split over about two blocks a compute unit: 4 x 4096 x 1024 40 and 61 us,
//                    whole 45 and 88. That reads x, f (f, dh) twice, in rows of 64 lanes
//                    (bf16 256 bytes: 1 x 4096 x 1024 16.6 us, of four values a lane 21.5)
template <class T, int V, int WV, int GATE, int DIR>
int choose_tiles(const ScanShape& s, const ScanPtrs& p, hipStream_t st) {
    constexpr int E = (int)sizeof(T);
    constexpr int kFull = 128 / (V * E), kHalf = std::min(64, 64 / (V * E));  // lanes over 128 and 64 bytes of channels
    const int64_t cus = device_cus();
    auto chains = [&](int bytes) { return (int64_t)s.batch * ((s.channels * (int64_t)E + bytes - 1) / bytes); };
    if (s.time <= 32) return launch_tiles<T, V, kFull, 128, 8 / V, GATE, DIR>(s, p, 1, st);
    if (s.time <= 128) return launch_tiles<T, V, kFull, 256, 8 / V, GATE, DIR>(s, p, 1, st);
    if (chains(128) * 4 >= cus * 3) return launch_tiles<T, V, kFull, 512, (DIR == 0 ? 16 : 8) / V, GATE, DIR>(s, p, 1, st);
    if (s.time <= 512 || chains(64) * 8 >= cus * 5) return launch_tiles<T, V, kHalf, 512, (DIR == 0 ? 32 : 8) / V, GATE, DIR>(s, p, 1, st);
    const int64_t wide = chains(64 * WV * E);
    constexpr int kValues = DIR == 0 && E == 2 ? 16 : 8;
    return launch_tiles<T, WV, 64, 512, kValues / WV, GATE, DIR>(s, p, (2 * cus + wide - 1) / wide, st);
}

// Whether V values of T may be moved as one: sizes, row distances and addresses.
template <class T, int V>
bool packs(const ScanShape& s, const std::initializer_list<const void*>& ptrs, const std::initializer_list<int64_t>& lds) {
    if (s.channels % V) return false;
    for (int64_t ld : lds)
        if (ld % V) return false;
    for (const void* p : ptrs)
        if (!aligned_to(p, sizeof(T) * V)) return false;
    return true;
}

// Up to this many steps a chain is walked by one thread, without tiles.
constexpr int kFewSteps = 8;

// Whether a tile's rows may lie 2^32 bytes apart, which its 32-bit distances do not
// reach: such a call walks each chain in one thread too.
template <class T>
bool far_apart(const ScanShape& s, const std::initializer_list<int64_t>& lds) {
    return (double)kLongestTile * (s.time_major ? s.batch : 1) * sizeof(T) * (double)std::max(std::max(lds), (int64_t)s.channels) >= 0x1p32;
}

template <class T, int V, int WV, int GATE>
int fwd_v(const ScanShape& s, const ScanFwd& a, hipStream_t st) {
    if (s.time <= kFewSteps || far_apart<T>(s, {a.ldx, a.ldf})) {
        const int64_t items = (int64_t)s.batch * (s.channels / V), blocks = (items + 255) / 256;
        if (blocks >= kMaxThreads / 256) return fail(SEERA_ERR_INVALID_ARGUMENT, "gated_scan: batch * channels is too large");
        hipLaunchKernelGGL((scan_fwd_steps<T, V, GATE>), dim3((unsigned)blocks), dim3(256), 0, st, a, s, items);
        SEERA_HIP_TRY(hipGetLastError());
        return SEERA_OK;
    }
    const ScanPtrs p{a.x, a.f, nullptr, nullptr, a.h, nullptr, nullptr, a.h0, a.hT, a.lengths, a.ldx, a.ldf, s.channels, 0};
    return choose_tiles<T, V, WV, GATE, 0>(s, p, st);
}

template <class T, int V, int WV, int GATE>
int bwd_v(const ScanShape& s, const ScanBwd& a, hipStream_t st) {
    if (s.time <= kFewSteps || far_apart<T>(s, {a.ldx, a.ldf, a.lddx, a.lddf})) {
        const int64_t items = (int64_t)s.batch * (s.channels / V), blocks = (items + 255) / 256;
        if (blocks >= kMaxThreads / 256) return fail(SEERA_ERR_INVALID_ARGUMENT, "gated_scan: batch * channels is too large");
        hipLaunchKernelGGL((scan_bwd_steps<T, V, GATE>), dim3((unsigned)blocks), dim3(256), 0, st, a, s, items);
        SEERA_HIP_TRY(hipGetLastError());
        return SEERA_OK;
    }
    const ScanPtrs p{a.x, a.f, a.h, a.dh, a.dx, a.df, a.h0, a.dhT, a.dh0, a.lengths, a.ldx, a.ldf, a.lddx, a.lddf};
    return choose_tiles<T, V, WV, GATE, 1>(s, p, st);
}

// Two values a lane where everything is aligned to pairs (fp32 narrow tiles take one).
template <class T, int GATE>
int fwd_t(const ScanShape& s, const ScanFwd& a, hipStream_t st) {
    constexpr int E = (int)sizeof(T);
    const auto ptrs = {a.x, a.f, (const void*)a.h};
    const auto lds = {a.ldx, a.ldf};
    if (packs<T, 2>(s, ptrs, lds)) return fwd_v<T, 4 / E, 2, GATE>(s, a, st);
    return fwd_v<T, 1, 1, GATE>(s, a, st);
}
template <class T, int GATE>
int bwd_t(const ScanShape& s, const ScanBwd& a, hipStream_t st) {
    constexpr int E = (int)sizeof(T);
    const auto ptrs = {GATE == SEERA_GATE_LINEAR ? a.f : a.x, a.f, a.h, a.dh, (const void*)a.dx, (const void*)a.df};
    const auto lds = {GATE == SEERA_GATE_LINEAR ? a.ldf : a.ldx, a.ldf, a.lddx, a.lddf};
    if (packs<T, 2>(s, ptrs, lds)) return bwd_v<T, 4 / E, 2, GATE>(s, a, st);
    return bwd_v<T, 1, 1, GATE>(s, a, st);
}
template <class T>
int fwd_gate(const ScanShape& s, const ScanFwd& a, hipStream_t st) {
    return s.gate == SEERA_GATE_LINEAR ? fwd_t<T, SEERA_GATE_LINEAR>(s, a, st) : fwd_t<T, SEERA_GATE_SIGMOID>(s, a, st);
}
template <class T>
int bwd_gate(const ScanShape& s, const ScanBwd& a, hipStream_t st) {
    return s.gate == SEERA_GATE_LINEAR ? bwd_t<T, SEERA_GATE_LINEAR>(s, a, st) : bwd_t<T, SEERA_GATE_SIGMOID>(s, a, st);
}

}  // namespace

int gated_scan_fwd(const ScanShape& s, const ScanFwd& a, hipStream_t st) {
    return s.dtype == SEERA_DTYPE_F32 ? fwd_gate<float>(s, a, st) : s.dtype == SEERA_DTYPE_F16 ? fwd_gate<f16_t>(s, a, st) : fwd_gate<bf16_t>(s, a, st);
}
int gated_scan_bwd(const ScanShape& s, const ScanBwd& a, hipStream_t st) {
    return s.dtype == SEERA_DTYPE_F32 ? bwd_gate<float>(s, a, st) : s.dtype == SEERA_DTYPE_F16 ? bwd_gate<f16_t>(s, a, st) : bwd_gate<bf16_t>(s, a, st);
}

}  // namespace seera
