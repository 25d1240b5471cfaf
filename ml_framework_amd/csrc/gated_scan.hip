// gated_scan.hip -- the gated linear recurrence over time, forward and
// backward (seera_hip_gated_scan_fwd / _bwd).
//
//   h_t = a_t h_{t-1} + b_t,   b = x (LINEAR) or (1 - a) x (SIGMOID)
//   c_t = a_t (dh_t + c_{t+1}),  g_t = dh_t + c_{t+1}   (backward; dh0 = c_0)
//
// Both are chains of affine maps c -> A c + B, one chain per (sequence,
// channel). The forward reads x, f and writes h; the backward reads x, f, h,
// dh and writes dx, df: memory bound.
#include <algorithm>

#include "io_types.h"
#include "runtime.h"
#include "sequence.h"

namespace seera {
namespace {

// a and 1 - a of a gate, each with its own small relative error: sigmoid is
// taken from e^-|f|, so that neither side cancels.
template <int GATE>
__device__ __forceinline__ void gates(float f, float& a, float& rest) {
    if (GATE == SEERA_GATE_LINEAR) {
        a = f;
        rest = 1.f;
    } else {
        const float e = __expf(-fabsf(f));
        const float s = e * __builtin_amdgcn_rcpf(1.f + e);  // the smaller of the two
        const float l = 1.f - s;                             // near 1: rounded without a bias
        a = f >= 0.f ? l : s;
        rest = f >= 0.f ? s : l;
    }
}

__device__ __forceinline__ int steps_of(const int* lengths, int b, int time) {
    return lengths ? min(max(lengths[b], 0), time) : time;
}

// One thread per sequence and V channels, step by step.
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
// A block of kTile threads owns CL * V channels of one sequence and walks its
// time segment in tiles. Each thread holds L consecutive steps of V channels in
// registers and composes them to one affine map; the maps are composed over a
// wave's slots (shuffles), then over the waves (shared memory), always in the
// order of time, so a result does not depend on timing. With its carry each
// thread then runs its steps again from registers: x, f (dh, h) are read once.
// The next tile's loads are issued before the present one is computed.
//
// DIR 0 runs forward (maps a, b), 1 backward in time (maps a, a dh).

constexpr int kTile = 512, kWaves = kTile / 64;

struct Segments {
    int count, steps;       // of the time axis; steps is a multiple of the tile
    float2* maps;           // [count][batch * channels]: a segment's composed map
    const float* carry;     // [count][batch * channels]: the state before a segment; null: h0 / dhT
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

template <class T, int V, int CL, int L, int GATE, int DIR, bool MAPS>
__global__ __launch_bounds__(kTile) void scan_tiles(ScanPtrs p, ScanShape s, Segments seg, int groups, int64_t blocks) {
    constexpr int SL = 64 / CL, kSlots = kWaves * SL, kSteps = kSlots * L;
    typedef Pack<T, V> P;
    __shared__ float2 totals[2][kWaves][CL][V];
    // neighbouring channel groups on one die: they share lines where rows are not aligned to them
    const int64_t chunk = (blocks + 7) / 8, id = (int64_t)(blockIdx.x & 7) * chunk + (blockIdx.x >> 3);
    if (id >= blocks) return;
    const int group = (int)(id % groups), b = (int)(id / groups % s.batch), part = (int)(id / groups / s.batch);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, cl = lane % CL, slot = lane / CL;
    const int segment = DIR == 0 ? part : seg.count - 1 - part;
    const int begin = segment * seg.steps, end = min(begin + seg.steps, s.time);
    const int n = steps_of(p.lengths, b, s.time);
    const int channel = (group * CL + cl) * V;
    const bool active = channel < s.channels;
    const int c = active ? channel : s.channels - V;  // loads stay inside the row
    const int64_t step = s.time_major ? s.batch : 1, row0 = s.time_major ? b : (int64_t)b * s.time;
    const int64_t state = (int64_t)b * s.channels + c, states = (int64_t)s.batch * s.channels;
    const int first = (wave * SL + slot) * L;  // of the thread's steps in a tile

    // step u of the walk is time t(u); beyond the segment's end it repeats the last
    auto time_of = [&](int u) { return DIR == 0 ? min(begin + u, end - 1) : max(end - 1 - u, begin); };
    auto load = [&](const void* base, int64_t ld, int u0, int shift, Steps<T, V, L>& to) {
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const int64_t row = row0 + max(time_of(u0 + first + i) - shift, 0) * step;
            to.v[i] = *(const P*)((const T*)base + row * ld + c);
        }
    };

    float carry[V], h0[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        carry[v] = MAPS ? 0.f : seg.carry ? seg.carry[segment * states + state + v] : p.init ? p.init[state + v] : 0.f;
        h0[v] = DIR == 1 && !MAPS && p.h0 ? p.h0[state + v] : 0.f;
    }
    float whole[V];  // MAPS: the product of the segment's a
#pragma unroll
    for (int v = 0; v < V; ++v) whole[v] = 1.f;

    constexpr bool kNeedX = DIR == 0 || (!MAPS && GATE == SEERA_GATE_SIGMOID), kNeedH = DIR == 1 && !MAPS;
    Steps<T, V, L> rx, rf, rd, rh, nx, nf, nd, nh;
    auto load_all = [&](int u0, Steps<T, V, L>& x, Steps<T, V, L>& f, Steps<T, V, L>& d, Steps<T, V, L>& h) {
        load(p.f, p.ldf, u0, 0, f);
        if (kNeedX) load(p.x, p.ldx, u0, 0, x);
        if (DIR == 1) load(p.dh, s.channels, u0, 0, d);
        if (kNeedH) load(p.h, s.channels, u0, 1, h);
    };
    const int length = end - begin;
    load_all(0, rx, rf, rd, rh);
    int parity = 0;
    for (int u0 = 0; u0 < length; u0 += kSteps, parity ^= 1) {
        if (u0 + kSteps < length) load_all(u0 + kSteps, nx, nf, nd, nh);
        float a[L][V], m[L][V];  // m: b, or dh
        float A[V], B[V];
#pragma unroll
        for (int v = 0; v < V; ++v) A[v] = 1.f, B[v] = 0.f;
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const int u = u0 + first + i;
            const bool live = u < length && (DIR == 0 ? begin + u : end - 1 - u) < n;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float rest;
                gates<GATE>(to_f32(rf.v[i].v[v]), a[i][v], rest);
                m[i][v] = DIR == 0 ? rest * to_f32(rx.v[i].v[v]) : to_f32(rd.v[i].v[v]);
                a[i][v] = live ? a[i][v] : 1.f;
                m[i][v] = live ? m[i][v] : 0.f;
                B[v] = DIR == 0 ? fmaf(a[i][v], B[v], m[i][v]) : a[i][v] * (m[i][v] + B[v]);
                A[v] *= a[i][v];
            }
        }
        // the composition of this slot and the wave's slots before it
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
        float mine[V];
#pragma unroll
        for (int v = 0; v < V; ++v) mine[v] = carry[v];
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float2 t = totals[parity][w][cl][v];
                carry[v] = fmaf(t.x, carry[v], t.y);
                if (MAPS) whole[v] *= t.x;
                if (w + 1 == wave) mine[v] = carry[v];
            }
        if (!MAPS) {
            float z[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                z[v] = mine[v];
                if (SL > 1) {
                    const float pa = __shfl_up(A[v], CL, 64), pb = __shfl_up(B[v], CL, 64);
                    if (slot > 0) z[v] = fmaf(pa, mine[v], pb);
                }
            }
#pragma unroll
            for (int i = 0; i < L; ++i) {
                const int u = u0 + first + i, t = time_of(u);
                const bool live = t < n;
                P o, o2;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if (DIR == 0) {
                        z[v] = fmaf(a[i][v], z[v], m[i][v]);
                        o.v[v] = from_f32<T>(live ? z[v] : 0.f);
                    } else {
                        const float g = m[i][v] + z[v];
                        z[v] = a[i][v] * g;
                        const float before = t > 0 ? to_f32(rh.v[i].v[v]) : h0[v];
                        float one = g, two = g * before;
                        if (GATE == SEERA_GATE_SIGMOID) {
                            // 1 - a again, from f: the difference would cancel for a near 1
                            float again, rest;
                            gates<GATE>(to_f32(rf.v[i].v[v]), again, rest);
                            one = g * rest;
                            two = one * (before - to_f32(rx.v[i].v[v])) * a[i][v];
                        }
                        o.v[v] = from_f32<T>(live ? one : 0.f);
                        o2.v[v] = from_f32<T>(live ? two : 0.f);
                    }
                }
                if (active && u < length) {
                    const int64_t row = row0 + t * step;
                    *(P*)((T*)p.out + row * p.ldo + c) = o;
                    if (DIR == 1) *(P*)((T*)p.out2 + row * p.ldo2 + c) = o2;
                }
            }
        }
        rx = nx, rf = nf, rd = nd, rh = nh;
    }
    if (!active || wave || slot) return;
    if (MAPS) {
#pragma unroll
        for (int v = 0; v < V; ++v) seg.maps[segment * states + state + v] = make_float2(whole[v], carry[v]);
    } else if (part == seg.count - 1 && p.last) {
#pragma unroll
        for (int v = 0; v < V; ++v) p.last[state + v] = carry[v];
    }
}

// The state before each segment, from the segments' maps in the order of the walk.
__global__ __launch_bounds__(256) void scan_carries(const float2* maps, const float* init, float* carry, int64_t states, int count, int reverse) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= states) return;
    float c = init ? init[i] : 0.f;
#pragma unroll 8
    for (int k = 0; k < count; ++k) {
        const int64_t at = (reverse ? count - 1 - k : k) * states + i;
        carry[at] = c;
        if (k + 1 < count) {
            const float2 m = maps[at];
            c = fmaf(m.x, c, m.y);
        }
    }
}

template <class T, int V, int CL, int L, int GATE, int DIR>
int launch_tiles(const ScanShape& s, const ScanPtrs& p, hipStream_t st) {
    constexpr int kSteps = kWaves * (64 / CL) * L;
    const int groups = (s.channels + CL * V - 1) / (CL * V);
    const int64_t chains = (int64_t)groups * s.batch, states = (int64_t)s.batch * s.channels;
    Segments seg{1, s.time, nullptr, nullptr};
    const int tiles = (s.time + kSteps - 1) / kSteps;
    // few chains: split time, so that every compute unit has a block
    const int64_t want = (2 * device_cus() + chains - 1) / chains;
    if (chains < device_cus() / 2 && tiles > 2) {
        const int per = (int)std::max<int64_t>(2, (tiles + want - 1) / want);
        seg.count = (tiles + per - 1) / per;
        seg.steps = per * kSteps;
    }
    const int64_t blocks = chains * seg.count;
    if (blocks > kMaxGridX / 2) return fail(SEERA_ERR_INVALID_ARGUMENT, "gated_scan: batch * channels is too large");
    auto grid = [](int64_t n) { return dim3((unsigned)((n + 7) / 8 * 8)); };
    if (seg.count > 1) {
        void* ws = nullptr;
        const size_t n = (size_t)seg.count * states;
        SEERA_TRY(workspace(n * (sizeof(float2) + sizeof(float)), &ws, st));
        seg.maps = (float2*)ws;
        float* carry = (float*)(seg.maps + n);
        hipLaunchKernelGGL((scan_tiles<T, V, CL, L, GATE, DIR, true>), grid(blocks - chains), dim3(kTile), 0, st, p, s, seg, groups, blocks - chains);
        SEERA_HIP_TRY(hipGetLastError());
        hipLaunchKernelGGL(scan_carries, dim3((unsigned)((states + 255) / 256)), dim3(256), 0, st, seg.maps, p.init, carry, states, seg.count, DIR);
        SEERA_HIP_TRY(hipGetLastError());
        seg.carry = carry;
    }
    hipLaunchKernelGGL((scan_tiles<T, V, CL, L, GATE, DIR, false>), grid(blocks), dim3(kTile), 0, st, p, s, seg, groups, blocks);
    SEERA_HIP_TRY(hipGetLastError());
    return SEERA_OK;
}

// Whether V values of T may be moved as one: sizes, row distances and addresses.
template <class T, int V>
bool packs(const ScanShape& s, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> lds) {
    if (s.channels % V) return false;
    for (int64_t ld : lds)
        if (ld % V) return false;
    for (const void* p : ptrs)
        if (!aligned_to(p, sizeof(T) * V)) return false;
    return true;
}

// Up to this many steps a chain is walked by one thread, without tiles.
constexpr int kFewSteps = 16;

template <class T, int V, int GATE>
int fwd_v(const ScanShape& s, const ScanFwd& a, hipStream_t st) {
    if (s.time <= kFewSteps) {
        const int64_t items = (int64_t)s.batch * (s.channels / V), blocks = (items + 255) / 256;
        if (blocks > kMaxGridX) return fail(SEERA_ERR_INVALID_ARGUMENT, "gated_scan: batch * channels is too large");
        hipLaunchKernelGGL((scan_fwd_steps<T, V, GATE>), dim3((unsigned)blocks), dim3(256), 0, st, a, s, items);
        SEERA_HIP_TRY(hipGetLastError());
        return SEERA_OK;
    }
    const ScanPtrs p{a.x, a.f, nullptr, nullptr, a.h, nullptr, nullptr, a.h0, a.hT, a.lengths, a.ldx, a.ldf, s.channels, 0};
    return launch_tiles<T, V, 128 / (V * (int)sizeof(T)), 16, GATE, 0>(s, p, st);
}

template <class T, int V, int GATE>
int bwd_v(const ScanShape& s, const ScanBwd& a, hipStream_t st) {
    if (s.time <= kFewSteps) {
        const int64_t items = (int64_t)s.batch * (s.channels / V), blocks = (items + 255) / 256;
        if (blocks > kMaxGridX) return fail(SEERA_ERR_INVALID_ARGUMENT, "gated_scan: batch * channels is too large");
        hipLaunchKernelGGL((scan_bwd_steps<T, V, GATE>), dim3((unsigned)blocks), dim3(256), 0, st, a, s, items);
        SEERA_HIP_TRY(hipGetLastError());
        return SEERA_OK;
    }
    const ScanPtrs p{a.x, a.f, a.h, a.dh, a.dx, a.df, a.h0, a.dhT, a.dh0, a.lengths, a.ldx, a.ldf, a.lddx, a.lddf};
    return launch_tiles<T, V, 128 / (V * (int)sizeof(T)), 8, GATE, 1>(s, p, st);
}

// Two 16-bit values a lane where everything is aligned to pairs, one otherwise.
template <class T>
int fwd_t(const ScanShape& s, const ScanFwd& a, hipStream_t st) {
    const bool linear = s.gate == SEERA_GATE_LINEAR;
    if (sizeof(T) == 2 && packs<T, 2>(s, {a.x, a.f, a.h}, {a.ldx, a.ldf}))
        return linear ? fwd_v<T, sizeof(T) == 2 ? 2 : 1, SEERA_GATE_LINEAR>(s, a, st) : fwd_v<T, sizeof(T) == 2 ? 2 : 1, SEERA_GATE_SIGMOID>(s, a, st);
    return linear ? fwd_v<T, 1, SEERA_GATE_LINEAR>(s, a, st) : fwd_v<T, 1, SEERA_GATE_SIGMOID>(s, a, st);
}
template <class T>
int bwd_t(const ScanShape& s, const ScanBwd& a, hipStream_t st) {
    const bool linear = s.gate == SEERA_GATE_LINEAR;
    if (sizeof(T) == 2 && packs<T, 2>(s, {linear ? a.f : a.x, a.f, a.h, a.dh, a.dx, a.df}, {linear ? a.ldf : a.ldx, a.ldf, a.lddx, a.lddf}))
        return linear ? bwd_v<T, sizeof(T) == 2 ? 2 : 1, SEERA_GATE_LINEAR>(s, a, st) : bwd_v<T, sizeof(T) == 2 ? 2 : 1, SEERA_GATE_SIGMOID>(s, a, st);
    return linear ? bwd_v<T, 1, SEERA_GATE_LINEAR>(s, a, st) : bwd_v<T, 1, SEERA_GATE_SIGMOID>(s, a, st);
}

}  // namespace

int gated_scan_fwd(const ScanShape& s, const ScanFwd& a, hipStream_t st) {
    return s.dtype == SEERA_DTYPE_F32 ? fwd_t<float>(s, a, st) : s.dtype == SEERA_DTYPE_F16 ? fwd_t<f16_t>(s, a, st) : fwd_t<bf16_t>(s, a, st);
}
int gated_scan_bwd(const ScanShape& s, const ScanBwd& a, hipStream_t st) {
    return s.dtype == SEERA_DTYPE_F32 ? bwd_t<float>(s, a, st) : s.dtype == SEERA_DTYPE_F16 ? bwd_t<f16_t>(s, a, st) : bwd_t<bf16_t>(s, a, st);
}

}  // namespace seera
