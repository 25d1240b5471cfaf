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
        const float q = __builtin_amdgcn_rcpf(1.f + e);
        const float s = e * q;
        a = f >= 0.f ? q : s;
        rest = f >= 0.f ? s : q;
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

template <class T, int V, int GATE>
int fwd_v(const ScanShape& s, const ScanFwd& a, hipStream_t st) {
    const int64_t items = (int64_t)s.batch * (s.channels / V), blocks = (items + 255) / 256;
    if (blocks > kMaxGridX) return fail(SEERA_ERR_INVALID_ARGUMENT, "gated_scan: batch * channels is too large");
    hipLaunchKernelGGL((scan_fwd_steps<T, V, GATE>), dim3((unsigned)blocks), dim3(256), 0, st, a, s, items);
    SEERA_HIP_TRY(hipGetLastError());
    return SEERA_OK;
}

template <class T, int V, int GATE>
int bwd_v(const ScanShape& s, const ScanBwd& a, hipStream_t st) {
    const int64_t items = (int64_t)s.batch * (s.channels / V), blocks = (items + 255) / 256;
    if (blocks > kMaxGridX) return fail(SEERA_ERR_INVALID_ARGUMENT, "gated_scan: batch * channels is too large");
    hipLaunchKernelGGL((scan_bwd_steps<T, V, GATE>), dim3((unsigned)blocks), dim3(256), 0, st, a, s, items);
    SEERA_HIP_TRY(hipGetLastError());
    return SEERA_OK;
}

template <class T>
int fwd_t(const ScanShape& s, const ScanFwd& a, hipStream_t st) {
    return s.gate == SEERA_GATE_LINEAR ? fwd_v<T, 1, SEERA_GATE_LINEAR>(s, a, st) : fwd_v<T, 1, SEERA_GATE_SIGMOID>(s, a, st);
}
template <class T>
int bwd_t(const ScanShape& s, const ScanBwd& a, hipStream_t st) {
    return s.gate == SEERA_GATE_LINEAR ? bwd_v<T, 1, SEERA_GATE_LINEAR>(s, a, st) : bwd_v<T, 1, SEERA_GATE_SIGMOID>(s, a, st);
}

}  // namespace

int gated_scan_fwd(const ScanShape& s, const ScanFwd& a, hipStream_t st) {
    return s.dtype == SEERA_DTYPE_F32 ? fwd_t<float>(s, a, st) : s.dtype == SEERA_DTYPE_F16 ? fwd_t<f16_t>(s, a, st) : fwd_t<bf16_t>(s, a, st);
}
int gated_scan_bwd(const ScanShape& s, const ScanBwd& a, hipStream_t st) {
    return s.dtype == SEERA_DTYPE_F32 ? bwd_t<float>(s, a, st) : s.dtype == SEERA_DTYPE_F16 ? bwd_t<f16_t>(s, a, st) : bwd_t<bf16_t>(s, a, st);
}

}  // namespace seera
