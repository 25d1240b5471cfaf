// norm_rows.h -- what the kernels of the block norm share (block_norm.hip,
// block_norm_f8.hip): sums over a row's threads, a gate's activation, and rows
// moved 16 bytes a lane at any alignment and length.
#pragma once

#include <type_traits>

#include "io_types.h"
#include "sequence.h"
#include "sequence_rules.h"

namespace seera {

// The sum over a wave's 64 lanes, in every lane. The lanes are added in a fixed
// order: along rows of 16, then over the four rows.
__device__ __forceinline__ float wave_sum(float v) {
    auto add = [&](auto ctrl, auto rows) {
        v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
    };
    add(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});  // row_shr:1
    add(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});  // row_shr:2
    add(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});  // row_shr:4
    add(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});  // row_shr:8
    add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // row_bcast:15
    add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});  // row_bcast:31
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// The sum over the NT threads of a row, with one barrier: `halves` is the block's
// own, kept over all of its sums.
template <int NT>
__device__ __forceinline__ float row_sum(float v, float* part, Halves& halves) {
    v = wave_sum(v);
    if (NT == 64) return v;
    constexpr int W = NT / 64;
    float* at = part + halves.next() * W;
    if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) s += at[w];
    return s;
}

// The activation of a gate.
__device__ __forceinline__ float act_of(int act, float g) {
    const float q = __builtin_amdgcn_rcpf(1.f + __expf(-g));
    return act == SEERA_GATE_ACT_SILU ? g * q : q;
}
// 16 bytes of a row, moved as one access at any alignment of T (the hardware
// takes unaligned addresses) and without a branch, so that nothing waits for a
// load before its values are used. The pack at column `want` lies at `c`: moved
// back where it would pass the row's end, so that some of its values belong to
// the pack before it, or all of them. Values lo <= i < hi are its own: only they
// enter sums and are stored. With CUT false (cols is a multiple of N) a pack is
// whole or has no value.
template <class T>
struct Wide {
    static constexpr int N = 16 / sizeof(T);
    T v[N];
};
template <int N, bool CUT>
struct Place {
    int c, lo, hi;
    __device__ Place(int want, int cols) {
        c = max(min(want, cols - N), 0);
        lo = CUT ? min(want - c, N) : want < cols ? 0 : N;
        hi = CUT ? min(N, cols - c) : N;
    }
    __device__ bool whole() const { return lo == 0 && (!CUT || hi == N); }
    __device__ bool own(int i) const { return CUT ? i >= lo && i < hi : lo == 0; }
    // sum + a b, of value i: not added where it is not the pack's own (a factor of 0 would
    // make an infinity there a NaN)
    __device__ float add(int i, float a, float b, float sum) const { return !CUT || own(i) ? fmaf(a, b, sum) : sum; }
    // a pack's part of a sum
    __device__ float part(float x) const { return CUT || lo == 0 ? x : 0.f; }
};
template <class T, bool CUT>
__device__ __forceinline__ void load_wide(Wide<T>& to, const T* row, const Place<Wide<T>::N, CUT>& at, int cols) {
    typedef uint32_t Bits __attribute__((ext_vector_type(4), aligned(2), may_alias));
    if (CUT && cols < Wide<T>::N) {
#pragma unroll
        for (int i = 0; i < Wide<T>::N; ++i) to.v[i] = i < at.hi ? row[i] : from_f32<T>(0.f);
        return;
    }
    // past the cache where rows share no line of it: forward 16384 x 2048 69 -> 64 us (and 60
    // with the stores); with cut rows the neighbour's line is lost, 8192 x 1501 30 -> 34
    const Bits w = CUT ? *(const Bits*)(row + at.c) : __builtin_nontemporal_load((const Bits*)(row + at.c));
    __builtin_memcpy(&to, &w, 16);
}
template <class T, bool CUT>
__device__ __forceinline__ void store_wide(T* row, const Place<Wide<T>::N, CUT>& at, const Wide<T>& from) {
    typedef uint32_t Bits __attribute__((ext_vector_type(4), aligned(2), may_alias));
    if (at.whole()) {
        Bits w;
        __builtin_memcpy(&w, &from, 16);
        __builtin_nontemporal_store(w, (Bits*)(row + at.c));
    } else if (CUT) {
#pragma unroll
        for (int i = 0; i < Wide<T>::N; ++i)
            if (at.own(i)) row[at.c + i] = from.v[i];
    }
}
// The N fp32 weights of a pack.
template <int N, bool CUT>
__device__ __forceinline__ void load_weights(float (&to)[N], const float* w, const Place<N, CUT>& at, int cols) {
    if (CUT && cols < N) {
#pragma unroll
        for (int i = 0; i < N; ++i) to[i] = i < at.hi ? w[i] : 0.f;
        return;
    }
    __builtin_memcpy(to, w + at.c, sizeof(to));
}

// The first half of the block norm's forward, for row `row` in the registers of NT
// threads (`tid` of them), K wide packs each: y becomes r' = r + rms(y) w1 act(g) s
// as it is kept, and is stored to r_out. The thread's part of the sum of its squares.
template <class T, int K, int NT, bool CUT>
__device__ __forceinline__ float residual_row(const NormFwd& p, const NormShape& s, int tid, int64_t row, float* part, Halves& halves, Wide<T> (&y)[K]) {
    constexpr int N = Wide<T>::N;
    typedef Place<N, CUT> At;
    const T* yr = (const T*)p.y + row * p.ldy;
    const T* gr = (const T*)p.g + row * p.ldg;
    const T* rr = (const T*)p.r + row * s.cols;
    auto place = [&](int k) { return At((k * NT + tid) * N, s.cols); };
    Wide<T> g[K], r[K];
#pragma unroll
    for (int k = 0; k < K; ++k) load_wide(y[k], yr, place(k), s.cols);
    if (p.g)
#pragma unroll
        for (int k = 0; k < K; ++k) load_wide(g[k], gr, place(k), s.cols);
    if (p.r)
#pragma unroll
        for (int k = 0; k < K; ++k) load_wide(r[k], rr, place(k), s.cols);
    float rstd1 = 1.f;
    if (p.w1) {
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const At at = place(k);
            float own = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) own = at.add(i, to_f32(y[k].v[i]), to_f32(y[k].v[i]), own);
            sum += at.part(own);
        }
        rstd1 = rsqrtf(row_sum<NT>(sum, part, halves) / s.cols + p.eps);
        if (p.rstd1 && tid == 0) p.rstd1[row] = rstd1;
    }
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const At at = place(k);
        float u[N], w[N];
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = to_f32(y[k].v[i]);
        if (p.w1) {
            load_weights(w, p.w1, at, s.cols);
#pragma unroll
            for (int i = 0; i < N; ++i) u[i] = u[i] * rstd1 * w[i];
        }
        if (p.g)
#pragma unroll
            for (int i = 0; i < N; ++i) u[i] *= act_of(s.act, to_f32(g[k].v[i]));
        if (p.s) {
            load_weights(w, p.s, at, s.cols);
#pragma unroll
            for (int i = 0; i < N; ++i) u[i] *= w[i];
        }
        if (p.r)
#pragma unroll
            for (int i = 0; i < N; ++i) u[i] += to_f32(r[k].v[i]);
        float own = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            y[k].v[i] = from_f32<T>(u[i]);  // as it is kept
            own = at.add(i, to_f32(y[k].v[i]), to_f32(y[k].v[i]), own);
        }
        sum += at.part(own);
    }
    // a row's packs may reach into each other: all of it is read before any is written
    if (CUT && NT > 64 && !p.w1) __syncthreads();
    if (p.r_out)
#pragma unroll
        for (int k = 0; k < K; ++k) store_wide((T*)p.r_out + row * s.cols, place(k), y[k]);
    return sum;
}

}  // namespace seera
