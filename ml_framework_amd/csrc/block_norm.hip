// block_norm.hip -- the norms after and before a block with its gate, residual
// scale and residual, forward and backward (seera_hip_block_norm_fwd / _bwd).
//
//   z = rms(y) w1, u = z act(g) s, r' = r + u, n = rms(r') w2
//   dr = dr' + rstd2 (q - r^ mean(q r^)),  q = dn w2, r^ = r' rstd2
//   dz = dr act(g) s, dg = dr s z act'(g), ds = sum dr z act(g), dw2 = sum dn r^
//   dy = rstd1 (k - y^ mean(k y^)),  k = dz w1, y^ = y rstd1, dw1 = sum dz y^
//
// Each value of a row is needed again after a sum over the row, so a row stays in
// registers: the forward moves 5 values an element, the backward 8, once each, and
// bytes bound both. 16384 x 2048 bf16: forward 60 us (5.6 TB/s; a large copy makes
// 5.35), backward 99 us (5.4). n is the norm of r' as it is stored: then the
// backward, which has only that, is exact. Not so in the backward of rows of more
// than 8192 columns (norm_bwd_rows), which reads rows twice and keeps its sums over
// rows in memory: 2048 x 16384 bf16 1.7 ms.
#include <algorithm>
#include <type_traits>

#include "io_types.h"
#include "runtime.h"
#include "sequence.h"
#include "sequence_rules.h"

namespace seera {
namespace {

constexpr int kThreads = 256;

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

__device__ __forceinline__ float block_sum(float v, float* part) {
    __syncthreads();
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) s += part[w];
    return s;
}

// The activation of a gate.
__device__ __forceinline__ float act_of(int act, float g) {
    const float q = __builtin_amdgcn_rcpf(1.f + __expf(-g));
    return act == SEERA_GATE_ACT_SILU ? g * q : q;
}
// The activation and its slope. The sigmoid's slope is the product of its two sides
// q and e^-g q: 1 - q has no digit left where q is near 1. (Below g = -88 that is
// infinity times 0, and the side is 1.)
struct Act {
    float of, slope;
};
__device__ __forceinline__ Act act_and_slope(int act, float g) {
    const float e = __expf(-g), q = __builtin_amdgcn_rcpf(1.f + e), d = q * fminf(e * q, 1.f);
    return act == SEERA_GATE_ACT_SILU ? Act{g * q, fmaf(g, d, q)} : Act{q, d};
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

// A row in the registers of NT threads, K wide packs each; ROWS rows a block.
template <class T, int K, int NT, int ROWS, bool CUT>
__global__ __launch_bounds__(NT * ROWS) void norm_fwd_rows(NormFwd p, NormShape s) {
    constexpr int N = Wide<T>::N;
    typedef Place<N, CUT> At;
    __shared__ float part[2 * (NT / 64) * ROWS];
    Halves halves;
    const int tid = threadIdx.x % NT;
    const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / NT;
    if (ROWS > 1 && row >= s.rows) return;  // whole waves: such rows take no barrier
    const T* yr = (const T*)p.y + row * p.ldy;
    const T* gr = (const T*)p.g + row * p.ldg;
    const T* rr = (const T*)p.r + row * s.cols;
    auto place = [&](int k) { return At((k * NT + tid) * N, s.cols); };
    Wide<T> y[K], g[K], r[K];
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
    if (!p.w2) return;
    const float rstd2 = rsqrtf(row_sum<NT>(sum, part, halves) / s.cols + p.eps);
    if (p.rstd2 && tid == 0) p.rstd2[row] = rstd2;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const At at = place(k);
        float w[N];
        load_weights(w, p.w2, at, s.cols);
#pragma unroll
        for (int i = 0; i < N; ++i) y[k].v[i] = from_f32<T>(to_f32(y[k].v[i]) * rstd2 * w[i]);
        store_wide((T*)p.n_out + row * s.cols, at, y[k]);
    }
}

// The backward of rows that lie in the registers of NT threads, K wide packs
// each. A block takes rows `blockIdx.x + k gridDim.x`, with NEXT the next row's
// loads in flight while the present one is computed, and keeps its sums over
// rows of dw1, ds, dw2 in registers: partial[block][3][cols].
template <class T, int K>
struct NormRow {
    Wide<T> y[K], g[K], r[K], d[K], n[K];
    float rstd1, rstd2;
};
template <class T, int K, int NT, bool NEXT, bool HOLD, bool CUT>
__global__ __launch_bounds__(NT) void norm_bwd_regs(NormBwd p, NormShape s, float* partial) {
    constexpr int N = Wide<T>::N;
    typedef Place<N, CUT> At;
    __shared__ float part[2 * (NT / 64)];
    Halves halves;  // over the rows: a row may have one sum or two
    const bool inner = p.w1 || p.g || p.s;
    float h1[K][N], hs[K][N], h2[K][N], sum1[K][N], sums[K][N], sum2[K][N];
    auto place = [&](int k) { return At((int)(k * NT + threadIdx.x) * N, s.cols); };
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < N; ++i) sum1[k][i] = sums[k][i] = sum2[k][i] = 0.f;
    }
    // the weights: held in registers, or read again for each row
    auto weights = [&](float (&to)[K][N], const float* w) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int i = 0; i < N; ++i) to[k][i] = 1.f;
            At at = place(k);
            if (!HOLD) asm volatile("" : "+v"(at.c));  // an address of this row's own: the loads stay in the loop
            if (w) load_weights(to[k], w, at, s.cols);
        }
    };
    if (HOLD) weights(h1, p.w1), weights(hs, p.s), weights(h2, p.w2);
    auto load = [&](NormRow<T, K>& to, int64_t row) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            At c = place(k);
            if (!HOLD) asm volatile("" : "+v"(c.c));  // as for the weights: 5 K addresses held over the rows would spill
            if (inner) load_wide(to.y[k], (const T*)p.y + row * p.ldy, c, s.cols);
            if (p.g) load_wide(to.g[k], (const T*)p.g + row * p.ldg, c, s.cols);
            if (p.w2) {
                load_wide(to.r[k], (const T*)p.r_out + row * s.cols, c, s.cols);
                load_wide(to.n[k], (const T*)p.dn + row * s.cols, c, s.cols);
            }
            if (p.dr_out) load_wide(to.d[k], (const T*)p.dr_out + row * s.cols, c, s.cols);
        }
        to.rstd1 = p.w1 ? p.rstd1[row] : 1.f;
        if (p.w2) to.rstd2 = p.rstd2[row];
    };
    const float inv = 1.f / s.cols;
    NormRow<T, K> now, next;
    int64_t row = blockIdx.x;
    if (NEXT) load(now, row);
    for (; row < s.rows; row += gridDim.x) {
        if (!NEXT) load(now, row);
        else if (row + gridDim.x < s.rows) load(next, row + gridDim.x);
        float d[K][N];
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < N; ++i) d[k][i] = p.dr_out ? to_f32(now.d[k].v[i]) : 0.f;
        if (p.w2) {
            if (!HOLD) weights(h2, p.w2);
            float dot = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const At at = place(k);
                float own = 0.f;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float hat = to_f32(now.r[k].v[i]) * now.rstd2, dn = to_f32(now.n[k].v[i]);
                    sum2[k][i] = fmaf(dn, hat, sum2[k][i]);
                    own = at.add(i, dn * h2[k][i], hat, own);
                }
                dot += at.part(own);
            }
            dot = row_sum<NT>(dot, part, halves) * inv;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float hat = to_f32(now.r[k].v[i]) * now.rstd2;
                    d[k][i] = fmaf(now.rstd2, to_f32(now.n[k].v[i]) * h2[k][i] - hat * dot, d[k][i]);
                }
        }
        if (!HOLD) weights(h1, p.w1), weights(hs, p.s);
        // a row's packs may reach into each other: all of it is read before any is written
        if (CUT && NT > 64 && !p.w2) __syncthreads();
        float dot = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            Wide<T> out;
            if (p.dr) {
#pragma unroll
                for (int i = 0; i < N; ++i) out.v[i] = from_f32<T>(d[k][i]);
                store_wide((T*)p.dr + row * s.cols, place(k), out);
            }
            if (p.g) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const Act act = act_and_slope(s.act, to_f32(now.g[k].v[i]));
                    const float z = to_f32(now.y[k].v[i]) * now.rstd1 * h1[k][i];
                    sums[k][i] = fmaf(d[k][i] * z, act.of, sums[k][i]);
                    d[k][i] *= hs[k][i];
                    out.v[i] = from_f32<T>(d[k][i] * z * act.slope);
                    d[k][i] *= act.of;
                }
                store_wide((T*)p.dg + row * p.lddg, place(k), out);
            } else if (p.s) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    sums[k][i] = fmaf(d[k][i], to_f32(now.y[k].v[i]) * now.rstd1 * h1[k][i], sums[k][i]);
                    d[k][i] *= hs[k][i];
                }
            }
            if (p.w1) {
                const At at = place(k);
                float own = 0.f;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float hat = to_f32(now.y[k].v[i]) * now.rstd1;
                    sum1[k][i] = fmaf(d[k][i], hat, sum1[k][i]);
                    d[k][i] *= h1[k][i];
                    own = at.add(i, d[k][i], hat, own);
                }
                dot += at.part(own);
            }
        }
        if (p.w1) {
            dot = row_sum<NT>(dot, part, halves) * inv;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < N; ++i) d[k][i] = now.rstd1 * (d[k][i] - to_f32(now.y[k].v[i]) * now.rstd1 * dot);
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            Wide<T> out;
#pragma unroll
            for (int i = 0; i < N; ++i) out.v[i] = from_f32<T>(d[k][i]);
            store_wide((T*)p.dy + row * p.lddy, place(k), out);
        }
        if (NEXT) now = next;
    }
    float* to = partial + (int64_t)blockIdx.x * 3 * s.cols;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const At at = place(k);
            const int c = at.c + i;
            if (!at.own(i)) continue;
            if (p.w1) to[c] = sum1[k][i];
            if (p.s) to[s.cols + c] = sums[k][i];
            if (p.w2) to[2 * s.cols + c] = sum2[k][i];
        }
}

// The backward of wider rows: partial[gridDim.x][3][cols] holds the sums over the
// block's rows of dw1, ds, dw2, read and written for each of them.
template <class T>
__global__ __launch_bounds__(kThreads) void norm_bwd_rows(NormBwd p, NormShape s, float* partial) {
    extern __shared__ float row_d[];
    __shared__ float part[kThreads / 64];
    float* sums = partial + (int64_t)blockIdx.x * 3 * s.cols;
    for (int c = threadIdx.x; c < 3 * s.cols; c += kThreads) sums[c] = 0.f;
    __syncthreads();
    for (int64_t row = blockIdx.x; row < s.rows; row += gridDim.x) {
        const T* y = (const T*)p.y + row * p.ldy;
        const T* g = (const T*)p.g + row * p.ldg;
        const int64_t at = row * s.cols;
        const float rstd1 = p.w1 ? p.rstd1[row] : 1.f, rstd2 = p.w2 ? p.rstd2[row] : 0.f;
        float mean = 0.f;
        if (p.w2) {
            for (int c = threadIdx.x; c < s.cols; c += kThreads) {
                const float hat = to_f32(((const T*)p.r_out)[at + c]) * rstd2, dn = to_f32(((const T*)p.dn)[at + c]);
                mean += dn * p.w2[c] * hat;
                sums[2 * s.cols + c] += dn * hat;
            }
            mean = block_sum(mean, part) / s.cols;
        }
        float mean1 = 0.f;
        for (int c = threadIdx.x; c < s.cols; c += kThreads) {
            float d = p.dr_out ? to_f32(((const T*)p.dr_out)[at + c]) : 0.f;
            if (p.w2) {
                const float hat = to_f32(((const T*)p.r_out)[at + c]) * rstd2;
                d += rstd2 * (to_f32(((const T*)p.dn)[at + c]) * p.w2[c] - hat * mean);
            }
            if (p.dr) ((T*)p.dr)[at + c] = from_f32<T>(d);
            const bool inner = p.w1 || p.g || p.s;
            const float yv = inner ? to_f32(y[c]) : 0.f;
            const float hat = yv * rstd1, z = p.w1 ? hat * p.w1[c] : yv;
            const Act act = p.g ? act_and_slope(s.act, to_f32(g[c])) : Act{1.f, 0.f};
            if (p.s) {
                sums[s.cols + c] += d * z * act.of;
                d *= p.s[c];
            }
            if (p.g) {
                ((T*)p.dg)[row * p.lddg + c] = from_f32<T>(d * z * act.slope);
                d *= act.of;
            }
            if (p.w1) {
                sums[c] += d * hat;
                d *= p.w1[c];
                mean1 += d * hat;
                row_d[c] = d;
            } else {
                ((T*)p.dy)[row * p.lddy + c] = from_f32<T>(d);
            }
        }
        if (p.w1) {
            mean1 = block_sum(mean1, part) / s.cols;
            for (int c = threadIdx.x; c < s.cols; c += kThreads)
                ((T*)p.dy)[row * p.lddy + c] = from_f32<T>(rstd1 * (row_d[c] - to_f32(y[c]) * rstd1 * mean1));
        }
    }
}

// out[k][c] = sum over blocks of partial[block][k][c], in a fixed order: 16
// interleaved chains, then their sum. 32 columns a block.
constexpr int kSumCols = 32, kSumRows = 16, kFlight = 16;
__global__ __launch_bounds__(kSumCols * kSumRows) void norm_bwd_sums(const float* partial, int blocks, int cols, float* dw1, float* ds, float* dw2) {
    __shared__ float part[kSumRows][kSumCols + 1];
    const int k = blockIdx.y, lane = threadIdx.x % kSumCols, chain = threadIdx.x / kSumCols, c = blockIdx.x * kSumCols + lane;
    float* out = k == 0 ? dw1 : k == 1 ? ds : dw2;
    if (!out) return;
    float sum = 0.f;
    if (c < cols) {
        // past the last block the last one again, not added
        for (int b = chain; b < blocks; b += kSumRows * kFlight) {
            float x[kFlight];
#pragma unroll
            for (int i = 0; i < kFlight; ++i) x[i] = partial[((int64_t)min(b + i * kSumRows, blocks - 1) * 3 + k) * cols + c];
#pragma unroll
            for (int i = 0; i < kFlight; ++i) sum += b + i * kSumRows < blocks ? x[i] : 0.f;
        }
    }
    part[chain][lane] = sum;
    __syncthreads();
    if (chain || c >= cols) return;
#pragma unroll
    for (int i = 1; i < kSumRows; ++i) sum += part[i][lane];
    out[c] = sum;
}

template <class T, int K, int NT, int ROWS>
int fwd_launch(NormShape s, NormFwd a, hipStream_t st) {
    // as many rows at once as a launch may have threads for
    constexpr int kMost = (int)std::min<int64_t>(kMaxThreads / NT / 2, 1 << 30);
    for (int left = s.rows; left > 0; left -= kMost) {
        s.rows = std::min(left, kMost);
        const dim3 grid((s.rows + ROWS - 1) / ROWS), block(NT * ROWS);
        if (s.cols % Wide<T>::N) hipLaunchKernelGGL((norm_fwd_rows<T, K, NT, ROWS, true>), grid, block, 0, st, a, s);
        else hipLaunchKernelGGL((norm_fwd_rows<T, K, NT, ROWS, false>), grid, block, 0, st, a, s);
        SEERA_HIP_TRY(hipGetLastError());
        auto on = [&](auto& p, int64_t ld) {
            if (p) p = (std::decay_t<decltype(p)>)((char*)p + s.rows * ld);
        };
        on(a.y, a.ldy * sizeof(T)), on(a.g, a.ldg * sizeof(T));
        on(a.r, s.cols * sizeof(T)), on(a.r_out, s.cols * sizeof(T)), on(a.n_out, s.cols * sizeof(T));
        on(a.rstd1, sizeof(float)), on(a.rstd2, sizeof(float));
    }
    return SEERA_OK;
}

// A row in one wave up to 32 (16-bit) or 16 (fp32) values a lane: no barrier, and
// many rows in flight (16 x 1024 bf16 in 4 us); wider ones in 256 or 1024 threads,
// two to four packs each: 4096 x 8192 fp16 63 us, 5.4 TB/s.
template <class T>
int fwd_t(const NormShape& s, const NormFwd& a, hipStream_t st) {
    constexpr int N = Wide<T>::N;
    const int packs = (s.cols + N - 1) / N;
    if (packs <= 64) return fwd_launch<T, 1, 64, 4>(s, a, st);
    if (packs <= 128) return fwd_launch<T, 2, 64, 4>(s, a, st);
    if (packs <= 256) return fwd_launch<T, 4, 64, 4>(s, a, st);
    if (packs <= 512) return fwd_launch<T, 2, 256, 1>(s, a, st);
    if (packs <= 1024) return fwd_launch<T, 4, 256, 1>(s, a, st);
    if (packs <= 2048) return fwd_launch<T, 2, 1024, 1>(s, a, st);
    if constexpr (N == 4) return fwd_launch<T, 4, 1024, 1>(s, a, st);
    return SEERA_OK;  // 16384 columns of 16 bits are 2048 packs
}

template <class T, int K, int NT, bool NEXT, bool HOLD>
void bwd_launch(const NormShape& s, const NormBwd& a, int blocks, float* to, hipStream_t st) {
    if (s.cols % Wide<T>::N) hipLaunchKernelGGL((norm_bwd_regs<T, K, NT, NEXT, HOLD, true>), dim3(blocks), dim3(NT), 0, st, a, s, to);
    else hipLaunchKernelGGL((norm_bwd_regs<T, K, NT, NEXT, HOLD, false>), dim3(blocks), dim3(NT), 0, st, a, s, to);
}

// Rows of more than 1024 packs: fp32 ones up to 8192 columns still fit.
template <class T>
void bwd_wide(const NormShape& s, const NormBwd& a, int blocks, float* to, hipStream_t st) {
    if constexpr (sizeof(T) == 4)
        if (s.cols <= 8192) return bwd_launch<T, 4, 512, false, false>(s, a, blocks, to, st);
    hipLaunchKernelGGL((norm_bwd_rows<T>), dim3(blocks), dim3(kThreads), s.cols * sizeof(float), st, a, s, to);
}

template <class T>
int bwd_t(const NormShape& s, const NormBwd& a, hipStream_t st) {
    constexpr int N = Wide<T>::N;
    const int packs = (s.cols + N - 1) / N;
    const int threads = packs <= 64 ? 64 : packs <= 128 ? 128 : packs <= 512 ? 256 : 512;
    // 512 threads a compute unit (16384 x 2048 100 us; 256: 140, 768: 113, 1024: 122, whose
    // partial sums cost more), and four rows a block before there are that many: 500 x 2048
    // 14.5 us, with one row a block 21.8
    const int64_t cus = device_cus(), most = cus * (512 / threads);
    const int blocks = (int)(s.rows <= cus ? s.rows : std::min(most, std::max<int64_t>(cus, s.rows / 4)));
    void* ws = nullptr;
    SEERA_TRY(workspace((size_t)std::max(blocks, 1) * 3 * s.cols * sizeof(float), &ws, st));
    if (blocks) {
        float* to = (float*)ws;
        if (packs <= 64) bwd_launch<T, 1, 64, true, true>(s, a, blocks, to, st);
        else if (packs <= 128) bwd_launch<T, 1, 128, true, true>(s, a, blocks, to, st);
        else if (packs <= 256) bwd_launch<T, 1, 256, true, true>(s, a, blocks, to, st);
        // two packs a thread and no next row: two blocks a compute unit, that wait at their
        // barriers in turn (4096 x 4096 bf16 68 us; one pack, 512 threads and the next row 72)
        else if (packs <= 512) bwd_launch<T, 2, 256, false, true>(s, a, blocks, to, st);
        else if (packs <= 1024) bwd_launch<T, 2, 512, N == 4, false>(s, a, blocks, to, st);
        else bwd_wide<T>(s, a, blocks, to, st);
        SEERA_HIP_TRY(hipGetLastError());
    }
    if (!a.w1 && !a.s && !a.w2) return SEERA_OK;
    hipLaunchKernelGGL(norm_bwd_sums, dim3((s.cols + kSumCols - 1) / kSumCols, 3), dim3(kSumCols * kSumRows), 0, st, (const float*)ws, blocks, s.cols,
                       a.w1 ? a.dw1 : nullptr, a.s ? a.ds : nullptr, a.w2 ? a.dw2 : nullptr);
    SEERA_HIP_TRY(hipGetLastError());
    return SEERA_OK;
}

}  // namespace

int block_norm_fwd(const NormShape& s, const NormFwd& a, hipStream_t st) {
    return s.dtype == SEERA_DTYPE_F32 ? fwd_t<float>(s, a, st) : s.dtype == SEERA_DTYPE_F16 ? fwd_t<f16_t>(s, a, st) : fwd_t<bf16_t>(s, a, st);
}
int block_norm_bwd(const NormShape& s, const NormBwd& a, hipStream_t st) {
    return s.dtype == SEERA_DTYPE_F32 ? bwd_t<float>(s, a, st) : s.dtype == SEERA_DTYPE_F16 ? bwd_t<f16_t>(s, a, st) : bwd_t<bf16_t>(s, a, st);
}

}  // namespace seera
