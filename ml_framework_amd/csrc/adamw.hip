// adamw.hip -- the AdamW step over many tensors, with moments in 32 bits or in
// 8-bit codes of which 128 share an exponent (seera_hip_adamw_step,
// seera_hip_adamw_state_values).
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
//
// Bytes bound: 28 a value with fp32 states and gradients, 16 with 8-bit states,
// bf16 gradients and a bf16 copy. 97 tensors of 97.6 M values: 501 us (5.5 TB/s; a
// large copy makes 5.35); with 8 bits, and the values read out (10 bytes), 472 us.
//
// Codes. v moves by a thousandth of itself in a step and a code's place is an
// eighth: rounded to nearest, v would never fall (a run on a noisy quadratic left
// it at a quarter of its value). So a value is rounded up or down with the
// remainder as probability, by bits of a hash, which leaves the mean right where
// each step has a seed of its own. And the shared exponent is a power of two: a
// scale that followed the largest value exactly would move every code off its place
// in every step, and round it again.
#include <algorithm>

#include "io_types.h"
#include "runtime.h"
#include "sequence.h"

// The moments are rounded to codes at places that depend on every bit, and a
// code is compared with that of another implementation of the same formulas:
// no multiply and add is contracted here.
#pragma clang fp contract(off)

namespace seera {
namespace {

constexpr int kBlock = 128;  // codes that share an exponent

// A 32-bit mix of the bits of x: two rounds of multiply and shift.
__host__ __device__ __forceinline__ uint32_t mix(uint32_t x) {
    x ^= x >> 16;
    x *= 0x6A09E667u;
    x ^= x >> 15;
    x *= 0xBB67AE85u;
    return x ^ (x >> 16);
}

// A code's value: 3 bits of mantissa below a field that stands for 2^(E - 127)
// at `top`; `code` without its sign.
__device__ __forceinline__ float decode(uint32_t code, uint32_t e, int top) {
    const float v = ldexpf(__uint_as_float(code << 20), (int)e - top);
    return e == 255 ? __uint_as_float(0x7fc00000u) : v;
}
// The code of a >= 0, rounded by 16 random bits (up to the top field's 1.875).
__device__ __forceinline__ uint32_t encode(float a, uint32_t e, int top, uint32_t random16) {
    return (__float_as_uint(ldexpf(a, top - (int)e)) + (random16 << 4)) >> 20;
}
// The exponent whose 1.875-fold reaches the block's largest value (its bits).
__device__ __forceinline__ uint32_t shared_exponent(uint32_t largest) { return largest >= 0x7f800000u ? 255u : (largest + 0x0fffffu) >> 23; }

// What a launch works on: up to kMost tensors (3.9 of the 4 KB that arguments may take) in the kernel's arguments, so that
// a step needs no copy to the device and may be captured in a graph. Thread block
// b works on values [(b - first) * kChunk, ...) of the last tensor with first <= b:
// 2048 values (0.54 M values 7.5 us, in shares of 4096 8.7; 97.6 M with 8 bits 475, 491).
constexpr int kMost = 48, kThreads = 256, kChunk = kThreads * 8;
struct Slot {
    float* param;      // adamw_values: where m's values go
    const void* grad;  // adamw_values: where v's values go
    void *m, *v;
    uint8_t *m_exp, *v_exp;
    void* param16;
    int64_t count;
    float keep;        // 1 - lr * weight_decay
    uint32_t key;      // of the rounding's random bits
};
struct Batch {
    Slot slot[kMost];
    unsigned first[kMost];
    uint8_t bits[kMost], grad_dtype[kMost], copy[kMost];
    int count;
};

// The block's slot, by one comparison in each of 48 lanes.
__device__ __forceinline__ int slot_of(const Batch& b) {
    const int lane = threadIdx.x & 63;
    const bool begun = lane < b.count && b.first[min(lane, kMost - 1)] <= blockIdx.x;
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(begun)) - 1);
}

// N consecutive values; the cut ones at the tensor's end one by one. Whole ones are
// one access at any alignment of T (the hardware takes unaligned addresses).
// STREAM: past the cache, for what this step alone touches: 97.6 M values in 519 us,
// 498 with the stores so and 470 with the loads too. Codes are loaded through it (eight
// bytes a lane share lines: 33.5 M values 153 us, 160 past it).
template <bool STREAM, class T, int N>
__device__ __forceinline__ void load_some(T (&to)[N], const void* from, int64_t i, int live) {
    const T* p = (const T*)from + i;
    if (live == N) {
        if constexpr (STREAM) {
            typedef uint32_t Bits __attribute__((ext_vector_type(sizeof(to) / 4), aligned(2), may_alias));
            const Bits w = __builtin_nontemporal_load((const Bits*)p);
            __builtin_memcpy(to, &w, sizeof(to));
        } else {
            __builtin_memcpy(to, p, sizeof(to));
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) to[k] = k < live ? p[k] : (T)0;
    }
}
template <class T, int N>
__device__ __forceinline__ void store_some(void* to, int64_t i, const T (&from)[N], int live) {
    T* p = (T*)to + i;
    if (live == N) {
        if constexpr (sizeof(from) >= 8) {
            typedef uint32_t Bits __attribute__((ext_vector_type(sizeof(from) / 4), aligned(1), may_alias));
            Bits w;
            __builtin_memcpy(&w, from, sizeof(from));
            __builtin_nontemporal_store(w, (Bits*)p);
        } else {
            __builtin_memcpy(p, from, sizeof(from));
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k < live) p[k] = from[k];
    }
}
template <class T, bool STREAM, int N>
__device__ __forceinline__ void load_as_f32(float (&to)[N], const void* from, int64_t i, int live) {
    T raw[N];
    load_some<STREAM>(raw, from, i, live);
#pragma unroll
    for (int k = 0; k < N; ++k) to[k] = to_f32(raw[k]);
}
template <bool STREAM, int N>
__device__ __forceinline__ void load_grads(float (&to)[N], const void* from, int dtype, int64_t i, int live) {
    if (dtype == SEERA_DTYPE_F32) load_as_f32<float, STREAM>(to, from, i, live);
    else if (dtype == SEERA_DTYPE_F16) load_as_f32<f16_t, STREAM>(to, from, i, live);
    else load_as_f32<bf16_t, STREAM>(to, from, i, live);
}
template <class T, int N>
__device__ __forceinline__ void store_rounded(void* to, int64_t i, const float (&from)[N], int live) {
    T raw[N];
#pragma unroll
    for (int k = 0; k < N; ++k) raw[k] = from_f32<T>(from[k]);
    store_some(to, i, raw, live);
}

// The largest of the 16 lanes of a row, in each of them.
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));  // row_ror:8
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
}

// The square root, rounded correctly from v = 2^-101 on: the hardware's is off by a
// unit at most, and the residuals of its two neighbours say which is nearest (all
// 2^24 values of [1, 4) checked). 0, infinity and NaN pass through; below 2^-101 the
// residuals lose bits, and the hardware takes denormals for 0.
__device__ __forceinline__ float root_of(float v) {
    const float s = __builtin_amdgcn_sqrtf(v);
    const float down = __uint_as_float(__float_as_uint(s) - 1), up = __uint_as_float(__float_as_uint(s) + 1);
    const float below = fmaf(-down, s, v), above = fmaf(-up, s, v);
    const float r = below <= 0.f ? down : s;
    return above > 0.f ? up : r;
}
// a / b, rounded correctly for a b whose reciprocal is normal and an a of 0 or from
// 2^-101 on: with a correctly rounded reciprocal (one Newton step on the hardware's;
// all 2^23 fractions checked) one step on the quotient rounds it correctly (Markstein
// 1990).
__device__ __forceinline__ float quotient_of(float a, float b) {
    float r = __builtin_amdgcn_rcpf(b);
    r = fmaf(fmaf(-b, r, 1.f), r, r);
    const float q = a * r;
    return __builtin_amdgcn_div_fixupf(fmaf(fmaf(-b, q, a), r, q), b, a);
}

// N values of the step: the moments and the parameter, each operation rounded
// correctly. PLAIN: for every v and eps; else root_of and quotient_of, for the 8-bit
// states, whose instructions count (97.6 M values with their reading out 472 us,
// PLAIN 484; the hardware's root and reciprocal alone, off by a unit, 465).
template <bool PLAIN, int N>
__device__ __forceinline__ void update(const AdamwStep& s, float keep, float scale, const float (&g)[N], float (&m)[N], float (&v)[N], float (&p)[N]) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const float gk = g[k] * scale;
        m[k] = m[k] * s.beta1 + gk * s.one_minus_beta1;
        v[k] = v[k] * s.beta2 + (gk * gk) * s.one_minus_beta2;
        const float size = s.step_size * m[k];
        if (PLAIN) p[k] = p[k] * keep - size / (sqrtf(v[k]) * s.inv_sqrt_corr2 + s.eps);
        else p[k] = p[k] * keep - quotient_of(size, root_of(v[k]) * s.inv_sqrt_corr2 + s.eps);
    }
}

template <int N>
__device__ __forceinline__ void store_params(const Slot& t, int copy, int64_t i, const float (&p)[N], int live) {
    store_some(t.param, i, p, live);
    if (copy == SEERA_DTYPE_F16) store_rounded<f16_t>(t.param16, i, p, live);
    else if (copy == SEERA_DTYPE_BF16) store_rounded<bf16_t>(t.param16, i, p, live);
}

// PLAIN8: update's PLAIN for the 8-bit states.
template <bool PLAIN8>
__global__ __launch_bounds__(kThreads) void adamw_many(Batch b, AdamwStep s) {
    const int at = slot_of(b);
    const Slot t = b.slot[at];
    const int bits = b.bits[at], dtype = b.grad_dtype[at], copy = b.copy[at];
    const int64_t begin = (int64_t)(blockIdx.x - b.first[at]) * kChunk;
    const int64_t end = min(begin + kChunk, t.count);
    const float scale = s.grad_scale ? *s.grad_scale : 1.f;
    if (bits == 32) {
        constexpr int N = 4;
#pragma unroll 2
        for (int64_t i = begin + threadIdx.x * N; i < end; i += kThreads * N) {
            const int live = (int)min((int64_t)N, t.count - i);
            float g[N], m[N], v[N], p[N];
            load_grads<true>(g, t.grad, dtype, i, live);
            load_some<true>(m, t.m, i, live);
            load_some<true>(v, t.v, i, live);
            load_some<true>(p, t.param, i, live);
            update<true>(s, t.keep, scale, g, m, v, p);
            store_some(t.m, i, m, live);
            store_some(t.v, i, v, live);
            store_params(t, copy, i, p, live);
        }
        return;
    }
    // 8 values a lane: the 16 lanes of a row hold the 128 that share an exponent
    constexpr int N = 8;
    for (int64_t i = begin + threadIdx.x * N; i < (end + kBlock - 1) / kBlock * kBlock; i += kThreads * N) {
        const int live = (int)max((int64_t)0, min((int64_t)N, t.count - i));
        const int64_t block = i / kBlock;
        float g[N], m[N], v[N], p[N];
        uint8_t cm[N], cv[N];
        load_grads<false>(g, t.grad, dtype, i, live);
        load_some<false>(cm, t.m, i, live);
        load_some<false>(cv, t.v, i, live);
        load_some<false>(p, t.param, i, live);
        uint32_t em = t.m_exp[block], ev = t.v_exp[block];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            m[k] = decode(cm[k] & 127, em, 15);
            if (cm[k] & 128) m[k] = -m[k];
            v[k] = decode(cv[k], ev, 31);
        }
        update<PLAIN8>(s, t.keep, scale, g, m, v, p);
        store_params(t, copy, i, p, live);
        uint32_t am = 0, av = 0;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (k < live) {
                am = max(am, __float_as_uint(m[k]) & 0x7fffffffu);
                av = max(av, __float_as_uint(v[k]) & 0x7fffffffu);
            }
        }
        em = shared_exponent(row_max(am));
        ev = shared_exponent(row_max(av));
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const uint32_t random = mix((uint32_t)(i + k) * 0x9E3779B9u + t.key);
            cm[k] = (uint8_t)(min(encode(fabsf(m[k]), em, 15, random & 0xffffu), 127u) | (m[k] < 0.f ? 128u : 0u));
            const uint32_t c = min(encode(v[k], ev, 31, random >> 16), 255u);
            cv[k] = (uint8_t)(v[k] > 0.f ? max(c, 1u) : c);
        }
        store_some(t.m, i, cm, live);
        store_some(t.v, i, cv, live);
        if ((threadIdx.x & 15) == 0) {
            t.m_exp[block] = (uint8_t)em;
            t.v_exp[block] = (uint8_t)ev;
        }
    }
}

__global__ __launch_bounds__(kThreads) void adamw_values(Batch b) {
    const int at = slot_of(b);
    const Slot t = b.slot[at];
    const int64_t begin = (int64_t)(blockIdx.x - b.first[at]) * kChunk;
    const int64_t end = min(begin + kChunk, t.count);
    float *m_out = t.param, *v_out = (float*)t.grad;
    if (b.bits[at] == 32) {
        constexpr int N = 4;
        for (int64_t i = begin + threadIdx.x * N; i < end; i += kThreads * N) {
            const int live = (int)min((int64_t)N, t.count - i);
            float x[N];
            if (m_out) load_some<false>(x, t.m, i, live), store_some(m_out, i, x, live);
            if (v_out) load_some<false>(x, t.v, i, live), store_some(v_out, i, x, live);
        }
        return;
    }
    // four values a lane and store, so that a wave writes 1 KB in one piece; two of
    // them in flight
    constexpr int N = 4, K = 2;
    for (int64_t i0 = begin + threadIdx.x * N; i0 < end; i0 += kThreads * N * K) {
        uint8_t cm[K][N], cv[K][N];
        uint32_t em[K], ev[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int64_t i = i0 + k * kThreads * N;
            if (i >= end) break;
            const int live = (int)min((int64_t)N, t.count - i);
            load_some<false>(cm[k], t.m, i, live);
            load_some<false>(cv[k], t.v, i, live);
            em[k] = t.m_exp[i / kBlock];
            ev[k] = t.v_exp[i / kBlock];
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int64_t i = i0 + k * kThreads * N;
            if (i >= end) break;
            const int live = (int)min((int64_t)N, t.count - i);
            float x[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                x[j] = decode(cm[k][j] & 127, em[k], 15);
                if (cm[k][j] & 128) x[j] = -x[j];
            }
            if (m_out) store_some(m_out, i, x, live);
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = decode(cv[k][j], ev[k], 31);
            if (v_out) store_some(v_out, i, x, live);
        }
    }
}

// Launches `kernel` over all tensors, kMost at a time (fewer where the grid of
// those would pass its limit). Nothing is launched where a tensor is refused.
template <class Fill, class Launch>
int batches(const seera_adamw_tensor* tensors, int n, Fill&& fill, Launch&& launch) {
    constexpr int64_t kMostBlocks = kMaxThreads / kThreads - 1;
    for (int i = 0; i < n; ++i)
        if (tensors[i].count > kMostBlocks * kChunk) return fail(SEERA_ERR_INVALID_ARGUMENT, "adamw: tensor %d is too large", i);
    Batch b;
    int64_t blocks = 0;
    b.count = 0;
    for (int i = 0; i < n; ++i) {
        const seera_adamw_tensor& t = tensors[i];
        if (t.count == 0) continue;
        const int64_t more = (t.count + kChunk - 1) / kChunk;
        if (b.count == kMost || blocks + more > kMostBlocks) {
            launch(b, (unsigned)blocks);
            SEERA_HIP_TRY(hipGetLastError());
            b.count = 0;
            blocks = 0;
        }
        Slot& s = b.slot[b.count];
        s.m = t.m, s.v = t.v, s.m_exp = t.m_exp, s.v_exp = t.v_exp, s.count = t.count;
        fill(s, t, i);
        b.first[b.count] = (unsigned)blocks;
        b.bits[b.count] = (uint8_t)t.state_bits;
        b.grad_dtype[b.count] = (uint8_t)t.grad_dtype;
        b.copy[b.count] = t.param16 ? (uint8_t)t.param16_dtype : 0;
        ++b.count;
        blocks += more;
    }
    if (b.count == 0) return SEERA_OK;
    launch(b, (unsigned)blocks);
    SEERA_HIP_TRY(hipGetLastError());
    return SEERA_OK;
}

}  // namespace

int adamw_step(const seera_adamw_tensor* tensors, int n, const AdamwStep& step, hipStream_t st) {
    return batches(
        tensors, n,
        [&](Slot& s, const seera_adamw_tensor& t, int i) {
            s.param = t.param, s.grad = t.grad, s.param16 = t.param16;
            s.keep = (float)(1.0 - step.lr * t.weight_decay);
            s.key = mix((uint32_t)i * 0x9E3779B9u + step.seed);
        },
        [&](const Batch& b, unsigned blocks) {
            // root_of takes denormals (roots below 1.1e-19) for 0: rounded away where they are added
            // to an eps of 2^25 times that
            if (step.eps >= 3.7e-12f * step.inv_sqrt_corr2) hipLaunchKernelGGL(adamw_many<false>, dim3(blocks), dim3(kThreads), 0, st, b, step);
            else hipLaunchKernelGGL(adamw_many<true>, dim3(blocks), dim3(kThreads), 0, st, b, step);
        });
}

int adamw_state_values(const seera_adamw_tensor* tensors, int n, float* const* m_values, float* const* v_values, hipStream_t st) {
    return batches(
        tensors, n, [&](Slot& s, const seera_adamw_tensor&, int i) { s.param = m_values[i], s.grad = v_values[i]; },
        [&](const Batch& b, unsigned blocks) { hipLaunchKernelGGL(adamw_values, dim3(blocks), dim3(kThreads), 0, st, b); });
}

}  // namespace seera
