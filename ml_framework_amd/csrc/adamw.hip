// adamw.hip -- the AdamW step over many tensors, with moments in 32 bits or in
// 8-bit codes of which 128 share an exponent (seera_hip_adamw_step,
// seera_hip_adamw_state_values).
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

__device__ __forceinline__ float load_grad(const void* g, int dtype, int64_t i) {
    return dtype == SEERA_DTYPE_F32 ? ((const float*)g)[i] : dtype == SEERA_DTYPE_F16 ? to_f32(((const f16_t*)g)[i]) : to_f32(((const bf16_t*)g)[i]);
}

// One block of 128 threads for 128 values.
__global__ __launch_bounds__(kBlock) void adamw_block(seera_adamw_tensor t, AdamwStep s, float keep, uint32_t key) {
    __shared__ uint32_t most[4];
    const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    const bool in = i < t.count;
    const bool codes = t.state_bits == 8;
    float m = 0.f, v = 0.f;
    if (in) {
        float g = load_grad(t.grad, t.grad_dtype, i);
        if (s.grad_scale) g *= *s.grad_scale;
        if (codes) {
            const uint32_t cm = ((const uint8_t*)t.m)[i], cv = ((const uint8_t*)t.v)[i];
            m = decode(cm & 127, t.m_exp[blockIdx.x], 15);
            if (cm & 128) m = -m;
            v = decode(cv, t.v_exp[blockIdx.x], 31);
        } else {
            m = ((const float*)t.m)[i];
            v = ((const float*)t.v)[i];
        }
        m = m * s.beta1 + g * s.one_minus_beta1;
        v = v * s.beta2 + (g * g) * s.one_minus_beta2;
        float p = t.param[i];
        p = p * keep - s.step_size * m / (sqrtf(v) * s.inv_sqrt_corr2 + s.eps);
        t.param[i] = p;
        if (t.param16) {
            if (t.param16_dtype == SEERA_DTYPE_F16) ((f16_t*)t.param16)[i] = from_f32<f16_t>(p);
            else ((bf16_t*)t.param16)[i] = from_f32<bf16_t>(p);
        }
        if (!codes) {
            ((float*)t.m)[i] = m;
            ((float*)t.v)[i] = v;
        }
    }
    if (!codes) return;
    uint32_t am = __float_as_uint(fabsf(m)), av = __float_as_uint(v) & 0x7fffffffu;
    for (int o = 32; o > 0; o >>= 1) {
        am = max(am, (uint32_t)__shfl_xor((int)am, o, 64));
        av = max(av, (uint32_t)__shfl_xor((int)av, o, 64));
    }
    if ((threadIdx.x & 63) == 0) {
        most[threadIdx.x >> 6] = am;
        most[2 + (threadIdx.x >> 6)] = av;
    }
    __syncthreads();
    const uint32_t em = shared_exponent(max(most[0], most[1])), ev = shared_exponent(max(most[2], most[3]));
    if (in) {
        const uint32_t random = mix((uint32_t)i * 0x9E3779B9u + key);
        ((uint8_t*)t.m)[i] = (uint8_t)(min(encode(fabsf(m), em, 15, random & 0xffffu), 127u) | (m < 0.f ? 128u : 0u));
        uint32_t cv = min(encode(v, ev, 31, random >> 16), 255u);
        if (v > 0.f && cv == 0) cv = 1;
        ((uint8_t*)t.v)[i] = (uint8_t)cv;
    }
    if (threadIdx.x == 0) {
        t.m_exp[blockIdx.x] = (uint8_t)em;
        t.v_exp[blockIdx.x] = (uint8_t)ev;
    }
}

__global__ __launch_bounds__(kBlock) void state_values(seera_adamw_tensor t, float* m_out, float* v_out) {
    const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (i >= t.count) return;
    if (t.state_bits == 32) {
        if (m_out) m_out[i] = ((const float*)t.m)[i];
        if (v_out) v_out[i] = ((const float*)t.v)[i];
        return;
    }
    if (m_out) {
        const uint32_t c = ((const uint8_t*)t.m)[i];
        const float a = decode(c & 127, t.m_exp[blockIdx.x], 15);
        m_out[i] = c & 128 ? -a : a;
    }
    if (v_out) v_out[i] = decode(((const uint8_t*)t.v)[i], t.v_exp[blockIdx.x], 31);
}

int blocks_of(int64_t count, unsigned* out) {
    const int64_t blocks = (count + kBlock - 1) / kBlock;
    if (blocks > kMaxGridX) return fail(SEERA_ERR_INVALID_ARGUMENT, "adamw: a tensor is too large");
    *out = (unsigned)blocks;
    return SEERA_OK;
}

}  // namespace

int adamw_step(const seera_adamw_tensor* tensors, int n, const AdamwStep& step, hipStream_t st) {
    for (int i = 0; i < n; ++i) {
        unsigned blocks = 0;
        SEERA_TRY(blocks_of(tensors[i].count, &blocks));
        if (!blocks) continue;
        hipLaunchKernelGGL(adamw_block, dim3(blocks), dim3(kBlock), 0, st, tensors[i], step, (float)(1.0 - step.lr * tensors[i].weight_decay),
                           mix((uint32_t)i * 0x9E3779B9u + step.seed));
        SEERA_HIP_TRY(hipGetLastError());
    }
    return SEERA_OK;
}

int adamw_state_values(const seera_adamw_tensor* tensors, int n, float* const* m_values, float* const* v_values, hipStream_t st) {
    for (int i = 0; i < n; ++i) {
        unsigned blocks = 0;
        SEERA_TRY(blocks_of(tensors[i].count, &blocks));
        if (!blocks || (!m_values[i] && !v_values[i])) continue;
        hipLaunchKernelGGL(state_values, dim3(blocks), dim3(kBlock), 0, st, tensors[i], m_values[i], v_values[i]);
        SEERA_HIP_TRY(hipGetLastError());
    }
    return SEERA_OK;
}

}  // namespace seera
