// f8.h -- values in 8 bits: e4m3 codes (sign, 4 bits of exponent, 3 of mantissa;
// largest 448, smallest 2^-9, no infinity) with an fp32 scale that 128 values of a
// row, or 128 x 128 of a weight matrix, share. Rows of codes are padded with zeros
// to a multiple of 128.
//
// scale = max|v| / 448, code = v / scale rounded to nearest even. A block of zeros
// has scale 0 (so has one whose scale is below fp32's smallest value), a block
// that holds an infinity or NaN scale NaN.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace seera {

constexpr int kF8Block = 128;
constexpr float kF8Largest = 448.f;

__host__ __device__ constexpr int64_t f8_padded(int64_t k) { return (k + kF8Block - 1) / kF8Block * kF8Block; }

// A block's scale, from the largest of its values' magnitudes as bits (bits: the
// integers' order is the floats', with infinity and NaN above all others).
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct F8Scale {
    float scale, up, divisor, inverse;
    __device__ explicit F8Scale(uint32_t largest) {
        const bool finite = largest < 0x7f800000u;
        scale = finite ? __uint_as_float(largest) / kF8Largest : __uint_as_float(0x7fc00000u);
        // tiny scales are lifted out of the range where their inverse overflows; where the scale
        // is NaN all factors are 0, so that finite values (a row's padding) have code 0
        up = !finite ? 0.f : scale < 0x1p-60f ? 0x1p64f : 1.f;
        divisor = finite ? scale * up : 0.f;
        inverse = scale > 0.f ? 1.f / divisor : 0.f;
    }
    // v / scale, rounded correctly (Markstein 1990: a quotient from a correctly
    // rounded reciprocal, corrected by its remainder): ties between codes are common
    // in 16-bit values and fall as the division has them
    __device__ __forceinline__ float quotient(float v) const {
        const float x = v * up, q = x * inverse;
        // (its sum of zeros is +0; a scale that fp32's denormals rounded down leaves quotients above 448)
        return copysignf(fminf(fabsf(fmaf(fmaf(-q, divisor, x), inverse, q)), kF8Largest), v);
    }
};

// Codes of four quotients.
__device__ __forceinline__ uint32_t f8_codes(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

}  // namespace seera
