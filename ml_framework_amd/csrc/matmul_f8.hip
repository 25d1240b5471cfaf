// matmul_f8.hip -- products of operands in 8 bits (seera_hip_matmul_f8):
//
//   C[m][n] = sum_b sa[m][b] sw[n / 128][b] sum_{k in block b} A[m][k] W[n][k] + bias[n]
//
// A block of 128 along K begins from zero; its sums are multiplied by the two scales
// and added to fp32 sums. W is the matrix instruction's first operand, so a lane holds
// four values of n of one m: the scale product is one number a lane, and a row of C
// is stored four values at a time. Both operands are permuted alike along K (lanes
// 16 g .. 16 g + 15 hold its 16-byte pieces g and g + 4), which changes no sum of products.
//
// 16-bit results take v_mfma_f32_16x16x128_f8f6f4. It cuts each product below 2^-13 of
// the largest of its group of 8 along K (measured; towards zero), and adds in fp32 from there:
// 1.4e-5 of the result, where rounding it to 16 bits is 1.7e-3 or 2e-4. An fp32 result
// is held to fp32's roundings: its codes are widened to fp16, which holds each of them,
// and multiplied by v_mfma_f32_16x16x32_f16, at half the rate (2e-8 of the result).
#include <algorithm>
#include <type_traits>

#include "f8.h"
#include "half_tile.h"
#include "inference.h"
#include "io_types.h"
#include "runtime.h"

namespace seera {
namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));

// 128 codes along K of 16 rows, and products of two of them.
struct Codes8 {  // as they are
    intx8 v;
    __device__ __forceinline__ Codes8() {}
    __device__ __forceinline__ explicit Codes8(intx8 c) : v(c) {}
};
struct Codes16 {  // as fp16
    half8 v[4];
    __device__ __forceinline__ Codes16() {}
    __device__ __forceinline__ explicit Codes16(intx8 c) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], 1.f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], 1.f, true);
            v[i / 2][i % 2 * 4] = (half_t)lo[0], v[i / 2][i % 2 * 4 + 1] = (half_t)lo[1];
            v[i / 2][i % 2 * 4 + 2] = (half_t)hi[0], v[i / 2][i % 2 * 4 + 3] = (half_t)hi[1];
        }
    }
};
template <class T>
using Codes = std::conditional_t<sizeof(T) == 4, Codes16, Codes8>;
__device__ __forceinline__ floatx4 products(const Codes8& w, const Codes8& a) {
    const floatx4 zero = {0.f, 0.f, 0.f, 0.f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, a.v, zero, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ floatx4 products(const Codes16& w, const Codes16& a) {
    floatx4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) p = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.v[i], a.v[i], p, 0, 0, 0);
    return p;
}
__device__ __forceinline__ intx8 fragment(const uint8_t* row, int lane) {
    const intx4 lo = *(const intx4*)(row + 16 * (lane >> 4)), hi = *(const intx4*)(row + 64 + 16 * (lane >> 4));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Four values of a row of C from column n on.
template <class T>
__device__ __forceinline__ void store4(const MatmulF8& g, int m, int n, floatx4 v) {
    T* c = (T*)g.c + (int64_t)m * g.ldc + n;
    if (n + 4 <= g.n) {
        Pack<T, 4> p;
        if (g.bias)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += g.bias[n + i];
#pragma unroll
        for (int i = 0; i < 4; ++i) p.v[i] = from_f32<T>(v[i]);
        __builtin_memcpy(c, &p, sizeof(p));  // at any alignment of T, as one access
        return;
    }
    for (int i = 0; n + i < g.n; ++i) c[i] = from_f32<T>(v[i] + (g.bias ? g.bias[n + i] : 0.f));
}

// A tile of 16 MT x 16 NT, with the blocks along K dealt to the waves of a workgroup
// and their sums joined in the waves' order. Operands go from memory to registers.
template <class T, int MT, int NT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void matmul_f8_split(MatmulF8 g) {
    __shared__ floatx4 sums[WAVES][MT * NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles_n = (g.n + 16 * NT - 1) / (16 * NT);
    const int n0 = (int)(blockIdx.x % tiles_n) * 16 * NT, m0 = (int)(blockIdx.x / tiles_n) * 16 * MT;
    const int64_t kp = (int64_t)g.blocks * kF8Block;
    const uint8_t* a[MT];
    const uint8_t* w[NT];
    const float* sa[MT];
    // rows past the end repeat the last one: their results are not stored
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t m = min(m0 + 16 * i + (lane & 15), g.m - 1);
        a[i] = g.a + m * kp;
        sa[i] = g.a_scales + m * g.blocks;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) w[j] = g.w + min(n0 + 16 * j + (lane & 15), g.n - 1) * kp;
    const float* sw = g.w_scales + (int64_t)(n0 / kF8Block) * g.blocks;
    floatx4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    for (int b = wave; b < g.blocks; b += WAVES) {
        Codes<T> fa[MT], fw[NT];
        float s[MT];
#pragma unroll
        for (int j = 0; j < NT; ++j) fw[j] = Codes<T>(fragment(w[j] + (int64_t)b * kF8Block, lane));
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            fa[i] = Codes<T>(fragment(a[i] + (int64_t)b * kF8Block, lane));
            s[i] = sa[i][b] * sw[b];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const floatx4 p = products(fw[j], fa[i]);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(p[e], s[i], acc[i][j][e]);
            }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) sums[wave][i * NT + j][lane] = acc[i][j];
    __syncthreads();
    for (int t = wave; t < MT * NT; t += WAVES) {
        floatx4 v = sums[0][t][lane];
#pragma unroll
        for (int k = 1; k < WAVES; ++k) v += sums[k][t][lane];
        const int m = m0 + 16 * (t / NT) + (lane & 15), n = n0 + 16 * (t % NT) + 4 * (lane >> 4);
        if (m < g.m) store4<T>(g, m, n, v);
    }
}

template <class T, int MT, int NT, int WAVES>
int launch_split(const MatmulF8& g, hipStream_t st) {
    const int64_t tiles = (int64_t)((g.n + 16 * NT - 1) / (16 * NT)) * ((g.m + 16 * MT - 1) / (16 * MT));
    if (tiles * 64 * WAVES >= kMaxThreads) return fail(SEERA_ERR_INVALID_ARGUMENT, "matmul_f8: the product is too large");
    hipLaunchKernelGGL((matmul_f8_split<T, MT, NT, WAVES>), dim3((uint32_t)tiles), dim3(64 * WAVES), 0, st, g);
    SEERA_HIP_TRY(hipGetLastError());
    return SEERA_OK;
}

template <class T>
int launch_t(const MatmulF8& g, hipStream_t st) {
    if (g.m <= 16) return launch_split<T, 1, 1, 8>(g, st);
    return launch_split<T, 4, 2, 4>(g, st);
}

}  // namespace

int matmul_f8(const MatmulF8& g, hipStream_t st) {
    return g.dtype == SEERA_DTYPE_F32 ? launch_t<float>(g, st) : g.dtype == SEERA_DTYPE_F16 ? launch_t<f16_t>(g, st) : launch_t<bf16_t>(g, st);
}

}  // namespace seera
