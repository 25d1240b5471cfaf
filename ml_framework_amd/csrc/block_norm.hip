// block_norm.hip -- the norms after and before a block with its gate, residual
// scale and residual, forward and backward (seera_hip_block_norm_fwd / _bwd).
#include <algorithm>

#include "io_types.h"
#include "runtime.h"
#include "sequence.h"

namespace seera {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float block_sum(float v, float* part) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) s += part[w];
    return s;
}

__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.f + __expf(-g)); }
__device__ __forceinline__ float act_of(int act, float g) { return act == SEERA_GATE_ACT_SILU ? g * sigmoid(g) : sigmoid(g); }
__device__ __forceinline__ float slope_of(int act, float g) {
    const float q = sigmoid(g), d = q * (1.f - q);
    return act == SEERA_GATE_ACT_SILU ? q + g * d : d;
}

template <class T>
__global__ __launch_bounds__(kThreads) void norm_fwd_row(NormFwd p, NormShape s) {
    extern __shared__ float row_r[];
    __shared__ float part[kThreads / 64];
    const int64_t row = blockIdx.x;
    const T* y = (const T*)p.y + row * p.ldy;
    const T* g = (const T*)p.g + row * p.ldg;
    const T* r = (const T*)p.r + row * s.cols;
    float rstd1 = 1.f;
    if (p.w1) {
        float sum = 0.f;
        for (int c = threadIdx.x; c < s.cols; c += kThreads) sum += to_f32(y[c]) * to_f32(y[c]);
        rstd1 = rsqrtf(block_sum(sum, part) / s.cols + p.eps);
        if (p.rstd1 && threadIdx.x == 0) p.rstd1[row] = rstd1;
    }
    float sum = 0.f;
    for (int c = threadIdx.x; c < s.cols; c += kThreads) {
        float u = to_f32(y[c]);
        if (p.w1) u = u * rstd1 * p.w1[c];
        if (p.g) u *= act_of(s.act, to_f32(g[c]));
        if (p.s) u *= p.s[c];
        if (p.r) u += to_f32(r[c]);
        const T kept = from_f32<T>(u);
        if (p.r_out) ((T*)p.r_out)[row * s.cols + c] = kept;
        u = to_f32(kept);
        row_r[c] = u;
        sum += u * u;
    }
    if (!p.w2) return;
    const float rstd2 = rsqrtf(block_sum(sum, part) / s.cols + p.eps);
    if (p.rstd2 && threadIdx.x == 0) p.rstd2[row] = rstd2;
    for (int c = threadIdx.x; c < s.cols; c += kThreads)
        ((T*)p.n_out)[row * s.cols + c] = from_f32<T>(row_r[c] * rstd2 * p.w2[c]);
}

// partial: [gridDim.x][3][cols] sums over the block's rows of dw1, ds, dw2.
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
            const float yv = inner ? to_f32(y[c]) : 0.f, gv = p.g ? to_f32(g[c]) : 0.f;
            const float hat = yv * rstd1, z = p.w1 ? hat * p.w1[c] : yv, act = p.g ? act_of(s.act, gv) : 1.f;
            if (p.s) {
                sums[s.cols + c] += d * z * act;
                d *= p.s[c];
            }
            if (p.g) {
                ((T*)p.dg)[row * p.lddg + c] = from_f32<T>(d * z * slope_of(s.act, gv));
                d *= act;
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

// out[k][c] = sum over blocks, in order, of partial[block][k][c].
__global__ __launch_bounds__(kThreads) void norm_bwd_sums(const float* partial, int blocks, int cols, float* dw1, float* ds, float* dw2) {
    const int i = blockIdx.x * kThreads + threadIdx.x;
    if (i >= 3 * cols) return;
    float* out = i < cols ? dw1 : i < 2 * cols ? ds : dw2;
    if (!out) return;
    float sum = 0.f;
    for (int b = 0; b < blocks; ++b) sum += partial[(int64_t)b * 3 * cols + i];
    out[i % cols] = sum;
}

template <class T>
int fwd_t(const NormShape& s, const NormFwd& a, hipStream_t st) {
    hipLaunchKernelGGL((norm_fwd_row<T>), dim3(s.rows), dim3(kThreads), s.cols * sizeof(float), st, a, s);
    SEERA_HIP_TRY(hipGetLastError());
    return SEERA_OK;
}

template <class T>
int bwd_t(const NormShape& s, const NormBwd& a, hipStream_t st) {
    const int blocks = std::min(s.rows, 1024);
    void* ws = nullptr;
    SEERA_TRY(workspace((size_t)std::max(blocks, 1) * 3 * s.cols * sizeof(float), &ws, st));
    if (blocks) {
        hipLaunchKernelGGL((norm_bwd_rows<T>), dim3(blocks), dim3(kThreads), s.cols * sizeof(float), st, a, s, (float*)ws);
        SEERA_HIP_TRY(hipGetLastError());
    }
    hipLaunchKernelGGL(norm_bwd_sums, dim3((3 * s.cols + kThreads - 1) / kThreads), dim3(kThreads), 0, st, (const float*)ws, blocks, s.cols,
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
