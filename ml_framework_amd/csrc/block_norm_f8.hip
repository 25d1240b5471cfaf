// block_norm_f8.hip -- the block norm's forward with its output in 8 bits
// (seera_hip_block_norm_fwd_f8): the operand of the next product.
//
//   r' = r + rms(y) w1 act(g) s,  n = rms(r') w2,  code = n / scale for each 128 columns
//
// As in norm_fwd_rows a row stays in registers. 128 columns are 16 lanes (32 with
// fp32) next to each other, so a block's largest value is found within them and
// nothing is moved but the inputs, r' and a byte a value.
#include <algorithm>

#include "f8.h"
#include "inference.h"
#include "norm_rows.h"
#include "runtime.h"

namespace seera {
namespace {

// The largest of LANES (16 or 32) lanes next to each other, in each of them.
template <int LANES>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    auto turn = [&](auto ctrl) { v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xf, 0xf, true)); };
    turn(std::integral_constant<int, 0x128>{});  // row_ror:8
    turn(std::integral_constant<int, 0x124>{});
    turn(std::integral_constant<int, 0x122>{});
    turn(std::integral_constant<int, 0x121>{});
    if constexpr (LANES == 32) v = max(v, (uint32_t)__builtin_amdgcn_ds_swizzle((int)v, 0x401f));  // lane ^ 16
    return v;
}

template <class T, int K, int NT, int ROWS, bool CUT>
__global__ __launch_bounds__(NT * ROWS) void norm_fwd_f8_rows(NormFwd p, NormShape s, uint8_t* codes, float* scales) {
    constexpr int N = Wide<T>::N, LANES = kF8Block / N;
    typedef Place<N, CUT> At;
    __shared__ float part[2 * (NT / 64) * ROWS];
    Halves halves;
    const int tid = threadIdx.x % NT;
    const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / NT;
    if (ROWS > 1 && row >= s.rows) return;  // whole waves: such rows take no barrier
    auto place = [&](int k) { return At((k * NT + tid) * N, s.cols); };
    Wide<T> y[K];
    const float sum = residual_row<T, K, NT, CUT>(p, s, tid, row, part, halves, y);
    const float rstd2 = p.w2 ? rsqrtf(row_sum<NT>(sum, part, halves) / s.cols + p.eps) : 1.f;
    const int padded = (int)f8_padded(s.cols);
    codes += row * padded;
    scales += row * (padded / kF8Block);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const At at = place(k);
        const int want = (k * NT + tid) * N;
        float n[N], w[N];
#pragma unroll
        for (int i = 0; i < N; ++i) n[i] = to_f32(y[k].v[i]);
        if (p.w2) {
            load_weights(w, p.w2, at, s.cols);
#pragma unroll
            for (int i = 0; i < N; ++i) n[i] = n[i] * rstd2 * w[i];
        }
        uint32_t largest = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            n[i] = at.own(i) ? n[i] : 0.f;
            largest = max(largest, magnitude(n[i]));
        }
        const F8Scale f(lanes_max<LANES>(largest));
#pragma unroll
        for (int i = 0; i < N; ++i) n[i] = f.quotient(n[i]);
        // the values that are the pack's own come first, the row's padding after them
        if constexpr (N == 8) {
            uint64_t c = (uint64_t)f8_codes(n[4], n[5], n[6], n[7]) << 32 | f8_codes(n[0], n[1], n[2], n[3]);
            if (CUT) c = at.lo < N ? c >> (8 * at.lo) : 0;
            if (want < padded) *(uint64_t*)(codes + want) = c;
        } else {
            uint32_t c = f8_codes(n[0], n[1], n[2], n[3]);
            if (CUT) c = at.lo < N ? c >> (8 * at.lo) : 0;
            if (want < padded) *(uint32_t*)(codes + want) = c;
        }
        if (want < padded && want % kF8Block == 0) scales[want / kF8Block] = f.scale;
    }
}

template <class T, int K, int NT, int ROWS>
int launch(NormShape s, NormFwd a, uint8_t* codes, float* scales, hipStream_t st) {
    // as many rows at once as a launch may have threads for
    constexpr int kMost = (int)std::min<int64_t>(kMaxThreads / NT / 2, 1 << 30);
    for (int left = s.rows; left > 0; left -= kMost) {
        s.rows = std::min(left, kMost);
        const dim3 grid((s.rows + ROWS - 1) / ROWS), block(NT * ROWS);
        if (s.cols % Wide<T>::N) hipLaunchKernelGGL((norm_fwd_f8_rows<T, K, NT, ROWS, true>), grid, block, 0, st, a, s, codes, scales);
        else hipLaunchKernelGGL((norm_fwd_f8_rows<T, K, NT, ROWS, false>), grid, block, 0, st, a, s, codes, scales);
        SEERA_HIP_TRY(hipGetLastError());
        auto on = [&](auto& p, int64_t ld) {
            if (p) p = (std::decay_t<decltype(p)>)((char*)p + s.rows * ld);
        };
        on(a.y, a.ldy * sizeof(T)), on(a.g, a.ldg * sizeof(T));
        on(a.r, s.cols * sizeof(T)), on(a.r_out, s.cols * sizeof(T));
        on(codes, f8_padded(s.cols)), on(scales, f8_padded(s.cols) / kF8Block * sizeof(float));
    }
    return SEERA_OK;
}

// Threads of a row as the plain forward has them (block_norm.hip), for the padded
// row: padding has threads of its own.
template <class T>
int launch_t(const NormShape& s, const NormFwd& a, uint8_t* codes, float* scales, hipStream_t st) {
    const int packs = (int)(f8_padded(s.cols) / Wide<T>::N);
    if (packs <= 64) return launch<T, 1, 64, 4>(s, a, codes, scales, st);
    if (packs <= 128) return launch<T, 2, 64, 4>(s, a, codes, scales, st);
    if (packs <= 256) return launch<T, 4, 64, 4>(s, a, codes, scales, st);
    if (packs <= 512) return launch<T, 2, 256, 1>(s, a, codes, scales, st);
    if (packs <= 1024) return launch<T, 4, 256, 1>(s, a, codes, scales, st);
    if (packs <= 2048) return launch<T, 2, 1024, 1>(s, a, codes, scales, st);
    if constexpr (Wide<T>::N == 4) return launch<T, 4, 1024, 1>(s, a, codes, scales, st);
    return SEERA_OK;  // 16384 columns of 16 bits are 2048 packs
}

}  // namespace

int block_norm_fwd_f8(const NormShape& s, const NormFwd& a, uint8_t* codes, float* scales, hipStream_t st) {
    return s.dtype == SEERA_DTYPE_F32   ? launch_t<float>(s, a, codes, scales, st)
           : s.dtype == SEERA_DTYPE_F16 ? launch_t<f16_t>(s, a, codes, scales, st)
                                        : launch_t<bf16_t>(s, a, codes, scales, st);
}

}  // namespace seera
