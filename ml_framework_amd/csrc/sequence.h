// sequence.h -- internal entry points of the sequence model's operators: the
// gated scan (gated_scan.hip), the block norm (block_norm.hip) and the AdamW
// step (adamw.hip). Arguments are checked by capi_sequence.cpp; all enqueue on
// `st` without synchronizing and return a SEERA_* status.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/seera_hip.h"

namespace seera {

// Threads that one launch may have along an axis.
constexpr int64_t kMaxThreads = (int64_t)1 << 32;

// Rows of a [batch, time] matrix of `channels` values, `ld` elements apart;
// row (b, t) is b * time + t, or t * batch + b where time_major.
struct ScanShape {
    int batch, time, channels;
    int gate, time_major, dtype;
};
struct ScanFwd {
    const void *x, *f;
    const float* h0;
    const int* lengths;
    void* h;
    float* hT;
    int64_t ldx, ldf;
};
struct ScanBwd {
    const void *x, *f;
    const float* h0;
    const int* lengths;
    const void *h, *dh;
    const float* dhT;
    void *dx, *df;
    float* dh0;
    int64_t ldx, ldf, lddx, lddf;
};
int gated_scan_fwd(const ScanShape& s, const ScanFwd& a, hipStream_t st);
int gated_scan_bwd(const ScanShape& s, const ScanBwd& a, hipStream_t st);

struct NormShape {
    int rows, cols, act, dtype;
};
struct NormFwd {
    const void *y, *g, *r;
    const float *w1, *s, *w2;
    void *r_out, *n_out;
    float *rstd1, *rstd2;
    int64_t ldy, ldg;
    float eps;
};
struct NormBwd {
    const void *y, *g, *r_out;
    const float *w1, *s, *w2, *rstd1, *rstd2;
    const void *dr_out, *dn;
    void *dy, *dg, *dr;
    float *dw1, *ds, *dw2;
    int64_t ldy, ldg, lddy, lddg;
};
int block_norm_fwd(const NormShape& s, const NormFwd& a, hipStream_t st);
int block_norm_bwd(const NormShape& s, const NormBwd& a, hipStream_t st);
// Columns a row of the block norm may have.
constexpr int kNormMaxCols = 16384;

// The step's constants, in the form the kernel uses them.
struct AdamwStep {
    float beta1, one_minus_beta1, beta2, one_minus_beta2;
    float step_size;       // lr / (1 - beta1^t)
    float inv_sqrt_corr2;  // 1 / sqrt(1 - beta2^t)
    float eps;
    double lr;
    uint32_t seed;
    const float* grad_scale;  // device, or null for 1
};
int adamw_step(const seera_adamw_tensor* tensors, int n, const AdamwStep& step, hipStream_t st);
int adamw_state_values(const seera_adamw_tensor* tensors, int n, float* const* m_values, float* const* v_values, hipStream_t st);

}  // namespace seera
