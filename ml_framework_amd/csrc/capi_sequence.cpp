// capi_sequence.cpp -- the extern "C" entry points of include/seera_hip.h for
// the sequence model's operators (gated scan, block norm, AdamW). Each checks
// its arguments before any device work; the plain forms run on the null stream
// and synchronize, the _async forms enqueue on the caller's stream.
#include <math.h>

#include "io_types.h"
#include "runtime.h"
#include "sequence.h"

using namespace seera;

namespace {

template <class F>
int now(F&& f) {
    clear_error();
    SEERA_TRY(f(nullptr));
    SEERA_HIP_TRY(hipDeviceSynchronize());
    note_device_synchronized();
    return SEERA_OK;
}
template <class F>
int later(void* stream, F&& f) {
    clear_error();
    SEERA_TRY(f(reinterpret_cast<hipStream_t>(stream)));
    note_async_work();
    return SEERA_OK;
}

int bad(const char* op, const char* what) { return fail(SEERA_ERR_INVALID_ARGUMENT, "%s: %s", op, what); }

// Each of `ptrs` must not be null and must be aligned to a value of `bytes`.
int required(const char* op, size_t bytes, std::initializer_list<const void*> ptrs) {
    for (const void* p : ptrs) {
        if (!p) return bad(op, "null device pointer");
        if (!aligned_to(p, bytes)) return bad(op, "a pointer is not aligned to its type");
    }
    return SEERA_OK;
}
// The same where a pointer is given.
int optional(const char* op, size_t bytes, std::initializer_list<const void*> ptrs) {
    for (const void* p : ptrs)
        if (!aligned_to(p, bytes)) return bad(op, "a pointer is not aligned to its type");
    return SEERA_OK;
}

// ---- gated scan ----

// `work`: whether there is a row to compute.
int scan_shape(const ScanShape& s, std::initializer_list<int64_t> lds, bool* work) {
    const char* op = "gated_scan";
    if (s.batch < 0 || s.time < 0 || s.channels < 0) return bad(op, "dims must be >= 0");
    if (s.time > 1 << 30) return bad(op, "time is above 2^30");  // tiles step past the end in int
    if (s.gate != SEERA_GATE_LINEAR && s.gate != SEERA_GATE_SIGMOID) return fail(SEERA_ERR_INVALID_ARGUMENT, "%s: unknown gate %d", op, s.gate);
    if (s.time_major != 0 && s.time_major != 1) return bad(op, "time_major must be 0 or 1");
    if (!dtype_bytes(s.dtype)) return fail(SEERA_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", op, s.dtype);
    for (int64_t ld : lds) {
        if (ld < s.channels) return bad(op, "a row distance is below channels");
        // keeps row * ld, in bytes, inside int64
        if (ld > (int64_t)1 << 40 || (double)s.batch * s.time * ld > 0x1p60) return bad(op, "a row distance is too large");
    }
    *work = s.time > 0;
    return SEERA_OK;
}

int scan_fwd(const ScanShape& s, const ScanFwd& a, hipStream_t st) {
    const char* op = "gated_scan";
    bool work;
    SEERA_TRY(scan_shape(s, {a.ldx, a.ldf}, &work));
    if (s.batch == 0 || s.channels == 0) return SEERA_OK;
    const size_t e = dtype_bytes(s.dtype);
    if (work) SEERA_TRY(required(op, e, {a.x, a.f, a.h}));
    SEERA_TRY(optional(op, 4, {a.h0, a.lengths, a.hT}));
    if (!work && !a.hT) return SEERA_OK;
    return gated_scan_fwd(s, a, st);
}

int scan_bwd(const ScanShape& s, ScanBwd a, hipStream_t st) {
    const char* op = "gated_scan";
    bool work;
    if (s.gate == SEERA_GATE_LINEAR) a.x = nullptr, a.ldx = s.channels;  // not read
    SEERA_TRY(scan_shape(s, {a.ldx, a.ldf, a.lddx, a.lddf}, &work));
    if (s.batch == 0 || s.channels == 0) return SEERA_OK;
    const size_t e = dtype_bytes(s.dtype);
    if (work) {
        SEERA_TRY(required(op, e, {a.f, a.h, a.dh, a.dx, a.df}));
        if (s.gate == SEERA_GATE_SIGMOID) SEERA_TRY(required(op, e, {a.x}));
    }
    SEERA_TRY(optional(op, 4, {a.h0, a.lengths, a.dhT, a.dh0}));
    if (!work && !a.dh0) return SEERA_OK;
    return gated_scan_bwd(s, a, st);
}

// ---- block norm ----

int norm_shape(const NormShape& s, std::initializer_list<int64_t> lds) {
    const char* op = "block_norm";
    if (s.rows < 0 || s.cols < 0) return bad(op, "dims must be >= 0");
    if (s.cols > kNormMaxCols) return fail(SEERA_ERR_INVALID_ARGUMENT, "%s: cols %d above %d", op, s.cols, kNormMaxCols);
    if (s.act != SEERA_GATE_ACT_SILU && s.act != SEERA_GATE_ACT_SIGMOID) return fail(SEERA_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", op, s.act);
    if (!dtype_bytes(s.dtype)) return fail(SEERA_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", op, s.dtype);
    for (int64_t ld : lds) {
        if (ld < s.cols) return bad(op, "a row distance is below cols");
        if (ld > (int64_t)1 << 30) return bad(op, "a row distance is too large");
    }
    return SEERA_OK;
}

int norm_fwd(const NormShape& s, const NormFwd& a, hipStream_t st) {
    const char* op = "block_norm";
    SEERA_TRY(norm_shape(s, {a.ldy, a.g ? a.ldg : s.cols}));
    if (!(a.eps >= 0.f)) return bad(op, "eps must be >= 0");
    if (!a.w2 && a.n_out) return bad(op, "n_out needs w2");
    if (s.rows == 0 || s.cols == 0) return SEERA_OK;
    const size_t e = dtype_bytes(s.dtype);
    SEERA_TRY(required(op, e, {a.y}));
    if (a.w2) SEERA_TRY(required(op, e, {a.n_out}));
    else SEERA_TRY(required(op, e, {a.r_out}));
    SEERA_TRY(optional(op, e, {a.g, a.r, a.r_out}));
    SEERA_TRY(optional(op, 4, {a.w1, a.s, a.w2, a.rstd1, a.rstd2}));
    return block_norm_fwd(s, a, st);
}

int norm_bwd(const NormShape& s, const NormBwd& a, hipStream_t st) {
    const char* op = "block_norm";
    SEERA_TRY(norm_shape(s, {a.w1 || a.g || a.s ? a.ldy : s.cols, a.g ? a.ldg : s.cols, a.lddy, a.g ? a.lddg : s.cols}));
    if (!a.w2 && a.dn) return bad(op, "dn needs w2");
    if (s.cols == 0) return SEERA_OK;
    const size_t e = dtype_bytes(s.dtype);
    if (a.w1) SEERA_TRY(required(op, 4, {a.w1, a.dw1}));
    if (a.s) SEERA_TRY(required(op, 4, {a.s, a.ds}));
    if (a.w2) SEERA_TRY(required(op, 4, {a.w2, a.dw2}));
    if (s.rows > 0) {
        SEERA_TRY(required(op, e, {a.dy}));
        if (a.w1) SEERA_TRY(required(op, 4, {a.rstd1}));
        if (a.w1 || a.g || a.s) SEERA_TRY(required(op, e, {a.y}));
        if (a.g) SEERA_TRY(required(op, e, {a.g, a.dg}));
        if (a.w2) {
            SEERA_TRY(required(op, e, {a.r_out, a.dn}));
            SEERA_TRY(required(op, 4, {a.rstd2}));
        } else {
            SEERA_TRY(required(op, e, {a.dr_out}));
        }
        SEERA_TRY(optional(op, e, {a.dr_out, a.dr}));
    }
    return block_norm_bwd(s, a, st);
}

// ---- AdamW ----

int adamw_tensors(const char* op, const seera_adamw_tensor* t, int n) {
    if (n < 0) return bad(op, "the number of tensors must be >= 0");
    if (n > 0 && !t) return bad(op, "null array of tensors");
    for (int i = 0; i < n; ++i) {
        if (t[i].count < 0) return fail(SEERA_ERR_INVALID_ARGUMENT, "%s: tensor %d has a negative count", op, i);
        if (t[i].state_bits != 32 && t[i].state_bits != 8)
            return fail(SEERA_ERR_INVALID_ARGUMENT, "%s: tensor %d has state_bits %d, not 32 or 8", op, i, t[i].state_bits);
        if (t[i].count == 0) continue;
        const bool codes = t[i].state_bits == 8;
        SEERA_TRY(required(op, codes ? 1 : 4, {t[i].m, t[i].v}));
        if (codes) SEERA_TRY(required(op, 1, {t[i].m_exp, t[i].v_exp}));
    }
    return SEERA_OK;
}

int step(const seera_adamw_tensor* t, int n, double lr, double beta1, double beta2, double eps, int64_t at, uint32_t seed,
         const float* grad_scale, hipStream_t st) {
    const char* op = "adamw_step";
    if (!isfinite(lr)) return bad(op, "lr must be finite");
    if (!(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1)) return bad(op, "betas must be in [0, 1)");
    if (!(eps >= 0)) return bad(op, "eps must be >= 0");
    if (at < 1) return bad(op, "step counts from 1");
    SEERA_TRY(adamw_tensors(op, t, n));
    SEERA_TRY(optional(op, 4, {grad_scale}));
    for (int i = 0; i < n; ++i) {
        if (!isfinite(t[i].weight_decay)) return fail(SEERA_ERR_INVALID_ARGUMENT, "%s: tensor %d has a weight_decay that is not finite", op, i);
        const int e = dtype_bytes(t[i].grad_dtype);
        if (!e) return fail(SEERA_ERR_INVALID_ARGUMENT, "%s: tensor %d has an unknown grad_dtype", op, i);
        if (t[i].param16 && t[i].param16_dtype != SEERA_DTYPE_F16 && t[i].param16_dtype != SEERA_DTYPE_BF16)
            return fail(SEERA_ERR_INVALID_ARGUMENT, "%s: tensor %d has a param16_dtype that is not fp16 or bf16", op, i);
        if (t[i].count == 0) continue;
        SEERA_TRY(required(op, 4, {t[i].param}));
        SEERA_TRY(required(op, e, {t[i].grad}));
        SEERA_TRY(optional(op, 2, {t[i].param16}));
    }
    AdamwStep s;
    s.beta1 = (float)beta1;
    s.one_minus_beta1 = (float)(1.0 - beta1);
    s.beta2 = (float)beta2;
    s.one_minus_beta2 = (float)(1.0 - beta2);
    s.step_size = (float)(lr / (1.0 - pow(beta1, (double)at)));
    s.inv_sqrt_corr2 = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)at)));
    s.eps = (float)eps;
    s.lr = lr;
    s.seed = seed;
    s.grad_scale = grad_scale;
    return adamw_step(t, n, s, st);
}

int values(const seera_adamw_tensor* t, int n, float* const* m, float* const* v, hipStream_t st) {
    const char* op = "adamw_state_values";
    SEERA_TRY(adamw_tensors(op, t, n));
    if (n > 0 && (!m || !v)) return bad(op, "null array of pointers");
    for (int i = 0; i < n; ++i) SEERA_TRY(optional(op, 4, {m[i], v[i]}));
    return adamw_state_values(t, n, m, v, st);
}

}  // namespace

extern "C" {

#define SCAN_FWD_ARGS                                                                                                       \
    const void *x, const void *f, const float *h0, const int *lengths, void *h, float *hT, int batch, int time,             \
        int channels, int64_t ldx, int64_t ldf, int gate, int time_major, int dtype
#define SCAN_FWD_CALL \
    [&](hipStream_t st) { return scan_fwd({batch, time, channels, gate, time_major, dtype}, {x, f, h0, lengths, h, hT, ldx, ldf}, st); }
int seera_hip_gated_scan_fwd(SCAN_FWD_ARGS) { return now(SCAN_FWD_CALL); }
int seera_hip_gated_scan_fwd_async(SCAN_FWD_ARGS, void* stream) { return later(stream, SCAN_FWD_CALL); }

#define SCAN_BWD_ARGS                                                                                                       \
    const void *x, const void *f, const float *h0, const int *lengths, const void *h, const void *dh, const float *dhT,     \
        void *dx, void *df, float *dh0, int batch, int time, int channels, int64_t ldx, int64_t ldf, int64_t lddx,          \
        int64_t lddf, int gate, int time_major, int dtype
#define SCAN_BWD_CALL                                                                                                       \
    [&](hipStream_t st) {                                                                                                   \
        return scan_bwd({batch, time, channels, gate, time_major, dtype},                                                   \
                        {x, f, h0, lengths, h, dh, dhT, dx, df, dh0, ldx, ldf, lddx, lddf}, st);                            \
    }
int seera_hip_gated_scan_bwd(SCAN_BWD_ARGS) { return now(SCAN_BWD_CALL); }
int seera_hip_gated_scan_bwd_async(SCAN_BWD_ARGS, void* stream) { return later(stream, SCAN_BWD_CALL); }

#define NORM_FWD_ARGS                                                                                                       \
    const void *y, const void *g, const void *r, const float *w1, const float *s, const float *w2, void *r_out,             \
        void *n_out, float *rstd1, float *rstd2, int rows, int cols, int64_t ldy, int64_t ldg, float eps, int act, int dtype
#define NORM_FWD_CALL \
    [&](hipStream_t st) { return norm_fwd({rows, cols, act, dtype}, {y, g, r, w1, s, w2, r_out, n_out, rstd1, rstd2, ldy, ldg, eps}, st); }
int seera_hip_block_norm_fwd(NORM_FWD_ARGS) { return now(NORM_FWD_CALL); }
int seera_hip_block_norm_fwd_async(NORM_FWD_ARGS, void* stream) { return later(stream, NORM_FWD_CALL); }

#define NORM_BWD_ARGS                                                                                                       \
    const void *y, const void *g, const void *r_out, const float *w1, const float *s, const float *w2, const float *rstd1,  \
        const float *rstd2, const void *dr_out, const void *dn, void *dy, void *dg, void *dr, float *dw1, float *ds,        \
        float *dw2, int rows, int cols, int64_t ldy, int64_t ldg, int64_t lddy, int64_t lddg, int act, int dtype
#define NORM_BWD_CALL                                                                                                       \
    [&](hipStream_t st) {                                                                                                   \
        return norm_bwd({rows, cols, act, dtype},                                                                           \
                        {y, g, r_out, w1, s, w2, rstd1, rstd2, dr_out, dn, dy, dg, dr, dw1, ds, dw2, ldy, ldg, lddy, lddg}, st); \
    }
int seera_hip_block_norm_bwd(NORM_BWD_ARGS) { return now(NORM_BWD_CALL); }
int seera_hip_block_norm_bwd_async(NORM_BWD_ARGS, void* stream) { return later(stream, NORM_BWD_CALL); }

int seera_hip_adamw_step(const seera_adamw_tensor* tensors, int n, double lr, double beta1, double beta2, double eps,
                         int64_t at, uint32_t seed, const float* grad_scale) {
    return now([&](hipStream_t st) { return step(tensors, n, lr, beta1, beta2, eps, at, seed, grad_scale, st); });
}
int seera_hip_adamw_step_async(const seera_adamw_tensor* tensors, int n, double lr, double beta1, double beta2, double eps,
                               int64_t at, uint32_t seed, const float* grad_scale, void* stream) {
    return later(stream, [&](hipStream_t st) { return step(tensors, n, lr, beta1, beta2, eps, at, seed, grad_scale, st); });
}
int seera_hip_adamw_state_values(const seera_adamw_tensor* tensors, int n, float* const* m_values, float* const* v_values) {
    return now([&](hipStream_t st) { return values(tensors, n, m_values, v_values, st); });
}
int seera_hip_adamw_state_values_async(const seera_adamw_tensor* tensors, int n, float* const* m_values,
                                       float* const* v_values, void* stream) {
    return later(stream, [&](hipStream_t st) { return values(tensors, n, m_values, v_values, st); });
}

}  // extern "C"
