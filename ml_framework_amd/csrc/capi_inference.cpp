// capi_inference.cpp -- the extern "C" entry points of include/seera_hip.h for the
// operators that a model answers with: the block norm with its output in 8 bits,
// weights in 8 bits, their product, sampling. Each checks its arguments before any
// device work; the plain forms run on the null stream and synchronize, the _async
// forms enqueue on the caller's stream.
#include "capi_args.h"
#include "f8.h"
#include "inference.h"

using namespace seera;

namespace {

// The largest matrix of codes: places in it, and its tiles' distances, stay in 63 bits.
bool too_many(double rows, double row) { return rows * row > 0x1p60; }

int norm_f8(const NormShape& s, const NormFwd& a, hipStream_t st) {
    const char* op = "block_norm_f8";
    if (s.rows < 0 || s.cols < 0) return bad(op, "dims must be >= 0");
    if (s.cols > kNormMaxCols) return fail(SEERA_ERR_INVALID_ARGUMENT, "%s: cols %d above %d", op, s.cols, kNormMaxCols);
    if (s.act != SEERA_GATE_ACT_SILU && s.act != SEERA_GATE_ACT_SIGMOID) return fail(SEERA_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", op, s.act);
    const size_t e = dtype_bytes(s.dtype);
    if (!e) return fail(SEERA_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", op, s.dtype);
    for (int64_t ld : {a.ldy, a.g ? a.ldg : s.cols}) {
        if (ld < s.cols) return bad(op, "a row distance is below cols");
        if (ld > (int64_t)1 << 30) return bad(op, "a row distance is too large");
    }
    if (!(a.eps >= 0.f)) return bad(op, "eps must be >= 0");
    if (s.rows == 0 || s.cols == 0) return SEERA_OK;
    SEERA_TRY(required(op, e, {a.y}));
    SEERA_TRY(required(op, 4, {a.scales}));
    SEERA_TRY(required(op, 16, {a.codes}));
    SEERA_TRY(optional(op, e, {a.g, a.r, a.r_out}));
    SEERA_TRY(optional(op, 4, {a.w1, a.s, a.w2}));
    return block_norm_fwd_f8(s, a, st);
}

int quantize(const QuantizeF8& a, hipStream_t st) {
    const char* op = "quantize_weights_f8";
    if (a.n < 0 || a.k < 0) return bad(op, "dims must be >= 0");
    const size_t e = dtype_bytes(a.dtype);
    if (!e) return fail(SEERA_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", op, a.dtype);
    if (a.transposed != 0 && a.transposed != 1) return bad(op, "transposed must be 0 or 1");
    if (a.ldw < (a.transposed ? a.k : a.n)) return bad(op, "ldw is below the length of a row");
    if (too_many(a.transposed ? a.n : a.k, (double)a.ldw)) return bad(op, "ldw is too large");
    if (a.k > 0x7fffff00 || a.n > 0x7fffff00) return bad(op, "n or k is too large");  // padded, they fit an int
    if (a.n == 0 || a.k == 0) return SEERA_OK;
    SEERA_TRY(required(op, e, {a.w}));
    SEERA_TRY(required(op, 4, {a.scales}));
    SEERA_TRY(required(op, 16, {a.codes}));
    return quantize_weights_f8(a, st);
}

int product(const MatmulF8& a, int k, hipStream_t st) {
    const char* op = "matmul_f8";
    if (a.m < 0 || a.n < 0 || k < 0) return bad(op, "dims must be >= 0");
    const size_t e = dtype_bytes(a.dtype);
    if (!e) return fail(SEERA_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", op, a.dtype);
    if (a.ldc < a.n) return bad(op, "ldc is below N");
    if (too_many(a.m, (double)a.ldc)) return bad(op, "ldc is too large");
    if (a.m > 0x7fffff00 || a.n > 0x7fffff00 || k > 0x7fffff00) return bad(op, "M, N or K is too large");  // padded, they fit an int
    if (a.m == 0 || a.n == 0) return SEERA_OK;
    SEERA_TRY(required(op, e, {a.c}));
    SEERA_TRY(optional(op, 4, {a.bias}));
    if (k > 0) {
        SEERA_TRY(required(op, 16, {a.a, a.w}));
        SEERA_TRY(required(op, 4, {a.a_scales, a.w_scales}));
    }
    return matmul_f8(a, st);
}

int draw(const Sample& a, hipStream_t st) {
    const char* op = "sample";
    if (a.rows < 0 || a.vocab < 0) return bad(op, "dims must be >= 0");
    if (a.vocab > kSampleMaxVocab) return fail(SEERA_ERR_INVALID_ARGUMENT, "%s: vocab %d above %d", op, a.vocab, kSampleMaxVocab);
    const size_t e = dtype_bytes(a.dtype);
    if (!e) return fail(SEERA_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", op, a.dtype);
    if (a.ld < a.vocab) return bad(op, "a row distance is below vocab");
    if (too_many(a.rows, (double)a.ld)) return bad(op, "a row distance is too large");
    if (a.rows == 0) return SEERA_OK;
    if (a.vocab > 0) SEERA_TRY(required(op, e, {a.logits}));
    SEERA_TRY(required(op, 4, {a.uniform, a.tokens}));
    SEERA_TRY(optional(op, 4, {a.temperature, a.top_k, a.top_p, a.min_p, a.logp}));
    return sample(a, st);
}

}  // namespace

extern "C" {

#define NORM_F8_ARGS                                                                                                        \
    const void *y, const void *g, const void *r, const float *w1, const float *s, const float *w2, void *r_out,             \
        uint8_t *codes, float *scales, int rows, int cols, int64_t ldy, int64_t ldg, float eps, int act, int dtype
#define NORM_F8_CALL                                                                                                        \
    [&](hipStream_t st) {                                                                                                   \
        return norm_f8({rows, cols, act, dtype}, {y, g, r, w1, s, w2, r_out, nullptr, nullptr, nullptr, ldy, ldg, eps,      \
                       codes, scales}, st);                                                                                 \
    }
int seera_hip_block_norm_fwd_f8(NORM_F8_ARGS) { return now(NORM_F8_CALL); }
int seera_hip_block_norm_fwd_f8_async(NORM_F8_ARGS, void* stream) { return later(stream, NORM_F8_CALL); }

#define QUANTIZE_ARGS const void *w, uint8_t *codes, float *scales, int n, int k, int64_t ldw, int transposed, int dtype
#define QUANTIZE_CALL [&](hipStream_t st) { return quantize({w, codes, scales, n, k, ldw, transposed, dtype}, st); }
int seera_hip_quantize_weights_f8(QUANTIZE_ARGS) { return now(QUANTIZE_CALL); }
int seera_hip_quantize_weights_f8_async(QUANTIZE_ARGS, void* stream) { return later(stream, QUANTIZE_CALL); }

#define MATMUL_F8_ARGS                                                                                                      \
    const uint8_t *a, const float *a_scales, const uint8_t *w, const float *w_scales, const float *bias, void *C, int M,    \
        int N, int K, int64_t ldc, int dtype
#define MATMUL_F8_CALL                                                                                                      \
    [&](hipStream_t st) {                                                                                                   \
        return product({a, a_scales, w, w_scales, bias, C, M, N, (int)(f8_padded(K) / kF8Block), ldc, dtype}, K, st);       \
    }
int seera_hip_matmul_f8(MATMUL_F8_ARGS) { return now(MATMUL_F8_CALL); }
int seera_hip_matmul_f8_async(MATMUL_F8_ARGS, void* stream) { return later(stream, MATMUL_F8_CALL); }

#define SAMPLE_ARGS                                                                                                         \
    const void *logits, const float *uniform, const float *temperature, const int *top_k, const float *top_p,               \
        const float *min_p, int *tokens, float *logp, int rows, int vocab, int64_t ld, int dtype
#define SAMPLE_CALL \
    [&](hipStream_t st) { return draw({logits, uniform, temperature, top_k, top_p, min_p, tokens, logp, rows, vocab, ld, dtype}, st); }
int seera_hip_sample(SAMPLE_ARGS) { return now(SAMPLE_CALL); }
int seera_hip_sample_async(SAMPLE_ARGS, void* stream) { return later(stream, SAMPLE_CALL); }

}  // extern "C"
