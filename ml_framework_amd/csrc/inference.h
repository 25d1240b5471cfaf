// inference.h -- internal entry points of the operators that a model answers with:
// the block norm with its output in 8 bits (block_norm.hip), weights in 8 bits
// (quantize_f8.hip), their product (matmul_f8.hip) and sampling (sample.hip).
// Arguments are checked by capi_inference.cpp; all enqueue on `st` without
// synchronizing and return a SEERA_* status.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sequence.h"

namespace seera {

// `a` without n_out and statistics; codes [rows][f8_padded(cols)], scales
// [rows][f8_padded(cols) / 128].
int block_norm_fwd_f8(const NormShape& s, const NormFwd& a, hipStream_t st);

// w is [k, n], or [n, k] where transposed, rows ldw elements apart.
struct QuantizeF8 {
    const void* w;
    uint8_t* codes;
    float* scales;
    int n, k;
    int64_t ldw;
    int transposed, dtype;
};
int quantize_weights_f8(const QuantizeF8& a, hipStream_t st);

struct MatmulF8 {
    const uint8_t* a;
    const float* a_scales;
    const uint8_t* w;
    const float* w_scales;
    const float* bias;
    void* c;
    int m, n, blocks;  // blocks of 128 of K
    int64_t ldc;
    int dtype;
};
int matmul_f8(const MatmulF8& a, hipStream_t st);

struct Sample {
    const void* logits;
    const float *uniform, *temperature;
    const int* top_k;
    const float *top_p, *min_p;
    int* tokens;
    float* logp;
    int rows, vocab;
    int64_t ld;
    int dtype;
};
int sample(const Sample& a, hipStream_t st);
// Tokens a row of logits may have: sums of weights of 40 bits stay below 2^62.
constexpr int kSampleMaxVocab = 1 << 22;

}  // namespace seera
