// zs_distill.h -- kernel arguments of distillation from a teacher's list and the
// layout of their scratch.
#pragma once
#include <hip/hip_runtime.h>
#include "zs_head_args.h"

// What the gradient of a row goes by. At an id of the list y = e * fi + e1 * f1
// - fp * p - fc * [the label] with e = 2^(x c - mc), outside it y = eo * fo +
// e1 * f1 (- fc) with eo = 2^(x co - mco); e1 = 2^(x c1 - m1).
struct ds_coef {
    float c, mc, c1, m1, fi, fo, f1, fp, fc;
    uint32_t lone;   // the label, where the list does not have it (~0 else)
    float co, mco;   // c and mc, or those of the outside ids' own maximum
};

struct ds_args {
    const void* logits;
    uint64_t ld, N;
    uint32_t V, K;
    const uint32_t* ids;
    const float* logp;
    const int64_t* labels;
    int64_t ignore;
    float c;                 // log2(e) / T
    double inv_t;            // 1 / T
    float kl, ce;            // the weights
    uint32_t tail;
    uint32_t two;            // CE is taken and T != 1: a second exponential per logit
    float* loss;
    float* stats;            // [N][4]
    const float* row_grad;
    uint64_t row_grad_stride;
    void* grad;
    uint64_t ld_grad;
    // scratch
    uint32_t chunks, recs;   // workgroups and records a row
    zs_div by_chunks;
    float4* rec;             // [N][recs] per wave: maximum, sums at T and at 1, the first outside the list
    ds_coef* coef;           // [N]
    float* p;                // [N][K] probability of an entry's id (an id listed twice has both), -1 for absent entries
};
#define DS_WAVE 2048         // values of a row that a wave takes
#define DS_LOSS 1
#define DS_GRAD 2
int ds_launch(const ds_args& a, uint32_t dtype, int what, hipStream_t stream);

// Chunks are counted from the 16-byte boundary at or below the row (7 values more).
inline uint64_t ds_work(ds_args& a, void* work) {
    char* p = (char*)work;
    a.chunks = (a.V + 7u + HD_CHUNK - 1u) / HD_CHUNK;
    a.recs = a.chunks * (HD_CHUNK / DS_WAVE);
    a.by_chunks = zs_div_of(a.chunks);
    a.rec = (float4*)p;
    p += hd_pad(a.N * a.recs * sizeof(float4));
    a.coef = (ds_coef*)p;
    p += hd_pad(a.N * sizeof(ds_coef));
    a.p = (float*)p;
    p += hd_pad(a.N * a.K * sizeof(float));
    return (uint64_t)(p - (char*)work);
}
