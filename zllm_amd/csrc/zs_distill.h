// zs_distill.h -- kernel arguments of distillation from a teacher's list.
#pragma once
#include <hip/hip_runtime.h>
#include "zs_internal.h"

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
    float* work;             // records
};
#define DS_LOSS 1
#define DS_GRAD 2
int ds_launch(const ds_args& a, uint32_t dtype, int what, hipStream_t stream);
// The scratch of N rows.
inline uint64_t ds_work_bytes(uint64_t N, uint32_t V) {
    (void)N;
    (void)V;
    return 0;
}
