// zs_beam.h -- kernel arguments of the beam step and of the reordering.
#pragma once
#include <hip/hip_runtime.h>
#include "zs_head_args.h"

struct bm_args {
    uint32_t width, K, n_eos, early;
    uint32_t eos[ZS_BEAM_MAX_EOS];
    float length_penalty;
    const float* scores;
    const unsigned long long* list;   // [groups*width][K]
    const double* norm;               // [groups*width][2] maximum, ln sum exp(x~ - maximum)
    const float* fin_score;
    const int32_t *fin_length, *fin_parent, *fin_token, *steps, *done;
    float* fin_score_o;
    int32_t *fin_length_o, *fin_parent_o, *fin_token_o, *steps_o, *done_o;
    int32_t *parent, *token;
    float* score_o;
    zs_div by_kw;   // ceil(K / 4)
};

// One state array: `total` columns of `unit` bytes per row in blocks of `cols`.
struct bm_state {
    char* base;
    uint64_t row_stride, outer_stride, inner_stride, cols, total;
    uint32_t n_inner, unit, first, blocks;   // blocks [first, first + blocks) of the launch
    zs_div by_cols, by_inner;                // (total < 2^31)
};
struct ro_args {
    const int32_t* parent;
    uint32_t width, n;
    bm_state s[ZS_REORDER_BATCH];
};
int ro_launch(const ro_args& a, uint32_t blocks, uint32_t groups, hipStream_t stream);
// Workgroups for `total` columns of a group's rows: a column per thread up to
// about 32 workgroups a CU over all groups, loops past that.
inline uint32_t ro_blocks(uint64_t total, uint32_t groups) {
    const uint64_t want = (total + 255u) / 256u, most = 32768u / groups + 1u;
    return (uint32_t)(want < most ? want : most);
}
