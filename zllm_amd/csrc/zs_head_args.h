// zs_head_args.h -- kernel arguments of the heads of rows (zs_head.hip) and the
// layout of their scratch.
#pragma once
#include <hip/hip_runtime.h>
#include "zs_internal.h"

#define HD_KMAX 128            // entries of a head at most
#define HD_ROWS (1u << 20)     // rows per launch at most

// The heads of R rows. For a teacher (d_ids) the list goes out as ids and
// log-probabilities; for the beam step into `list` (bits of x~ << 32 | id,
// ~0 for none) and `lse`, of the rows whose beam lives.
struct hd_args {
    const void* logits;
    uint64_t ld, R;
    uint32_t V, K;
    float c;                    // log2(e) / T
    double inv_t;               // 1 / T
    const uint32_t* allow;
    uint32_t allow_words;
    // beam step
    const float* scores;        // NULL: every row is taken
    const int32_t* done;
    uint32_t width;
    unsigned long long* list;   // [R][K]
    double* lse;                // [R]
    // teacher
    uint32_t* ids;
    float* logp;
    float* lse_out;
};
int hd_head_launch(const hd_args& a, uint32_t dtype, hipStream_t stream);

// The scratch of R rows: (beam) the lists and normalisers.
inline uint64_t hd_pad(uint64_t n) { return (n + 255u) & ~(uint64_t)255u; }
inline uint64_t hd_work_bytes(uint64_t R, uint32_t V, uint32_t K, bool beam) {
    (void)V;
    return beam ? hd_pad(R * K * 8u) + hd_pad(R * 8u) : 0u;
}
inline void hd_work(hd_args& a, void* work, bool beam) {
    char* p = (char*)work;
    if (beam) {
        a.list = (unsigned long long*)p;
        p += hd_pad(a.R * a.K * 8u);
        a.lse = (double*)p;
        p += hd_pad(a.R * 8u);
    }
}
