// zs_head_args.h -- kernel arguments of the heads of rows (zs_head.hip) and the
// layout of their scratch.
#pragma once
#include <hip/hip_runtime.h>
#include "zs_internal.h"

#define HD_KMAX 128            // entries of a head at most
#define HD_WAVE 2048           // values of a row that a wave of the head's pass takes
#define HD_CHUNK 8192          // values that a workgroup takes
#define HD_GROUPS 5120         // groups of a row at most (the pick holds their maxima in registers)
#define HD_BLOCKS (1u << 22)   // workgroups per launch at most

// n / d for n < 2^31 by a product: n / d = mulhi(n, mul) >> (sh - 32), d >= 2,
// with mul = ceil(2^sh / d) and 2^sh the first power at or above 2^31 d (the
// excess e = mul d - 2^sh < d gives n e < 2^31 d <= 2^sh). sh 0: d is 1.
struct zs_div {
    uint32_t mul, sh;
};
inline zs_div zs_div_of(uint64_t d) {
    zs_div q = {0, 0};
    if (d <= 1 || d >= 1ull << 31) return q;
    q.sh = 31;
    while (1ull << (q.sh - 31) < d) q.sh++;
    q.mul = (uint32_t)(((1ull << q.sh) + d - 1) / d);
    return q;
}
#if defined(__HIPCC__)
__device__ __forceinline__ uint32_t zs_quot(uint32_t n, zs_div q) { return q.sh ? __umulhi(n, q.mul) >> (q.sh - 32u) : n; }
#endif

// The heads of R rows. For a teacher (d_ids) the list goes out as ids and
// log-probabilities; for the beam step into `list` (bits of x~ << 32 | id,
// ~0 for none) and `norm`, of the rows whose beam lives.
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
    double* norm;               // [R][2] maximum, ln sum exp(x~ - maximum)
    uint32_t* count;            // [R / width] rows of the request that are done (cleared by the pass)
    // the pass: group maxima and, per wave, (maximum, sum exp((x - maximum) / T))
    uint32_t chunks;            // workgroups a row
    zs_div by_chunks, by_width;
    uint32_t gstride, recs;     // groups and records a row
    uint32_t* gmax;             // [R][gstride] keys
    float2* rec;                // [R][recs]
    // teacher
    uint32_t* ids;
    float* logp;
    float* lse_out;
};
struct bm_args;
int hd_head_launch(const hd_args& a, const bm_args* beam, uint32_t dtype, hipStream_t stream);   // beam: the step too

// log2 of the values in a group: 64, or 16 where a row has few groups for the
// list that is wanted (a threshold from group maxima is close only when there
// are several times K of them), or 256 where 64 would make more than HD_GROUPS.
// By 16 and by 64, us: 256 f32 rows of 20000 13.8 and 16.6 for K = 64, 20.8 and
// 25.5 for 128; of 32000 16.6 and 17.9, 23.5 and 28.4; 2048 of 50257 for 128 110
// and 113; bf16 52 and 61 (2048 rows of 20000, K = 128).
inline uint32_t hd_group_shift(uint32_t V, uint32_t K) {
    if ((V >> 6) + 2u > HD_GROUPS) return 8;
    return (V >> 6) >= 8u * K || (V >> 4) + 2u > HD_GROUPS ? 6 : 4;
}
// The scratch of R rows: the pass's and, for the beam step, the lists and
// normalisers. A row's first value may lie up to 15 bytes behind a 16-byte
// boundary, from which groups and chunks are counted: 7 values more.
inline uint64_t hd_pad(uint64_t n) { return (n + 255u) & ~(uint64_t)255u; }
inline uint64_t hd_work(hd_args& a, void* work, bool beam) {
    char* p = (char*)work;
    const uint32_t gs = hd_group_shift(a.V, a.K);
    a.chunks = (a.V + 7u + HD_CHUNK - 1u) / HD_CHUNK;
    a.recs = a.chunks * (HD_CHUNK / HD_WAVE);
    a.by_chunks = zs_div_of(a.chunks);
    a.by_width = zs_div_of(a.width);
    a.gstride = (a.V + 7u + (1u << gs) - 1u) >> gs;
    a.gmax = (uint32_t*)p;
    p += hd_pad(a.R * a.gstride * 4u);
    a.rec = (float2*)p;
    p += hd_pad(a.R * a.recs * 8u);
    if (beam) {
        a.list = (unsigned long long*)p;
        p += hd_pad(a.R * a.K * 8u);
        a.norm = (double*)p;
        p += hd_pad(a.R * 16u);
        a.count = (uint32_t*)p;
        p += hd_pad(a.R * 4u);
    }
    return (uint64_t)(p - (char*)work);
}
inline uint64_t hd_work_bytes(uint64_t R, uint32_t V, uint32_t K, bool beam) {
    hd_args a{};
    a.R = R;
    a.V = V;
    a.K = K;
    return hd_work(a, (void*)256, beam);
}
