// zs_head.hip -- the head of a row of logits: its K largest values with their
// ids and its log-normaliser, for a teacher's lists (zs_teacher_topk) and for
// the beam step (zs_beam.hip).
#include "zs_head.h"

#define HR_NT 512

// Adds into lds[256] the histogram of 8-bit digits and returns, by the whole
// workgroup, the digit that holds the need-th key from above and what is
// still needed inside it.
template <int NT>
__device__ __forceinline__ void hr_digit(const uint32_t* hist, uint32_t need, uint32_t* u) {
    if (threadIdx.x < 64) {
        const uint32_t t = threadIdx.x;
        uint32_t c[4], loc = 0;
#pragma unroll
        for (int q = 0; q < 4; q++) { c[q] = hist[255u - 4u * t - (uint32_t)q]; loc += c[q]; }
        const uint32_t inc = wave_incl_scan_u(loc);
        uint32_t before = inc - loc;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if (before < need && need <= before + c[q]) { u[0] = 255u - 4u * t - (uint32_t)q; u[1] = need - before; }
            before += c[q];
        }
    }
    __syncthreads();
}

// One workgroup a row: the maximum, the sum, then a radix selection of the
// K-th key over passes of the row.
template <int DT, bool MASK>
__global__ __launch_bounds__(HR_NT) void zs_k_head_row(hd_args a, uint64_t r0) {
    constexpr int E = hd_elem<DT>::E, NW = HR_NT / 64;
    __shared__ unsigned long long list[HD_KMAX];
    __shared__ uint32_t hist[256], u[4], shu[NW];
    __shared__ float shf[NW];
    __shared__ double shd[NW];
    const uint64_t r = r0 + blockIdx.x;
    if (!hd_live(a, r)) return;
    const hd_row<DT> row(a.logits, a.ld, r, a.V);
    const uint32_t* allow = MASK ? a.allow + r * a.allow_words : nullptr;
    const uint32_t t = threadIdx.x;
    auto values = [&](uint32_t j, float (&x)[E]) {
        row.get(j, x, -INFINITY);
        uint32_t b = ~0u;
        if (MASK) b = hd_allow<E>(allow, a.allow_words, row.id0(j));
#pragma unroll
        for (int q = 0; q < E; q++) x[q] = (b >> q & 1u) ? hd_clean(x[q]) : -INFINITY;
    };
    float x[E], m = -INFINITY;
    for (uint32_t j = t; j < row.nvec; j += HR_NT) {
        values(j, x);
#pragma unroll
        for (int q = 0; q < E; q++) m = fmaxf(m, x[q]);
    }
    m = block_max_f<HR_NT>(m, shf);
    const float mr = m > -INFINITY ? m : 0.0f;
    float s = 0.0f;
    for (uint32_t j = t; j < row.nvec; j += HR_NT) {
        values(j, x);
#pragma unroll
        for (int q = 0; q < E; q++) x[q] = __builtin_amdgcn_exp2f((x[q] - mr) * a.c);
        s += hd_sum(x);
    }
    const double sum = block_sum_d<HR_NT>((double)s, shd);
    const double lse = hd_lse(mr, a.inv_t, sum);
    // the K-th key: its digits from the top, `need` of the keys equal so far
    uint32_t mask = 0, key = 0, need = a.K, all = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (t < 256) hist[t] = 0;
        __syncthreads();
        for (uint32_t j = t; j < row.nvec; j += HR_NT) {
            values(j, x);
#pragma unroll
            for (int q = 0; q < E; q++) {
                const uint32_t k = hd_key(x[q]);
                if (k && (k & mask) == key) atomicAdd(&hist[k >> shift & 255u], 1u);
            }
        }
        __syncthreads();
        if (shift == 24) {
            all = block_sum_u<HR_NT>(t < 256 ? hist[t] : 0u, shu);
            if (all <= a.K) break;
        }
        hr_digit<HR_NT>(hist, need, u);
        key |= u[0] << shift;
        mask |= 0xffu << shift;
        need = u[1];
        __syncthreads();
    }
    // those above it in any order, those equal to it by id
    if (t == 0) u[2] = 0;
    const bool every = all <= a.K;
    uint32_t taken = 0;
    __syncthreads();
    for (uint32_t j0 = 0; j0 < row.nvec; j0 += HR_NT) {
        const uint32_t j = j0 + t;
        uint32_t k[E], n = 0;
        if (j < row.nvec) {
            values(j, x);
#pragma unroll
            for (int q = 0; q < E; q++) { k[q] = hd_key(x[q]); n += !every && k[q] == key ? 1u : 0u; }
        } else {
#pragma unroll
            for (int q = 0; q < E; q++) k[q] = 0u;
        }
        uint32_t tot = 0, at = 0;
        if (!every) at = taken + block_excl_scan_u<HR_NT>(n, shu, &tot);
        taken += tot;
#pragma unroll
        for (int q = 0; q < E; q++) {
            const bool tie = !every && k[q] == key;
            if (tie ? at < need : every ? k[q] != 0u : k[q] > key)
                list[atomicAdd(&u[2], 1u)] = ((unsigned long long)(~k[q]) << 32) | (uint32_t)(row.id0(j) + q);
            at += tie ? 1u : 0u;
        }
    }
    __syncthreads();
    const uint32_t n = u[2];
    uint32_t np2 = 64;
    while (np2 < n) np2 <<= 1;
    if (t >= n && t < np2) list[t] = ~0ull;
    __syncthreads();
    block_bitonic_u64<HR_NT>(list, (int)np2);
    hd_put(a, r, t, t < n ? list[t] : ~0ull, lse);
}

int hd_head_launch(const hd_args& a, uint32_t dtype, hipStream_t stream) {
    for (uint64_t r0 = 0; r0 < a.R; r0 += HD_ROWS) {
        const dim3 grid((uint32_t)(a.R - r0 < HD_ROWS ? a.R - r0 : HD_ROWS));
#define HR_GO(DT)                                                                                                    \
    if (a.allow) hipLaunchKernelGGL((zs_k_head_row<DT, true>), grid, dim3(HR_NT), 0, stream, a, r0);                 \
    else hipLaunchKernelGGL((zs_k_head_row<DT, false>), grid, dim3(HR_NT), 0, stream, a, r0)
        if (dtype == ZS_F32) { HR_GO(ZS_F32); }
        else if (dtype == ZS_F16) { HR_GO(ZS_F16); }
        else { HR_GO(ZS_BF16); }
#undef HR_GO
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
