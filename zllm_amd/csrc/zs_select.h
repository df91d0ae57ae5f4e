// zs_select.h -- the first K of the keys that a workgroup holds in registers.
#pragma once
#include "zs_dev.h"

// Of the workgroup's E * NT places (t, t + NT, ...: bit e), the first K
// by (key desc, place asc); places of key 0 are none. Radix selection of the
// K-th key over the digits in which the keys differ, then the places at it in
// order. Called by every thread; hist: 256 words, u: 4 words.
template <int NT, int E>
__device__ __forceinline__ uint32_t zs_first(const uint32_t (&k)[E], uint32_t K, uint32_t* hist, uint32_t* u) {
    constexpr uint32_t NW = NT / 64;
    static_assert(3 * NW <= 256 && E * NW <= 256 && NT == 256, "one histogram holds the counts");
    const uint32_t t = threadIdx.x, lane = (uint32_t)zs_lane(), wid = (uint32_t)zs_wid();
    uint32_t lo = ~0u, hi = 0, n = 0, all = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        if (!k[e]) continue;
        lo = min(lo, k[e]);
        hi = max(hi, k[e]);
        n++;
        all |= 1u << e;
    }
    lo = zs_wave_reduce(lo, [](uint32_t x, uint32_t y) { return min(x, y); });
    hi = zs_wave_reduce(hi, [](uint32_t x, uint32_t y) { return max(x, y); });
    n = wave_sum_u(n);
    if (lane == 0) { hist[wid] = lo; hist[NW + wid] = hi; hist[2 * NW + wid] = n; }
    __syncthreads();
    n = 0;
#pragma unroll
    for (uint32_t w = 0; w < NW; w++) {
        lo = min(lo, hist[w]);
        hi = max(hi, hist[NW + w]);
        n += hist[2 * NW + w];
    }
    __syncthreads();
    if (n <= K) return all;
    // key: the K-th once its digits are known; those above the first in which
    // the keys differ are hi's
    int shift = lo != hi ? (31 - __clz((int)(lo ^ hi))) & ~7 : -8;
    uint32_t mask = shift < 0 ? ~0u : shift == 24 ? 0u : ~0u << (shift + 8);
    uint32_t key = hi & mask, need = K;
    for (; shift >= 0; shift -= 8) {
        hist[t] = 0;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; e++)
            if (k[e] && (k[e] & mask) == key) atomicAdd(&hist[(k[e] >> shift) & 255u], 1u);
        __syncthreads();
        if (t < 64) {
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
        key |= u[0] << shift;
        mask |= 0xffu << shift;
        need = u[1];
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
        const uint32_t c = (uint32_t)__popcll(__ballot(k[e] == key));
        if (lane == 0) hist[(uint32_t)e * NW + wid] = c;
    }
    __syncthreads();
    uint32_t run = 0, first = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const unsigned long long m = __ballot(k[e] == key);
        uint32_t before = run;
#pragma unroll
        for (uint32_t w = 0; w < NW; w++) {
            const uint32_t c = hist[(uint32_t)e * NW + w];
            before += w < wid ? c : 0u;
            run += c;
        }
        before = __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, before));
        if (k[e] > key || (k[e] == key && before < need)) first |= 1u << e;
    }
    __syncthreads();
    return first;
}
