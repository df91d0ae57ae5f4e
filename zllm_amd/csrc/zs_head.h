// zs_head.h -- rows of logits in any of the three types, from any element on:
// what beam search (zs_beam.hip), the teacher's lists (zs_head.hip) and
// distillation (zs_distill.hip) read rows through.
#pragma once
#include <hip/hip_runtime.h>
#include "zs_internal.h"
#include "zs_dev.h"
#include "zs_head_args.h"

// A row is read as 16-byte vectors of E elements. It may start at any element
// of its type: vectors are counted from the 16-byte boundary at or below the
// row's first element, and the ids of vector j are j * E - shift + q. Only the
// first and the last vector can hold ids outside the row; those two are read
// element by element, so that nothing outside the row is touched.
typedef uint32_t hd_u4 __attribute__((ext_vector_type(4)));
template <int DT> struct hd_elem;
template <> struct hd_elem<ZS_F32> { typedef float T; static constexpr int E = 4; };
template <> struct hd_elem<ZS_F16> { typedef _Float16 T; static constexpr int E = 8; };
template <> struct hd_elem<ZS_BF16> { typedef uint16_t T; static constexpr int E = 8; };

__device__ __forceinline__ float hd_float(float v) { return v; }
__device__ __forceinline__ float hd_float(_Float16 v) { return (float)v; }
__device__ __forceinline__ float hd_float(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }

template <int DT>
__device__ __forceinline__ void hd_unpack(const hd_u4& v, float (&x)[hd_elem<DT>::E]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (DT == ZS_F32) {
            x[i] = __uint_as_float(w[i]);
        } else if constexpr (DT == ZS_BF16) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            typedef _Float16 h2 __attribute__((ext_vector_type(2)));
            const h2 h = __builtin_bit_cast(h2, w[i]);
            x[2 * i] = (float)h[0];
            x[2 * i + 1] = (float)h[1];
        }
    }
}
// Rounded to nearest even; what the type cannot hold becomes infinite.
template <int DT>
__device__ __forceinline__ uint32_t hd_pack2(float a, float b) {
    if constexpr (DT == ZS_BF16) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        const b2 v = {(__bf16)a, (__bf16)b};
        return __builtin_bit_cast(uint32_t, v);
    } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const h2 v = {(_Float16)a, (_Float16)b};
        return __builtin_bit_cast(uint32_t, v);
    }
}

template <int DT>
struct hd_row {
    typedef typename hd_elem<DT>::T T;
    static constexpr int E = hd_elem<DT>::E;
    const T* row;
    uint32_t shift, V, nvec;
    __device__ __forceinline__ hd_row(const void* base, uint64_t ld, uint64_t r, uint32_t V_) {
        row = reinterpret_cast<const T*>(base) + r * ld;
        V = V_;
        shift = (uint32_t)((uintptr_t)row & 15u) / (uint32_t)sizeof(T);
        nvec = (V + shift + E - 1u) / E;
    }
    __device__ __forceinline__ int id0(uint32_t j) const { return (int)(j * E) - (int)shift; }
    __device__ __forceinline__ bool inside(uint32_t j) const { const int i = id0(j); return i >= 0 && (uint32_t)i + E <= V; }
    __device__ __forceinline__ hd_u4 load(uint32_t j) const { return zs_gload(reinterpret_cast<const hd_u4*>(row + id0(j))); }
    // one that is not read again (7.2 TB/s of a large read where plain loads reach 6.5)
    __device__ __forceinline__ hd_u4 once(uint32_t j) const {
        return __builtin_nontemporal_load((const __attribute__((address_space(1))) hd_u4*)(row + id0(j)));
    }
    // the vector as it stands, -inf where it has no id of the row
    __device__ __forceinline__ hd_u4 raw(uint32_t j) const {
        if (inside(j)) return load(j);
        uint32_t w[4];
        const int i = id0(j);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if constexpr (DT == ZS_F32) {
                w[k] = (uint32_t)(i + k) < V ? __float_as_uint(row[i + k]) : 0xff800000u;
            } else {
                constexpr uint32_t none = DT == ZS_F16 ? 0xfc00u : 0xff80u;
                const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
                const uint32_t lo = (uint32_t)(i + 2 * k) < V ? p[i + 2 * k] : none;
                const uint32_t hi = (uint32_t)(i + 2 * k + 1) < V ? p[i + 2 * k + 1] : none;
                w[k] = lo | hi << 16;
            }
        }
        const hd_u4 v = {w[0], w[1], w[2], w[3]};
        return v;
    }
    __device__ __forceinline__ float at(uint32_t id) const { return hd_float(zs_gload(row + id)); }
    // a vector of no ids
    static __device__ __forceinline__ hd_u4 none() {
        constexpr uint32_t w = DT == ZS_F32 ? 0xff800000u : DT == ZS_F16 ? 0xfc00fc00u : 0xff80ff80u;
        const hd_u4 v = {w, w, w, w};
        return v;
    }
    // vectors j, j + step, ... of a workgroup, -inf where they have no id of
    // the row; the loads are in flight together
    template <int U>
    __device__ __forceinline__ void take(uint32_t j, uint32_t step, bool whole, hd_u4 (&v)[U]) const {
        if (whole) {
#pragma unroll
            for (int u = 0; u < U; u++) v[u] = once(j + (uint32_t)u * step);
            return;
        }
        // whole vectors lo .. hi, if any, and those before and behind them
        const uint32_t lo = shift ? 1u : 0u, hi = (V + shift) / E;   // (hi: one behind)
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t i = j + (uint32_t)u * step;
            v[u] = none();
            if (i >= lo && i < hi) v[u] = once(i);
        }
        if (lo > 0u && j == 0u) v[0] = raw(0);
        if (hi + 1u == nvec && hi >= lo && (nvec - 1u - j) % step == 0u && nvec - 1u >= j) {
            const hd_u4 w = raw(nvec - 1u);
#pragma unroll
            for (int u = 0; u < U; u++) v[u] = j + (uint32_t)u * step == nvec - 1u ? w : v[u];
        }
    }
    // the vector's values; `none` where it has no id of the row
    __device__ __forceinline__ void get(uint32_t j, float (&x)[E], float none) const {
        if (inside(j)) {
            hd_unpack<DT>(load(j), x);
            return;
        }
        const int i = id0(j);
#pragma unroll
        for (int q = 0; q < E; q++) x[q] = i + q >= 0 && (uint32_t)(i + q) < V ? at((uint32_t)(i + q)) : none;
    }
};

// The allow bits of ids i .. i + E - 1 (bit q: id i + q); i may be negative
// and past V, where the bits are unspecified (such ids are no ids of the row).
template <int E>
__device__ __forceinline__ uint32_t hd_allow(const uint32_t* words, uint32_t nwords, int i) {
    const uint32_t p = (uint32_t)max(i, 0), w = p >> 5, s = p & 31u;
    if (w >= nwords) return 0u;
    uint64_t two = zs_gload(words + w);
    if (s + E > 32u && w + 1u < nwords) two |= (uint64_t)zs_gload(words + w + 1u) << 32;
    const uint32_t b = (uint32_t)(two >> s);
    return i < 0 ? b << (uint32_t)(-i) : b;
}

// The sum of E values as a tree: a running sum that holds the largest term
// takes one rounding per vector, not one per value (rows whose first value
// has most of the mass lost 5e-7 of their sum to a chain of 300 values).
template <int E>
__device__ __forceinline__ float hd_sum(const float (&e)[E]) {
    if constexpr (E == 4) return (e[0] + e[1]) + (e[2] + e[3]);
    else return ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
}

// The factor of the exponent for values of at most m: c, as long as the rounding
// of m c stays below 64 and 2^ it a float. Past that the next float below m lies
// at least 2^6 / c under it, so that every value but m itself has no mass, and
// with a power of two that takes m to 2^125 (or as far as there is one) neither
// has its next value, and m's own product is exact.
__device__ __forceinline__ float hd_factor(float m, float c) {
    const uint32_t e = __float_as_uint(m) >> 23 & 255u;
    return fabsf(m * c) < 0x1p31f ? c : __uint_as_float(min(379u - e, 254u) << 23);
}

// A value as the heads of rows see it: NaN counts as -inf (nothing is known of
// it), +inf as the largest number (an id that is certain; several share).
__device__ __forceinline__ float hd_clean(float x) { return fminf(x == x ? x : -INFINITY, __FLT_MAX__); }
// Order of the candidates: a larger key is a larger value, -0 and +0 are one
// value; 0 is no candidate (-inf).
__device__ __forceinline__ uint32_t hd_key(float x) { return x > -INFINITY ? zs_total_key(x + 0.0f) : 0u; }

#define HD_LOG2E 1.44269504088896340736

// A row's normaliser: its maximum m and lns = ln sum exp((x - m) / T), -inf for
// no mass. Kept apart: their sum would lose lns where m is large (a row that
// is all at a mask's 1e30 has probabilities of 1 / V, not of 1).
struct hd_norm {
    double m, lns;
};

// Is row r's head wanted?
__device__ __forceinline__ bool hd_live(const hd_args& a, uint64_t r) {
    return !a.scores || (!a.done[zs_quot((uint32_t)r, a.by_width)] && fabsf(a.scores[r]) <= __FLT_MAX__);   // (beams' rows number below 2^31)
}
// Place t of row r, e = ~key << 32 | id (~0: none), for every t < K, and for 0
// and 1 whatever K is: the normaliser's halves go out with them.
__device__ __forceinline__ void hd_put(const hd_args& a, uint64_t r, uint32_t t, unsigned long long e, hd_norm o) {
    const bool some = e != ~0ull;
    const float x = zs_key_to_float(~(uint32_t)(e >> 32));
    if (a.ids) {
        if (t >= a.K) return;
        a.ids[r * a.K + t] = some ? (uint32_t)e : 0xffffffffu;
        a.logp[r * a.K + t] = some ? (float)(((double)x - o.m) * a.inv_t - o.lns) : -INFINITY;
        if (t == 0) a.lse_out[r] = o.lns > -INFINITY ? (float)(o.m * a.inv_t + o.lns) : -INFINITY;
    } else {
        // (past the L2, which other parts of the GPU do not share)
        if (t < a.K)
            __hip_atomic_store(a.list + r * a.K + t, some ? ((unsigned long long)zs_f2u(x) << 32) | (uint32_t)e : ~0ull,
                               __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (t < 2) __hip_atomic_store(a.norm + r * 2u + t, t ? o.lns : o.m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}
