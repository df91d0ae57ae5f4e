// zs_ce.hip -- cross entropy of the vocabulary head from hidden states, and its
// gradient, without the logits.
#include <hip/hip_runtime.h>
#include "zs_ce.h"
#include "zs_head.h"

#define CE_NT 256
#define CE_SELF 256u   // rows up to which a workgroup goes through all labels by itself

// e^x for x <= 0. The rounding of x log2(e) alone is 2^-24 x of the result, 1e-6 at
// the -15 of an ordinary tail: nothing beside 16-bit gradients, but of an f32
// gradient's error the most, which so takes what the product leaves too.
__device__ __forceinline__ float ce_exp2(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_exp2f(x);
#else
    return x;
#endif
}
template <int DT>
__device__ __forceinline__ float ce_exp(float x) {
    constexpr float L = 1.44269504f, L1 = 1.92596299e-8f;   // log2(e) and what f32 leaves of it
    const float y = x * L, e = ce_exp2(y);
    if constexpr (DT != ZS_F32) return e;
    const float r = __builtin_fmaf(x, L1, __builtin_fmaf(x, L, -y));
    return x > -100.0f ? __builtin_fmaf(e, r * 0.69314718f, e) : e;   // (r is no number at -inf)
}
// The power of two that brings the piece's gradients of logits to at most 2^15:
// f16 has few exponents (row weights of 1 / N alone would leave most of a row
// below its normal numbers). The other types need none.
template <int DT>
__device__ __forceinline__ int ce_shift(const ce_args& a) {
    if constexpr (DT != ZS_F16) return 0;
    const uint32_t m = zs_wave_reduce(a.st->amax[zs_lane()], [](uint32_t x, uint32_t y) { return max(x, y); });
    if (m == 0u) return 0;
    const int s = 15 - ((int)(m >> 23) - 126);
    return s > 100 ? 100 : s;
}
__device__ __forceinline__ uint32_t ce_rows(const ce_args& a) {   // of the piece that have a label
    const uint32_t n = a.st->rows;
    return n <= a.lo ? 0u : n - a.lo < a.R ? n - a.lo : a.R;
}
__device__ __forceinline__ uint32_t ce_sub(const ce_args& a, uint32_t id) { return id >> (31 - __builtin_clz(a.sub)); }   // the part that has it
template <int DT>
__device__ __forceinline__ float ce_load(const void* p, uint64_t i) {
    return hd_float(reinterpret_cast<const typename hd_elem<DT>::T*>(p)[i]);
}
// four values to out + at, those before `end`
template <int DT>
__device__ __forceinline__ void ce_store4(void* out, uint64_t at, const float (&v)[4], uint32_t n, bool vec) {
    if constexpr (DT == ZS_F32) {
        float* o = (float*)out + at;
        if (vec) *(float4*)o = make_float4(v[0], v[1], v[2], v[3]);
        else
            for (uint32_t i = 0; i < 4u; i++)
                if (i < n) o[i] = v[i];
    } else {
        uint16_t* o = (uint16_t*)out + at;
        const uint2 u = make_uint2(hd_pack2<DT>(v[0], v[1]), hd_pack2<DT>(v[2], v[3]));
        if (vec) *(uint2*)o = u;
        else {
            const uint16_t s[4] = {(uint16_t)u.x, (uint16_t)(u.x >> 16), (uint16_t)u.y, (uint16_t)(u.y >> 16)};
            for (uint32_t i = 0; i < 4u; i++)
                if (i < n) o[i] = s[i];
        }
    }
}
template <int DT>
__device__ __forceinline__ void ce_zero(void* row, uint32_t n) {
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        if constexpr (DT == ZS_F32) ((float*)row)[i] = 0.0f;
        else ((uint16_t*)row)[i] = 0;
    }
}

// The rows with a label in order, behind them the others from the end on.
__global__ __launch_bounds__(1024) void zs_k_ce_rows(ce_args a) {
    __shared__ uint32_t sh[16];
    const uint32_t t = threadIdx.x, w = t >> 6, l = t & 63u;
    uint32_t done = 0;
    for (uint64_t r0 = 0; r0 < a.N; r0 += 1024u) {
        const uint64_t r = r0 + t;
        const bool in = r < a.N, has = in && a.labels[r] != a.ignore;
        const uint64_t m = __ballot(has);
        if (l == 0u) sh[w] = (uint32_t)__popcll(m);
        __syncthreads();
        uint32_t before = done + (uint32_t)__popcll(m & ((1ull << l) - 1u)), all = 0;
        for (uint32_t i = 0; i < 16u; i++) {
            before += i < w ? sh[i] : 0u;
            all += sh[i];
        }
        if (has) a.idx[before] = (uint32_t)r;
        else if (in) a.idx[a.N - 1u - (uint32_t)(r - before)] = (uint32_t)r;
        done += all;
        __syncthreads();
    }
    if (t == 0u) a.st->rows = done;
}

// Row lo + i: its hidden state to the operand (zeros behind the last row), and its
// label; rows without one get their zeros.
template <int DT>
__global__ __launch_bounds__(CE_NT) void zs_k_ce_pack(ce_args a) {
    __shared__ float shf[CE_NT / 64];
    const uint32_t i = blockIdx.x, t = threadIdx.x;
    const uint64_t plane = (uint64_t)a.R * a.Dp;
    uint16_t* o = a.h + (uint64_t)i * a.Dp;
    if (i == 0u && t < 64u) a.st->amax[t] = 0u;
    uint32_t n, mine = 0;
    if (a.N <= CE_SELF) {
        // few rows: each workgroup finds out for itself which row is its own (a launch less)
        __shared__ uint32_t all, own;
        if (t < 64u) {
            uint32_t with = 0;
            for (uint32_t r0 = 0; r0 < a.N; r0 += 64u) {
                const uint32_t r = r0 + t;
                const bool has = r < a.N && a.labels[r] != a.ignore;
                const uint64_t m = __ballot(has);
                const uint32_t before = with + (uint32_t)__popcll(m & ((1ull << t) - 1u));
                if (r < a.N && (has ? before : a.N - 1u - (r - before)) == i) own = r;
                with += (uint32_t)__popcll(m);
            }
            if (t == 0u) all = with;
        }
        __syncthreads();
        n = all;
        mine = own;
        if (t == 0u && i < a.N) a.idx[i] = mine;
        if (t == 0u && i == 0u) a.st->rows = n;
    } else {
        n = ce_rows(a);
        if (a.lo + (uint64_t)i < a.N) mine = a.idx[a.lo + i];
    }
    if (i >= n) {
        if (i < (n + CE_TILE - 1u) / CE_TILE * CE_TILE) {
            if (a.h)
                for (int p = 0; p < (DT == ZS_F32 ? 3 : 1); p++) ce_zero<ZS_F16>(o + p * plane, a.Dp);
            if (DT == ZS_F32 && a.h2) {
                for (int p = 0; p < 2; p++) ce_zero<ZS_F16>(a.h2 + p * plane + (uint64_t)i * a.Dp, a.Dp);
                if (t == 0u) a.row[i].sh = 0;
            }
        }
        if (a.lo + (uint64_t)i < a.N) {
            const uint64_t r = mine;
            if (t == 0u) a.loss[r] = a.lse[r] = 0.0f;
            if (a.dh) ce_zero<DT>((char*)a.dh + r * a.ld_dh * (DT == ZS_F32 ? 4u : 2u), a.D);
        }
        return;
    }
    const uint64_t r = mine;
    const int64_t label = a.labels[r];
    const bool bad = label < 0 || label >= (int64_t)a.V;
    const uint64_t hr = r * a.ld_h;
    int sh2 = 0;
    if (DT == ZS_F32 && a.h2) {
        float top = 0.0f;
        for (uint32_t d = t; d < a.D; d += CE_NT) top = fmaxf(top, fabsf(ce_load<DT>(a.hidden, hr + d)));
        sh2 = zs_split2_of(block_max_f<CE_NT>(top, shf));
        if (t == 0u) a.row[i].sh = sh2;
    }
    const bool vec = DT != ZS_F32 && a.D % 8u == 0u && a.ld_h % 8u == 0u && ((uintptr_t)a.hidden & 15u) == 0u;
    if (vec)
        for (uint32_t d = t * 8u; d < a.Dp; d += CE_NT * 8u) {
            hd_u4 u = {0u, 0u, 0u, 0u};
            if (d < a.D) u = zs_gload((const hd_u4*)((const uint16_t*)a.hidden + hr + d));
            *(hd_u4*)(o + d) = u;
        }
    for (uint32_t d = vec ? a.Dp : t; d < a.Dp; d += CE_NT) {
        if constexpr (DT == ZS_F32) {
            const float x = d < a.D ? ce_load<DT>(a.hidden, hr + d) : 0.0f;
            uint16_t p[3], p2[2];
            if (a.h) {
                zs_split3(x, p);
                for (int k = 0; k < 3; k++) o[k * plane + d] = p[k];
            }
            if (!a.h2) continue;
            zs_split2(x, sh2, p2);
            for (int k = 0; k < 2; k++) a.h2[k * plane + (uint64_t)i * a.Dp + d] = p2[k];
        } else {
            o[d] = d < a.D ? ((const uint16_t*)a.hidden)[hr + d] : (uint16_t)0;
        }
    }
    if (t == 0u) a.row[i].label = bad ? ~0u : (uint32_t)label;
}

// An f32 weight as two planes, row by row (each by a wave): its largest number, by that
// the power of two that it is scaled by, and its numbers once more, from the caches.
// (One power for the whole weight would leave nothing of the others where one row has
// a number that bans it.) Bound by memory: 50257 x 896 in 67 us, 240 MB read, 180 written.
__global__ __launch_bounds__(CE_NT) void zs_k_ce_split(ce_args a) {
    typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));   // (a row may begin at any number)
    const uint64_t plane = (uint64_t)a.V * a.Dp;
    const uint32_t l = (uint32_t)zs_lane(), whole = a.D & ~3u;
    for (uint32_t v = blockIdx.x * (CE_NT / 64) + zs_wid(); v < a.Vp; v += gridDim.x * (CE_NT / 64)) {
        if (v >= a.V) {
            if (l == 0u) a.wsh[v] = 0;
            continue;
        }
        const float* row = (const float*)a.weight + v * a.ld_w;
        float top = 0.0f;
#pragma unroll 4
        for (uint32_t d = l * 4u; d < whole; d += 256u) {
            const f4 x = *(const f4*)(row + d);
            top = fmaxf(top, fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
        }
        if (whole + l < a.D) top = fmaxf(top, fabsf(row[whole + l]));
        top = wave_max_f(top);
        const int sw = top == 0.0f ? 141 : zs_split2_of(top);   // (a row of zeros: as the smallest, or its entry over it would be the largest)
        if (l == 0u) a.wsh[v] = sw;
        uint16_t* o = a.w + (uint64_t)v * a.Dp;
#pragma unroll 2
        for (uint32_t d = l * 8u; d < a.Dp; d += 512u) {
            uint16_t p[8][2];
            if (d + 8u <= a.D) {
                const f4 x = *(const f4*)(row + d), y = *(const f4*)(row + d + 4u);
#pragma unroll
                for (int k = 0; k < 4; k++) zs_split2(x[k], sw, p[k]), zs_split2(y[k], sw, p[k + 4]);
            } else {
#pragma unroll
                for (uint32_t k = 0; k < 8u; k++) zs_split2(d + k < a.D ? row[d + k] : 0.0f, sw, p[k]);
            }
#pragma unroll
            for (int q = 0; q < 2; q++) {
                hd_u4 u;
#pragma unroll
                for (int k = 0; k < 4; k++) u[k] = (uint32_t)p[2 * k][q] | (uint32_t)p[2 * k + 1][q] << 16;
                *(hd_u4*)(o + q * plane + d) = u;
            }
        }
    }
}
// A 16-bit weight in rows of Dp, where its own rows do not serve. A row may begin at
// any element.
template <int DT>
__global__ __launch_bounds__(CE_NT) void zs_k_ce_weight(ce_args a) {
    const uint32_t per = a.Dp / 8u;   // (at most 2^33 of them in all: the ids go over y where they are many)
    for (uint64_t v0 = (uint64_t)blockIdx.y * 65536u; v0 < a.V; v0 += (uint64_t)gridDim.y * 65536u) {
        const uint32_t ids = (uint32_t)(a.V - v0 < 65536u ? a.V - v0 : 65536u);
        for (uint32_t i = blockIdx.x * CE_NT + threadIdx.x; i < ids * per; i += gridDim.x * CE_NT) {
            const uint64_t v = v0 + i / per;
            const uint32_t j = i % per;
            const hd_row<DT> row(a.weight, a.ld_w, v, a.D);
            const uint32_t d0 = j * 8u;
            typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));   // (a row's eight values may lie anywhere)
            hd_u4 x;
            if (d0 + 8u <= a.D) {
                x = zs_gload((const u4*)(row.row + d0));
            } else {
                const uint16_t* r = (const uint16_t*)row.row;
#pragma unroll
                for (uint32_t k = 0; k < 4u; k++) {
                    const uint32_t d = d0 + 2u * k;
                    x[k] = (d < a.D ? (uint32_t)r[d] : 0u) | (d + 1u < a.D ? (uint32_t)r[d + 1u] << 16 : 0u);
                }
            }
            *(hd_u4*)(a.w + v * a.Dp + d0) = x;
        }
    }
}

template <int DT>
__device__ __forceinline__ tp_mat ce_mat_w(const ce_args& a, bool slow) {
    const bool own = a.w != nullptr;
    const uint16_t* p = own ? a.w : (const uint16_t*)a.weight;
    const uint64_t plane = (uint64_t)a.V * a.Dp;
    const uint32_t d = own ? a.Dp : a.D;
    tp_mat m = {{p, p + plane, p + 2 * plane}, own ? a.Dp : a.ld_w, slow ? d : a.V, slow ? a.V : d};
    return m;
}
__device__ __forceinline__ tp_mat ce_mat_raw(const ce_args& a, bool slow) {   // f32, as it lies
    tp_mat m = {{(const uint16_t*)a.weight}, a.ld_w, slow ? a.D : a.V, slow ? a.V : a.D};
    return m;
}
// (f32: the weight's gradient, whose rows of the other operands differ in size by any
// factor, by three planes each; the others by two)
template <int DT>
__device__ __forceinline__ tp_mat ce_mat_h(const ce_args& a, bool slow) {
    const uint64_t plane = (uint64_t)a.R * a.Dp;
    const uint16_t* p = DT == ZS_F32 && !slow && !a.raw ? a.h2 : a.h;
    tp_mat m = {{p, p + plane, p + 2 * plane}, a.Dp, slow ? a.Dp : ce_rows(a), slow ? a.R : a.Dp};
    return m;
}
template <int DT>
__device__ __forceinline__ tp_mat ce_mat_dl(const ce_args& a, bool slow) {
    const uint64_t plane = (uint64_t)a.R * a.Vp;
    const uint16_t* p = DT == ZS_F32 && !slow && !a.raw ? a.dl2 : a.dl;
    tp_mat m = {{p, p + plane, p + 2 * plane}, a.Vp, slow ? a.Vp : ce_rows(a), slow ? a.R : a.Vp};
    return m;
}

// The tiles of the products: 256 x 256, or 128 x 64 where there are few rows.
// The logits' gradient d in 16 bits is off by half a step of the type. Over many rows
// and ids that adds 0.7 of the outputs' own rounding to their error; in few rows, where
// one d is most of a gradient's row, it may be the double. There the products wait for
// memory, and what the rounding leaves is multiplied too.
constexpr int ce_kind(int dt, bool thin, bool weight) {
    return dt == ZS_F32 ? (weight ? TP_THREE : TP_TWO) : !thin ? dt : dt == ZS_F16 ? TP_REST_F16 : TP_REST_BF16;
}
template <int KIND, bool THIN, bool AS, bool BS>
using ce_tile = tp_tile<KIND, THIN ? 1 : 4, THIN ? 2 : 4, THIN ? 4 : 2, AS, BS>;
template <int RAW, class T, bool SLOW> struct ce_or_raw { typedef tp_raw_tile<SLOW, RAW == 2> type; };
template <class T, bool SLOW> struct ce_or_raw<0, T, SLOW> { typedef T type; };
template <int MT, int NT>
__device__ __forceinline__ void ce_none(tp_acc (&c)[MT][NT]) {
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int q = 0; q < 16; q++) c[i][j][q] = 0.0f;
}
__device__ __forceinline__ uint32_t ce_over(uint32_t n, uint32_t d) { return (n + d - 1u) / d; }

// Logits of a tile of ids (m) and rows (n), of which only what a softmax over the
// vocabulary needs leaves the registers: per row and wave (128 ids, or 32) their
// maximum and the sum of exponentials relative to it, for the gradient the
// exponentials, and of the block of ids that has the row's label the logits.
// Bound by the matrix cores (4096 rows of 4096, 151936 ids, bf16: 4151 us, 1228
// TFLOP/s, 70 % of the clocks), with the exponentials behind each tile's products;
// few rows by the weight's bytes (5 rows of 1024, 32000 ids: 12.7 us, 5.2 TB/s).
template <int DT, bool GRAD, bool THIN, int RAW>
__global__ __launch_bounds__(CE_NT, 1) void zs_k_ce_logits(ce_args a) {
    typedef typename ce_or_raw<RAW, ce_tile<DT == ZS_F32 ? TP_TWO : DT, THIN, false, false>, false>::type T;
    constexpr int MT = T::M, NT = T::N;
    const uint32_t n = ce_rows(a), mt = a.Vp / T::BM, nt = ce_over(n, T::BN), t = tp_place(blockIdx.x, mt * nt);
    if (t == ~0u) return;
    const uint2 at = tp_order(t, mt, nt);
    const tp_mat mw = RAW ? ce_mat_raw(a, false) : ce_mat_w<DT>(a, false), mh = ce_mat_h<DT>(a, false);
    T tile(mw, mh, at.x, at.y);
    tp_acc c[MT][NT];
    ce_none(c);
    const uint32_t block = tile.m0 + T::wm() * (32 * MT);
    uint32_t lab[NT], own = 0u;   // own, a bit for each j: the block has the row's label (found out beside the first loads)
#pragma unroll
    for (int j = 0; j < NT; j++) lab[j] = tile.n_of(j) < n ? a.row[tile.n_of(j)].label : ~0u;
    tile.run(0, a.Dp / TP_KSTEP, c, [&] {
#pragma unroll
        for (int j = 0; j < NT; j++) own |= lab[j] - block < 32u * MT ? 1u << j : 0u;
    });
    if constexpr (DT == ZS_F32 && !RAW) {
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int4 w = *(const int4*)(a.wsh + tile.m_of(i, q));
                const int sw[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    const int back = -a.row[tile.n_of(j)].sh;
#pragma unroll
                    for (int k = 0; k < 4; k++) c[i][j][4 * q + k] = ldexpf(c[i][j][4 * q + k], back - sw[k]);
                }
            }
    }
    // The logits of the label's block, of which the row's loss and the block's gradient
    // are made: errors that the label's products have in common with the others' cancel
    // in the differences, and the others' exponentials, all there is of a certain row's
    // loss and of p - 1, are kept from the label's. (Values that go out, not a sum without
    // the label here: accumulators changed or read on a second way cost an evaluation of
    // 4100 us 70 to 230.)
#pragma unroll
    for (int j = 0; j < NT; j++)
        if (own >> j & 1u)
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const float v[4] = {c[i][j][4 * q], c[i][j][4 * q + 1], c[i][j][4 * q + 2], c[i][j][4 * q + 3]};
                    ce_store4<ZS_F32>(a.own, (uint64_t)tile.n_of(j) * (32 * MT) + (tile.m_of(i, q) - block), v, 4, true);
                }
    const uint32_t sub = at.x * (T::BM / (32 * MT)) + T::wm();
    constexpr bool LEAD = GRAD && DT == ZS_F32 && !RAW;
    // The largest exponential over its id's power of two, by which the gradient's planes
    // are scaled: 1 over the least of the block's powers, or half of that, where the others
    // are at most twice it (as of most weights); else (0) each is looked at, which for all
    // blocks took 118 us of 1024 rows' 1055 over 140910 x 869.
    float over = 0.0f;
    if constexpr (LEAD)
        if (a.lead) {
            uint32_t lo = ~0u, hi = 0u;
#pragma unroll
            for (uint32_t k = 0; k < 32u * MT; k += 64u) {
                const uint32_t id = block + k + (uint32_t)zs_lane() % (32u * MT);
                const uint32_t w = id < a.V ? (uint32_t)(a.wsh[id] + 1024) : ~0u;
                lo = min(lo, w);
                hi = max(hi, w == ~0u ? 0u : w);
            }
            lo = zs_wave_reduce(lo, [](uint32_t x, uint32_t y) { return min(x, y); });
            hi = zs_wave_reduce(hi, [](uint32_t x, uint32_t y) { return max(x, y); });
            if (hi <= lo + 1u && lo != ~0u) over = ldexpf(1.0f, 1024 - (int)lo);
        }
    if (tile.m0 + T::BM > a.V) {
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int q = 0; q < 16; q++)
                if (tile.m_of(i, q / 4) + (uint32_t)(q & 3) >= a.V)
#pragma unroll
                    for (int j = 0; j < NT; j++) c[i][j][q] = -INFINITY;
    }
    float m, s;
    auto largest = [&](int j) {
        m = -INFINITY;
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int q = 0; q < 16; q++) m = fmaxf(m, c[i][j][q]);
        m = fmaxf(m, zs_lane_xor<32>(m));
    };
    auto part = [&](int j, float unit) {
        s += zs_lane_xor<32>(s);
        if (zs_lane() < 32) a.stat[(uint64_t)tile.n_of(j) * a.subs + sub] = make_float2(m, s * unit);
    };
    if constexpr (GRAD && DT != ZS_F32) {
        uint16_t* e = (uint16_t*)a.e + (uint64_t)(tile.n0 + T::wn() * (32 * NT)) * a.Vp + tile.m0 + T::wm() * (32 * MT);
        tile.rows(
            largest,
            [&](int i, int j, int q) {
                const float m0 = m > -INFINITY ? m : 0.0f;
                float x[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    x[k] = ce_exp2(__builtin_fmaf(c[i][j][4 * q + k] - m0, 1.44269504f, CE_E_SHIFT));
                    s += x[k];
                }
                return make_uint2(hd_pack2<ZS_F16>(x[0], x[1]), hd_pack2<ZS_F16>(x[2], x[3]));
            },
            [&](int j) { part(j, 1.0f / CE_E_SCALE); }, [&](uint32_t r, uint32_t v, hd_u4 x) { *(hd_u4*)(e + (uint64_t)r * a.Vp + v) = x; });
    } else {
#pragma unroll
        for (int j = 0; j < NT; j++) {
            largest(j);
            const float m0 = m > -INFINITY ? m : 0.0f;
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    float x[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        x[k] = ce_exp<DT>(c[i][j][4 * q + k] - m0);
                        s += x[k];
                    }
                    if constexpr (GRAD) ce_store4<ZS_F32>(a.e, (uint64_t)tile.n_of(j) * a.Vp + tile.m_of(i, q), x, 4, true);
                }
            part(j, 1.0f);
            if constexpr (LEAD)
                if (a.lead) {
                    float lead = m > -INFINITY ? over : 0.0f;
                    if (over == 0.0f) {
#pragma unroll
                        for (int i = 0; i < MT; i++)
#pragma unroll
                            for (int q = 0; q < 4; q++) {
                                const int4 w = *(const int4*)(a.wsh + tile.m_of(i, q));
                                const int sw[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                                for (int k = 0; k < 4; k++) lead = fmaxf(lead, ldexpf(ce_exp<DT>(c[i][j][4 * q + k] - m0), -sw[k]));
                            }
                        lead = fmaxf(lead, zs_lane_xor<32>(lead));
                    }
                    if (zs_lane() < 32) a.lead[(uint64_t)tile.n_of(j) * a.subs + sub] = lead;
                }
        }
    }
}

// A row's normaliser and loss from its parts, and what its gradient goes by. With m
// the row's largest logit, rest the others' exponentials relative to it and s = rest
// + exp(z_label - m), 1 - p is rest / s and the loss ln s - (z_label - m), of two numbers
// that are not negative: nothing cancels.
template <int DT, bool GRAD>
__global__ __launch_bounds__(CE_NT) void zs_k_ce_loss(ce_args a) {
    __shared__ float shf[CE_NT / 64], at_;
    __shared__ double shd[CE_NT / 64];
    const uint32_t i = blockIdx.x, t = threadIdx.x;
    if (i >= ce_rows(a)) return;
    const float2* st = a.stat + (uint64_t)i * a.subs;
    const float y = t < a.sub ? a.own[(uint64_t)i * a.sub + t] : 0.0f;
    const uint32_t label = a.row[i].label, own = ce_sub(a, label), id = own * a.sub + t;
    const bool none = label == ~0u;   // (outside the vocabulary: it has no block)
    const bool in = !none && t < a.sub && id < a.V;
    if (t == (none ? 0u : (label & (a.sub - 1u)))) at_ = none ? -INFINITY : y;
    float m = in ? y : -INFINITY;
    for (uint32_t k = t; k < a.subs; k += CE_NT)
        if (k != own) m = fmaxf(m, st[k].x);
    m = block_max_f<CE_NT>(m, shf);
    const float m0 = m > -INFINITY ? m : 0.0f;
    const float at = at_;   // (written in front of the maximum's barriers)
    double rest = in && id != label ? (double)ce_exp<ZS_F32>(y - m0) : 0.0;
    for (uint32_t k = t; k < a.subs; k += CE_NT) {
        const float2 v = st[k];
        if (k != own) rest += (double)(v.y * ce_exp<DT>(v.x - m0));
    }
    rest = block_sum_d<CE_NT>(rest, shd);
    const double below = (double)at - (double)m0, e = DT == ZS_F32 ? exp(below) : (double)ce_exp<ZS_F32>(at - m0);
    const double s = rest + e, ln = log1p(below == 0.0 ? rest : s - 1.0), lse = (double)m0 + ln;
    const uint32_t r = a.idx[a.lo + i];
    if (t == 0u) {
        a.lse[r] = (float)lse;
        a.loss[r] = (float)((none ? NAN : ln - below) + (double)a.zw * lse * lse);
    }
    if constexpr (GRAD) {
        const float g = a.row_grad[r * a.row_grad_stride];
        const double k1 = 1.0 + 2.0 * (double)a.zw * lse, bad = none ? NAN : g;
        const float f = (float)(bad * k1 / s);
        float lead = 0.0f;   // (of the row's entries over their ids' powers of two, the largest)
        if (DT == ZS_F32 && a.lead) {
            if (in && id != label) lead = ldexpf(f * ce_exp<ZS_F32>(y - m0), -a.wsh[id]);
            lead = fabsf(lead);
            for (uint32_t k = t; k < a.subs; k += CE_NT)
                if (k != own) lead = fmaxf(lead, fabsf(f * ce_exp<DT>(st[k].x - m0)) * a.lead[(uint64_t)i * a.subs + k]);
            lead = block_max_f<CE_NT>(lead, shf);
        }
        for (uint32_t k = t; k < a.subs; k += CE_NT) a.fac[(uint64_t)i * a.subs + k] = f * ce_exp<DT>(st[k].x - m0);
        if (t == 0u) {
            // g (k1 p - 1) at the label, at most g k1 rest / s at the others
            const double others = k1 * (rest / s);
            const float fix = (float)(bad * (2.0 * (double)a.zw * lse - others));
            const float top = fmaxf(fabsf(fix), fabsf((float)((double)g * others)));
            a.row[i].fix = fix;
            a.row[i].fac = f;
            a.row[i].m = m0;
            if (DT == ZS_F32 && a.lead) a.row[i].sd = zs_split2_of(fmaxf(lead, none ? 0.0f : fabsf(ldexpf(fix, -a.wsh[label]))));
            if (DT == ZS_F16 && top < INFINITY) atomicMax(&a.st->amax[i & 63u], __float_as_uint(top));
        }
    }
}

// Exponentials (of the label's block the logits) to the gradient of the logits, in
// their place (f32: to three planes); zeros in the rows up to where the products over
// the rows end. Bound by memory: 8192 x 151936 in 795 us, 6.4 TB/s. (A pass of its own,
// as a row's sum is known only when all of its tiles are done.)
template <int DT>
__global__ __launch_bounds__(CE_NT) void zs_k_ce_grad(ce_args a) {
    const uint32_t i = blockIdx.y, n = ce_rows(a), v0 = (blockIdx.x * CE_NT + threadIdx.x) * 8u;
    const int sh = ce_shift<DT>(a);   // (by whole waves)
    if (i >= (n + TP_KSTEP - 1u) / TP_KSTEP * TP_KSTEP || v0 >= a.Vp) return;
    const uint64_t at = (uint64_t)i * a.Vp + v0;
    float x[8];
    if (i < n) {
        const ce_row row = a.row[i];
        if ((row.label ^ v0) < a.sub) {
            // the label's block, from its logits
            const float* z = a.own + (uint64_t)i * a.sub + (v0 & (a.sub - 1u));
            const float f = ldexpf(row.fac, sh), fix = ldexpf(row.fix, sh);
            const float4 u = *(const float4*)z, w = *(const float4*)(z + 4);
            const float y[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
            for (uint32_t k = 0; k < 8u; k++) x[k] = v0 + k >= a.V ? 0.0f : v0 + k == row.label ? fix : f * ce_exp<ZS_F32>(y[k] - row.m);
        } else {
            const float f = ldexpf(a.fac[(uint64_t)i * a.subs + ce_sub(a, v0)], sh) * (DT == ZS_F32 ? 1.0f : 1.0f / CE_E_SCALE);
            if constexpr (DT == ZS_F32) {
                const float4 u = *(const float4*)((const float*)a.e + at), w = *(const float4*)((const float*)a.e + at + 4);
                const float y[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
                for (int k = 0; k < 8; k++) x[k] = y[k] * f;
            } else {
                const hd_u4 u = *(const hd_u4*)((const uint16_t*)a.e + at);
                hd_unpack<ZS_F16>(u, x);
                for (int k = 0; k < 8; k++) x[k] *= f;
            }
        }
    } else {
        for (int k = 0; k < 8; k++) x[k] = 0.0f;
    }
    if constexpr (DT == ZS_F32) {
        const uint64_t plane = (uint64_t)a.R * a.Vp;
        if (a.dl) {
            uint16_t p[8][3];
            for (int k = 0; k < 8; k++) zs_split3(x[k], p[k]);
            for (int q = 0; q < 3; q++) {
                hd_u4 o;
                for (int k = 0; k < 4; k++) o[k] = (uint32_t)p[2 * k][q] | (uint32_t)p[2 * k + 1][q] << 16;
                *(hd_u4*)(a.dl + q * plane + at) = o;
            }
        }
        if (a.dl2) {
            uint16_t p[8][2];
            const int sd = i < n ? a.row[i].sd : 0;
            const int4 u = *(const int4*)(a.wsh + v0), w = *(const int4*)(a.wsh + v0 + 4);
            const int sw[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
            for (int k = 0; k < 8; k++) zs_split2(x[k], sd - sw[k], p[k]);
            for (int q = 0; q < 2; q++) {
                hd_u4 o;
                for (int k = 0; k < 4; k++) o[k] = (uint32_t)p[2 * k][q] | (uint32_t)p[2 * k + 1][q] << 16;
                *(hd_u4*)(a.dl2 + q * plane + at) = o;
            }
        }
    } else {
        hd_u4 o;
        for (int k = 0; k < 4; k++) o[k] = hd_pack2<DT>(x[2 * k], x[2 * k + 1]);
        *(hd_u4*)(a.dl + at) = o;
        if (a.thin) {
            float y[8];
            hd_unpack<DT>(o, y);
            for (int k = 0; k < 4; k++) o[k] = hd_pack2<DT>(x[2 * k] - y[2 * k], x[2 * k + 1] - y[2 * k + 1]);
            *(hd_u4*)(a.dl + (uint64_t)a.R * a.Vp + at) = o;
        }
    }
}

// A gradient's tile of 16-bit values, whole rows at a time: out[row(r)] for the
// wave's rows r, from column d0 on, columns before D. (Not read again here: stored
// past the caches, one row's step over 151936 x 4096 bf16 weights takes 1010 us for
// 1087, over 58134 x 3456 f32 ones 611 for 696. Rows at
// any element share their lines' ends and are left to the caches: 7 rows' step over
// 140910 x 869 f32 weights takes 664 past them, 590 so.)
template <int DT, class T, class P, class I>
__device__ __forceinline__ void ce_out(const T& tile, void* out, uint64_t ld, uint32_t D, uint32_t d0, const P& put, const I& row) {
    uint16_t* o = (uint16_t*)out;
    if (d0 >= D) return;
    typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));   // (a row may begin at any element)
    const auto none = [](int) {};
    if (D % 8u == 0u) {
        tile.rows(none, put, none, [&](uint32_t r, uint32_t m, hd_u4 v) {
            const uint64_t to = row(r);
            if (to != ~0ull && d0 + m < D) __builtin_nontemporal_store((u4)v, (u4*)(o + to * ld + d0 + m));
        });
    } else {
        tile.rows(none, put, none, [&](uint32_t r, uint32_t m, hd_u4 v) {
            const uint64_t to = row(r);
            if (to == ~0ull || d0 + m >= D) return;
            uint16_t* p = o + to * ld + d0 + m;
            if (d0 + m + 8u <= D) *(u4*)p = v;
            else
                for (uint32_t k = 0; k < D - d0 - m; k++) p[k] = (uint16_t)(v[k >> 1] >> (k & 1u) * 16u);
        });
    }
}

// Into how many parts of the vocabulary the products over it go, so that all CUs
// have work: with the rows that there are, which the host does not know.
struct ce_cut {
    uint32_t mt, nt, parts, steps;   // tiles; parts, of so many steps
};
template <class T>
__device__ __forceinline__ ce_cut ce_parts(const ce_args& a) {
    ce_cut p;
    const uint32_t all = a.Vp / TP_KSTEP;
    p.mt = ce_over(a.D, T::BM);
    p.nt = ce_over(ce_rows(a), T::BN);
    const uint32_t tiles = p.mt * p.nt;
    uint32_t s = tiles ? a.units / tiles : 1u;
    s = s < all / 16u ? s : all / 16u;
    s = s ? s : 1u;
    p.steps = (ce_over(all, s) + 3u) & ~3u;
    p.parts = ce_over(all, p.steps);
    return p;
}

// Gradient of the hidden states, a tile of columns (m) and rows (n), over the
// vocabulary or a part of it: 8192 x 4096 have 512 tiles, two rounds of the card's
// CUs, but 1024 rows of 1024 have 16, which without the cut would be all that works.
template <int DT, bool THIN, int RAW>
__global__ __launch_bounds__(CE_NT, 1) void zs_k_ce_dhidden(ce_args a) {
    typedef typename ce_or_raw<RAW, ce_tile<ce_kind(DT, THIN, false), THIN, true, false>, true>::type T;
    constexpr int MT = T::M, NT = T::N;
    const ce_cut p = ce_parts<T>(a);
    const uint32_t n = ce_rows(a), tiles = p.mt * p.nt, u = tp_place(blockIdx.x, tiles * p.parts);
    if (u == ~0u) return;
    const uint32_t part = u / tiles, k0 = part * p.steps, all = a.Vp / TP_KSTEP;
    const uint2 at = tp_order(u - part * tiles, p.mt, p.nt);
    const tp_mat mw = RAW ? ce_mat_raw(a, true) : ce_mat_w<DT>(a, true), md = ce_mat_dl<DT>(a, false);
    T tile(mw, md, at.x, at.y);
    tp_acc c[MT][NT];
    ce_none(c);
    tile.run(k0, all - k0 < p.steps ? all - k0 : p.steps, c);
    const float un = ldexpf(1.0f, -ce_shift<DT>(a));
    if constexpr (DT == ZS_F32 && !RAW) {
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const int back = -a.row[tile.n_of(j)].sd;   // (rows past the last are not stored; ids' powers are in both operands)
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int q = 0; q < 16; q++) c[i][j][q] = ldexpf(c[i][j][q], back);
        }
    }
    if (DT == ZS_F32 || p.parts > 1u) {
        const bool vec = a.D % 4u == 0u && a.ld_dh % 4u == 0u && ((uintptr_t)a.dh & 15u) == 0u;
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const uint32_t r = tile.n_of(j);
            if (r >= n) continue;
            const uint64_t row = p.parts > 1u ? 0u : a.idx[a.lo + r];
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const uint32_t d = tile.m_of(i, q);
                    if (d >= a.D) continue;
                    const float v[4] = {c[i][j][4 * q] * un, c[i][j][4 * q + 1] * un, c[i][j][4 * q + 2] * un, c[i][j][4 * q + 3] * un};
                    if (p.parts > 1u) ce_store4<ZS_F32>(a.part, ((uint64_t)part * (p.nt * T::BN) + r) * a.Dm + d, v, 4, true);
                    else ce_store4<DT>(a.dh, row * a.ld_dh + d, v, a.D - d, vec);
                }
        }
        return;
    }
    if constexpr (DT != ZS_F32) {
        const uint32_t r0 = tile.n0 + T::wn() * (32 * NT);
        ce_out<DT>(tile, a.dh, a.ld_dh, a.D, tile.m0 + T::wm() * (32 * MT),
                   [&](int i, int j, int q) {
                       return make_uint2(hd_pack2<DT>(c[i][j][4 * q] * un, c[i][j][4 * q + 1] * un),
                                         hd_pack2<DT>(c[i][j][4 * q + 2] * un, c[i][j][4 * q + 3] * un));
                   },
                   [&](uint32_t r) { return r0 + r < n ? (uint64_t)a.idx[a.lo + r0 + r] : ~0ull; });
    }
}
// The parts' sums, a row's 256 columns by 64 threads with four columns each, four
// times over the parts.
template <int DT, bool THIN>
__global__ __launch_bounds__(CE_NT) void zs_k_ce_join(ce_args a) {
    typedef ce_tile<ce_kind(DT, THIN, false), THIN, true, false> T;
    __shared__ float4 sh[3][64];
    const uint32_t l = threadIdx.x & 63u, w = threadIdx.x >> 6, d = (blockIdx.y * 64u + l) * 4u, n = ce_rows(a);
    const ce_cut p = ce_parts<T>(a);
    if (p.parts < 2u) return;
    const uint64_t step = (uint64_t)p.nt * T::BN * a.Dm;
    for (uint32_t i = blockIdx.x; i < n; i += gridDim.x) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (d < a.D) {
            const float* x = a.part + (uint64_t)i * a.Dm + d;
#pragma unroll 4
            for (uint32_t s = w; s < p.parts; s += 4u) {
                const float4 y = *(const float4*)(x + s * step);
                v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
            }
        }
        __syncthreads();   // (the row before is read)
        if (w > 0u) sh[w - 1u][l] = v;
        __syncthreads();
        if (w > 0u || d >= a.D) continue;
        for (int k = 0; k < 3; k++) {
            const float4 y = sh[k][l];
            v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
        }
        const float o[4] = {v.x, v.y, v.z, v.w};
        ce_store4<DT>(a.dh, (uint64_t)a.idx[a.lo + i] * a.ld_dh + d, o, a.D - d, a.D % 4u == 0u && a.ld_dh % 4u == 0u && ((uintptr_t)a.dh & 15u) == 0u);
    }
}

// Gradient of the weight, a tile of columns (m) of ids (n), over the piece's rows.
// (Of few rows there is little to multiply and much to write: three workgroups of
// 128 x 128 a CU. In f32 the planes' addresses, picked at run time, lie in private
// memory: over a few rows, where a plane ends every step or two, the products wait for
// them.) 151936 x 4096 over 8192 rows: 7344 us, 1388 TFLOP/s; over one f32 row, 58134 x
// 3456: 185 us, 4.3 TB/s written.
template <int DT, bool THIN>
__global__ __launch_bounds__(CE_NT, THIN ? 3 : 1) void zs_k_ce_dweight(ce_args a) {
    typedef tp_tile<ce_kind(DT, THIN, true), THIN ? 2 : 4, THIN ? 2 : 4, 2, true, true> T;
    const uint32_t n = ce_rows(a), mt = ce_over(a.D, T::BM), nt = a.Vp / T::BN, t = tp_place(blockIdx.x, mt * nt);
    if (t == ~0u) return;
    const uint2 at = tp_order(t, mt, nt);
    const tp_mat mh = ce_mat_h<DT>(a, true), md = ce_mat_dl<DT>(a, true);
    T tile(mh, md, at.x, at.y);
    tp_acc c[T::M][T::N];
    ce_none(c);
    tile.run(0, ce_over(n, TP_KSTEP), c);
    const float un = ldexpf(1.0f, -ce_shift<DT>(a));
    if constexpr (DT == ZS_F16) {
#pragma unroll
        for (int i = 0; i < T::M; i++)
#pragma unroll
            for (int j = 0; j < T::N; j++)
#pragma unroll
                for (int q = 0; q < 16; q++) c[i][j][q] *= un;
    }
    const bool vec = a.D % 4u == 0u && a.ld_dw % 4u == 0u && ((uintptr_t)a.dw & 15u) == 0u;
    if (!a.first || !a.last) {
#pragma unroll
        for (int j = 0; j < T::N; j++) {
            const uint32_t id = tile.n_of(j);
            if (id >= a.V) continue;
#pragma unroll
            for (int i = 0; i < T::M; i++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const uint32_t d = tile.m_of(i, q);
                    if (d >= a.D) continue;
                    float v[4] = {c[i][j][4 * q], c[i][j][4 * q + 1], c[i][j][4 * q + 2], c[i][j][4 * q + 3]};
                    float* acc = a.acc + (uint64_t)id * a.Dm + d;
                    if (!a.first) {
                        const float4 p = *(const float4*)acc;
                        v[0] += p.x, v[1] += p.y, v[2] += p.z, v[3] += p.w;
                    }
                    if (!a.last) ce_store4<ZS_F32>(acc, 0, v, 4, true);
                    else ce_store4<DT>(a.dw, (uint64_t)id * a.ld_dw + d, v, a.D - d, vec);
                }
        }
        return;
    }
    const uint32_t id0 = tile.n0 + T::wn() * (32 * T::N);
    if constexpr (DT == ZS_F32) {
        const uint32_t d0 = tile.m0 + T::wm() * (32 * T::M);
        if (d0 >= a.D) return;
        const auto get = [&](int i, int j, int q) { return make_float4(c[i][j][4 * q], c[i][j][4 * q + 1], c[i][j][4 * q + 2], c[i][j][4 * q + 3]); };
        const auto row = [&](uint32_t r) { return id0 + r < a.V ? (float*)a.dw + (uint64_t)(id0 + r) * a.ld_dw + d0 : (float*)nullptr; };
        if (vec) tile.template words<true>(get, row, a.D - d0);
        else tile.template words<false>(get, row, a.D - d0);
    } else {
        ce_out<DT>(tile, a.dw, a.ld_dw, a.D, tile.m0 + T::wm() * (32 * T::M),
                   [&](int i, int j, int q) {
                       return make_uint2(hd_pack2<DT>(c[i][j][4 * q], c[i][j][4 * q + 1]), hd_pack2<DT>(c[i][j][4 * q + 2], c[i][j][4 * q + 3]));
                   },
                   [&](uint32_t r) { return id0 + r < a.V ? (uint64_t)(id0 + r) : ~0ull; });
    }
}

template <int DT, bool THIN, int RAW>
static void ce_products(const ce_args& a, hipStream_t stream) {
    const dim3 wg(CE_NT);
    const uint32_t bm = THIN ? CE_THIN_M : CE_TILE, rt = THIN ? (a.N + CE_THIN - 1u) / CE_THIN : a.R / CE_TILE, vt = a.Vp / bm, dt = (a.D + bm - 1u) / bm;
    const dim3 grid(tp_places(vt * rt));
    if (!(a.want & (CE_DH | CE_DW))) {
        hipLaunchKernelGGL((zs_k_ce_logits<DT, false, THIN, RAW>), grid, wg, 0, stream, a);
        hipLaunchKernelGGL((zs_k_ce_loss<DT, false>), dim3(a.R), wg, 0, stream, a);
        return;
    }
    hipLaunchKernelGGL((zs_k_ce_logits<DT, true, THIN, RAW>), grid, wg, 0, stream, a);
    hipLaunchKernelGGL((zs_k_ce_loss<DT, true>), dim3(a.R), wg, 0, stream, a);
    hipLaunchKernelGGL(zs_k_ce_grad<DT>, dim3((a.Vp / 8u + CE_NT - 1u) / CE_NT, a.R), wg, 0, stream, a);
    if (a.want & CE_DH) {
        hipLaunchKernelGGL((zs_k_ce_dhidden<DT, THIN, RAW>), dim3(tp_places(dt * rt > a.units ? dt * rt : a.units)), wg, 0, stream, a);
        hipLaunchKernelGGL((zs_k_ce_join<DT, THIN>), dim3(a.R < 1024u ? a.R : 1024u, (a.D + 255u) / 256u), wg, 0, stream, a);
    }
    if (a.want & CE_DW) {
        constexpr uint32_t E = THIN ? CE_THIN_M : CE_TILE;
        hipLaunchKernelGGL((zs_k_ce_dweight<DT, THIN>), dim3(tp_places((a.D + E - 1u) / E * (a.Vp / E))), wg, 0, stream, a);
    }
}
template <int DT>
static void ce_go(ce_args a, hipStream_t stream) {
    const dim3 wg(CE_NT);
    if (a.N > CE_SELF) hipLaunchKernelGGL(zs_k_ce_rows, dim3(1), dim3(1024), 0, stream, a);
    if constexpr (DT == ZS_F32) {
        const uint32_t rows = a.Vp / (CE_NT / 64);
        if (a.w) hipLaunchKernelGGL(zs_k_ce_split, dim3(rows < 8192u ? rows : 8192u), wg, 0, stream, a);
    } else if (a.w) {
        hipLaunchKernelGGL(zs_k_ce_weight<DT>, dim3(8192, (a.V + 65535u) / 65536u), wg, 0, stream, a);
    }
    for (uint32_t p = 0; p < a.pieces; p++) {
        a.lo = p * a.R;
        a.first = p == 0u;
        a.last = p + 1u == a.pieces;
        hipLaunchKernelGGL(zs_k_ce_pack<DT>, dim3(a.R), wg, 0, stream, a);
        constexpr int ONE = DT == ZS_F32 ? 1 : 0;   // (f32 alone has them)
        if (a.raw == 1u) ce_products<DT, true, ONE>(a, stream);
        else if (a.raw) ce_products<DT, true, 2 * ONE>(a, stream);
        else if (a.thin) ce_products<DT, true, false>(a, stream);
        else ce_products<DT, false, false>(a, stream);
    }
}
int ce_launch(const ce_args& a, uint32_t dtype, hipStream_t stream) {
    if (dtype == ZS_F32) ce_go<ZS_F32>(a, stream);
    else if (dtype == ZS_F16) ce_go<ZS_F16>(a, stream);
    else ce_go<ZS_BF16>(a, stream);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <int DT>
__global__ __launch_bounds__(CE_NT) void zs_k_ce_clear(char* p, uint32_t rows, uint32_t cols, uint64_t ld) {
    for (uint64_t r = blockIdx.x; r < rows; r += gridDim.x) ce_zero<DT>(p + r * ld * (DT == ZS_F32 ? 4u : 2u), cols);
}
int ce_clear(void* p, uint32_t rows, uint32_t cols, uint64_t ld, uint32_t dtype, hipStream_t stream) {
    const dim3 grid(rows < 16384u ? rows : 16384u), wg(CE_NT);
    if (dtype == ZS_F32) hipLaunchKernelGGL(zs_k_ce_clear<ZS_F32>, grid, wg, 0, stream, (char*)p, rows, cols, ld);
    else hipLaunchKernelGGL(zs_k_ce_clear<ZS_F16>, grid, wg, 0, stream, (char*)p, rows, cols, ld);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
