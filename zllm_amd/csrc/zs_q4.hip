// zs_q4.hip -- logits of a vocabulary head held in 4 bits with scales per group
// of columns.
#include <hip/hip_runtime.h>
#include "zs_q4.h"
#include "zs_head.h"
#include "zs_tile.h"

#define Q4_NT 256

typedef float q4_f4 __attribute__((ext_vector_type(4)));
typedef uint32_t q4_u4 __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------ quantising, laying out
// A group's scale and minimum from its extremes, then its codes, two to a byte.
// Without minima w ~ scale * (code - 8) with scale = max |w| / 7; with them
// w ~ scale * code + min with scale = (max - min) / 15. Both are rounded to f16
// first and the codes taken by the rounded ones; a scale of 0 has codes of 0 (8). A
// group with a NaN or an infinity has a scale that is one, and so has its row's logits.
template <int DT>
__global__ __launch_bounds__(Q4_NT) void zs_k_q4_quantize(q4_pack_args a) {
    const uint32_t per = a.D / a.group, w = zs_wid(), l = zs_lane();
    const uint64_t groups = (uint64_t)a.V * per;
    typedef typename hd_elem<DT>::T T;
    for (uint64_t g = (uint64_t)blockIdx.x * (Q4_NT / 64) + w; g < groups; g += (uint64_t)gridDim.x * (Q4_NT / 64)) {
        const uint64_t v = g / per;
        const uint32_t c0 = (uint32_t)(g - v * per) * a.group;
        const T* x = reinterpret_cast<const T*>(a.weight) + v * a.ld_w + c0;
        float y[2] = {0.0f, 0.0f};
        const bool in = 2u * l < a.group;
        float lo = INFINITY, hi = -INFINITY;
        if (in)
            for (int i = 0; i < 2; i++) {
                y[i] = hd_float(x[2u * l + i]);
                lo = fminf(lo, y[i]), hi = fmaxf(hi, y[i]);
            }
        hi = wave_max_f(hi);
        lo = -wave_max_f(-lo);
        _Float16 s, m = (_Float16)0.0f;
        if (a.mins) {
            s = (_Float16)((hi - lo) / 15.0f);
            m = (_Float16)lo;
        } else {
            s = (_Float16)(fmaxf(fabsf(lo), fabsf(hi)) / 7.0f);
        }
        // (the extremes pass over a NaN)
        if (__ballot(y[0] != y[0] || y[1] != y[1])) s = (_Float16)NAN;
        const float sf = (float)s, mf = (float)m;
        uint32_t code = 0;
        for (int i = 0; i < 2; i++) {
            float q = sf != 0.0f ? rintf(a.mins ? (y[i] - mf) / sf : y[i] / sf) : 0.0f;
            q = fminf(fmaxf(a.mins ? q : q + 8.0f, 0.0f), 15.0f);
            code |= (uint32_t)q << (4 * i);
        }
        if (in) a.codes[(v * a.D + c0) / 2u + l] = (uint8_t)code;
        if (l == 0u) {
            a.scales[g] = __builtin_bit_cast(uint16_t, s);
            if (a.mins) a.mins[g] = __builtin_bit_cast(uint16_t, m);
        }
    }
}
// One workgroup a tile of 16 rows and 128 columns: its words, scales and minima
// (zeros past the last row or column).
__global__ __launch_bounds__(64) void zs_k_q4_pack(q4_pack_args a) {
    const uint32_t l = threadIdx.x, per = 128u / a.group;
    const uint64_t n = (uint64_t)a.at.tiles * a.at.blocks;
    for (uint64_t t = blockIdx.x; t < n; t += gridDim.x) {
        const uint64_t v0 = t / a.at.blocks * 16u, v = v0 + (l & 15u);
        const uint32_t c0 = (uint32_t)(t % a.at.blocks) * 128u;
        q4_u4 o;
        for (uint32_t b = 0; b < 4u; b++) {
            const uint32_t c = c0 + b * 32u + (l >> 4) * 8u;
            uint32_t word = 0;
            if (v < a.V && c < a.D)
                for (uint32_t j = 0; j < 4u; j++) {
                    const uint32_t two = a.codes[(v * a.D + c) / 2u + j];
                    const uint32_t pair = (two & 15u) << 3 | (two >> 4) << 19;
                    word |= j ? pair << (4u * j) | pair >> (32u - 4u * j) : pair;
                }
            o[b] = word;
        }
        *(q4_u4*)(a.head + t * 1024u + l * 16u) = o;
        for (uint32_t i = l; i < 16u * per; i += 64u) {
            const uint64_t r = v0 + i / per, g = c0 / a.group + i % per;
            const bool in = r < a.V && g < a.D / a.group;
            const uint64_t to = t * 16u * per + i, from = r * (a.D / a.group) + g;
            ((uint16_t*)(a.head + a.at.scales))[to] = in ? a.scales[from] : (uint16_t)0;
            if (a.mins) ((uint16_t*)(a.head + a.at.mins))[to] = in ? a.mins[from] : (uint16_t)0;
        }
    }
}

// ------------------------------------------------------------------ hidden states
// A wave's part of a row: 128 columns, two a lane, to the rows the kernels take and
// to their sums over the groups, times what zs_k_q4_batch starts from.
__device__ __forceinline__ void q4_sums(const q4_x_args& a, uint64_t r, uint32_t b, double t) {
    const uint32_t l = zs_lane(), per = 128u / a.group;
    t += zs_lane_xor<1>(t);
    t += zs_lane_xor<2>(t);
    t += zs_lane_xor<4>(t);
    t += zs_lane_xor<8>(t);
    if (a.group > 32u) t += zs_lane_xor<16>(t);
    if (a.group > 64u) t += zs_lane_xor<32>(t);
    if (l % (a.group / 2u) == 0u) a.sums[((uint64_t)b * per + l / (a.group / 2u)) * a.Bp + r] = (float)(t * (double)a.off);
}
template <int DT>
__global__ __launch_bounds__(Q4_NT) void zs_k_q4_rows(q4_x_args a) {
    const uint32_t l = zs_lane(), blocks = (a.D + 127u) / 128u;
    const uint64_t all = (uint64_t)a.B * blocks;
    for (uint64_t i = (uint64_t)blockIdx.x * (Q4_NT / 64) + zs_wid(); i < all; i += (uint64_t)gridDim.x * (Q4_NT / 64)) {
        const uint64_t r = i / blocks;
        const uint32_t b = (uint32_t)(i - r * blocks), d = b * 128u + l * 2u;
        const typename hd_elem<DT>::T* x = (const typename hd_elem<DT>::T*)a.hidden + r * a.ld_h + d;
        float v[2] = {0.0f, 0.0f};
        if (d < a.D)
            for (int k = 0; k < 2; k++) {
                v[k] = hd_float(x[k]);
                if (a.out) a.out[r * a.D + d + k] = __builtin_bit_cast(uint16_t, x[k]);
            }
        if (a.sums) q4_sums(a, r, b, (double)v[0] + (double)v[1]);
    }
}
// f32 rows as two f16 of the number scaled by a power of two of the row (zs_split2),
// by which the logits are scaled back. Their sums are of what the two f16 hold: what
// these leave of the number would otherwise be in the logits 24 (16) times.
__global__ __launch_bounds__(Q4_NT) void zs_k_q4_rows_f32(q4_x_args a) {
    __shared__ float sh[Q4_NT / 64];
    const uint32_t l = zs_lane(), blocks = (a.D + 127u) / 128u;
    const uint64_t r = blockIdx.x, n = (uint64_t)a.B * a.D;
    const float* x = (const float*)a.hidden + r * a.ld_h;
    float top = 0.0f;
    for (uint32_t d = threadIdx.x; d < a.D; d += Q4_NT) top = fmaxf(top, fabsf(x[d]));
    const int s = zs_split2_of(block_max_f<Q4_NT>(top, sh));
    if (threadIdx.x == 0u) a.shift[r] = s;
    for (uint32_t b = zs_wid(); b < blocks; b += Q4_NT / 64) {
        const uint32_t d = b * 128u + l * 2u;
        double v = 0.0;
        if (d < a.D) {
            uint16_t p[2][2];
            for (int k = 0; k < 2; k++) {
                zs_split2(x[d + k], s, p[k]);
                for (int q = 0; q < 2; q++) v += (double)__builtin_bit_cast(_Float16, p[k][q]);
            }
            for (int q = 0; q < 2; q++) *(uint32_t*)(a.out + q * n + r * a.D + d) = (uint32_t)p[0][q] | (uint32_t)p[1][q] << 16;
        }
        if (a.sums) q4_sums(a, r, b, v);
    }
}

// ------------------------------------------------------------------ logits
// A code q becomes the 16-bit float 16 + q by a shift and one and-or: the
// leading mantissa bits of a number between 16 and 32 count ones. What that adds
// comes off by the matrix cores too: c0 = sum x * -24 (-16 with minima) is the
// sum the products start from. Operand register j holds columns 2 j, 2 j + 1.
template <int DT>
struct q4_num {
    static constexpr uint32_t ONE = DT != ZS_BF16 ? 6 : 3;                                   // log2 of a unit's bits
    static constexpr uint32_t BASE = DT != ZS_BF16 ? 0x4c004c00u : 0x41804180u, MASK = 0x000f000fu << ONE;
    static constexpr uint32_t M16 = DT != ZS_BF16 ? 0xcc00cc00u : 0xc180c180u, M24 = DT != ZS_BF16 ? 0xce00ce00u : 0xc1c0c1c0u;
    uint32_t mask, base;
    __device__ __forceinline__ q4_num() {
        // in a scalar and a vector register, which one and-or takes: of two
        // literals it takes none, and the compiler makes two instructions of it
        mask = MASK, base = BASE;
        asm volatile("" : "+s"(mask), "+v"(base));
    }
    __device__ __forceinline__ q4_u4 operand(uint32_t w) const {
        q4_u4 o;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int r = 4 * j + 3 - (int)ONE;   // to the right, around (only the last pair lies across the ends)
            o[j] = ((r == 0 ? w : j == 3 ? w >> r | w << (32 - r) : r > 0 ? w >> r : w << -r) & mask) | base;
        }
        return o;
    }
    static __device__ __forceinline__ q4_f4 mul(q4_u4 a, q4_u4 b, q4_f4 c) {
#if defined(__HIP_DEVICE_COMPILE__)
        if constexpr (DT != ZS_BF16) {
            typedef _Float16 h8 __attribute__((ext_vector_type(8)));
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
        } else {
            typedef __bf16 b8 __attribute__((ext_vector_type(8)));
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
        }
#else
        return c;
#endif
    }
};

// T tiles of 16 ids by up to 16 rows of hidden states: each wave takes a part of
// the columns, their sums are joined through shared memory. Codes, scales and
// hidden states of the next 128 columns are on their way while these are used.
// Bound by the codes' bytes, with up to 40 % of the vector units for operands and
// scales beside them: 1 row of 4096, 32000 ids, 15 us (4.9 TB/s; 151936 ids 61 us, 5.8),
// 16 rows of 2048, 128256 ids with minima 32 us (4.8).
// NI is how many of a lane's four rows there are: row b of the hidden states has
// place 4 (b % 4) + b / 4 among the operand's, so that up to 4 rows are the first
// of their lane, up to 8 the first two.
template <int DT, int G, bool MINS, int T, int NI>
struct q4_few {
    static constexpr int P = DT == ZS_F32 ? 2 : 1, PER = 128 / G;
    typedef q4_num<DT> num;
    typedef _Float16 hv __attribute__((ext_vector_type(PER)));
    struct regs {
        q4_u4 w[T], x[P][4];
        hv s[T], m[MINS ? T : 1];
    };
    const q4_args& a;
    const num nm;
    uint64_t tile[T];
    const uint16_t* x;
    uint32_t l;
    q4_f4 acc[T];

    __device__ __forceinline__ q4_few(const q4_args& a_, uint32_t t0) : a(a_) {
        l = (uint32_t)zs_lane();
        const uint32_t r = (l & 3u) * 4u + ((l & 15u) >> 2);
        x = (const uint16_t*)a.hidden + (r < a.B ? r : a.B - 1u) * a.ld_h + (l >> 4) * 8u;
#pragma unroll
        for (int t = 0; t < T; t++) {
            tile[t] = (uint64_t)(t0 + t < a.at.tiles ? t0 + t : a.at.tiles - 1u) * a.at.blocks;
            acc[t] = q4_f4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    __device__ __forceinline__ void get(uint32_t b, regs& g) const {
#pragma unroll
        for (int t = 0; t < T; t++) {
            const uint64_t at = tile[t] + b;
            // (not read again)
            g.w[t] = __builtin_nontemporal_load((const __attribute__((address_space(1))) q4_u4*)(a.head + at * 1024u + l * 16u));
            g.s[t] = zs_gload((const hv*)(a.head + a.at.scales + (at * 16u + (l & 15u)) * (PER * 2)));
            if constexpr (MINS) g.m[t] = zs_gload((const hv*)(a.head + a.at.mins + (at * 16u + (l & 15u)) * (PER * 2)));
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            // (past the last column the last 32 again: the scales there are 0)
            const uint32_t d = b * 128u + k * 32u, at = d < a.D ? d : a.D - 32u;
#pragma unroll
            for (int p = 0; p < P; p++) g.x[p][k] = zs_gload((const q4_u4*)(x + p * a.plane + at));
        }
    }
    // (a group's products are scaled when the next group's are on their way)
    __device__ __forceinline__ void mul(const regs& g) {
        const uint32_t o = MINS ? num::M16 : num::M24;
        const q4_u4 off = {o, o, o, o};
        q4_f4 c0[PER], d[PER][T];
        auto scaled = [&](int q) {
#pragma unroll
            for (int t = 0; t < T; t++) {
                const float sf = (float)g.s[t][q], mf = MINS ? (float)g.m[MINS ? t : 0][q] * -0.0625f : 0.0f;
#pragma unroll
                for (int i = 0; i < NI; i++) {
                    acc[t][i] = __builtin_fmaf(sf, d[q][t][i], acc[t][i]);
                    if (MINS) acc[t][i] = __builtin_fmaf(mf, c0[q][i], acc[t][i]);
                }
            }
        };
#pragma unroll
        for (int q = 0; q < PER; q++) {
            c0[q] = q4_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = q * (G / 32); k < (q + 1) * (G / 32); k++)
#pragma unroll
                for (int p = 0; p < P; p++) c0[q] = num::mul(g.x[p][k], off, c0[q]);
        }
#pragma unroll
        for (int q = 0; q < PER; q++) {
#pragma unroll
            for (int k = q * (G / 32); k < (q + 1) * (G / 32); k++)
#pragma unroll
                for (int t = 0; t < T; t++) {
                    const q4_u4 op = nm.operand(g.w[t][k]);
#pragma unroll
                    for (int p = 0; p < P; p++) d[q][t] = num::mul(g.x[p][k], op, k == q * (G / 32) && p == 0 ? c0[q] : d[q][t]);
                }
            if (q > 0) scaled(q - 1);
        }
        scaled(PER - 1);
    }
    __device__ __forceinline__ void run(uint32_t b0, uint32_t b1) {
        if (b0 >= b1) return;
        regs g0, g1;
        get(b0, g0);
        tp_in_order();
        for (; b0 + 1u < b1; b0 += 2u) {
            get(b0 + 1u, g1);
            tp_in_order();
            mul(g0);
            get(b0 + 2u < b1 ? b0 + 2u : b0 + 1u, g0);
            tp_in_order();
            mul(g1);
        }
        if (b0 < b1) mul(g0);
    }
};
template <int DT, int G, bool MINS, int T, int KS, int NI>
__global__ __launch_bounds__(KS * 64) void zs_k_q4_logits(q4_args a) {
    __shared__ q4_f4 sh[KS][T][64];
    const uint32_t w = (uint32_t)__builtin_amdgcn_readfirstlane(zs_wid()), t0 = blockIdx.x * T;
    q4_few<DT, G, MINS, T, NI> q(a, t0);
    q.run(a.at.blocks * w / KS, a.at.blocks * (w + 1u) / KS);
#pragma unroll
    for (int t = 0; t < T; t++) sh[w][t][q.l] = q.acc[t];
    __syncthreads();
    for (uint32_t t = w; t < T; t += KS) {
        q4_f4 v = sh[0][t][q.l];
        for (int k = 1; k < KS; k++) v += sh[k][t][q.l];
        const uint32_t id = (t0 + t) * 16u + (q.l & 15u);
        if (id >= a.V) continue;
#pragma unroll
        for (uint32_t i = 0; i < NI; i++) {
            const uint32_t row = i * 4u + (q.l >> 4);
            if (row < a.B) a.logits[row * a.ld + id] = DT == ZS_F32 ? ldexpf(v[i], -a.shift[row]) : v[i];
        }
    }
}

// The same for more rows: 16 RT rows by 64 T ids a workgroup, its waves side by
// side along the ids. The hidden states of 128 columns at a time come to shared
// memory as operands (lane l's 16 bytes at 16 l), two steps ahead of their use,
// and the waves' codes and scales to registers likewise. (Groups of 32: one step in
// three waits for all loads, as the compiler makes the next step's first operands
// before that step begins.)
// Bound by the instructions: 64 rows of 4096, 151936 ids, groups of 32, 119 us, the
// vector units busy for 54 %, the matrix cores for 29 % of it, one beside the other
// in part only; 320 rows, groups of 128, 411 us, 49 and 46 % (969 TFLOP/s).
template <int DT, int G, bool MINS, int T, int RT>
struct q4_batch {
    static constexpr int P = DT == ZS_F32 ? 2 : 1, PER = 128 / G, PIECES = P * RT * 4;
    static constexpr int LOADS = T * (MINS ? 3 : 2) + P * RT + 1, STAGE = PIECES * 1024 + 1024;
    typedef q4_num<DT> num;
    typedef _Float16 hv __attribute__((ext_vector_type(PER)));
    struct regs {
        q4_u4 w[T];
        hv s[T], m[MINS ? T : 1];
    };
    const q4_args& a;
    uint32_t tile[T];
    const uint16_t* x[RT];
    const float* sums;
    uint32_t l, w, kcol;
    num nm;
    q4_f4 acc[T][RT];

    __device__ __forceinline__ q4_batch(const q4_args& a_, uint32_t t0, uint32_t r0) : a(a_) {
        l = (uint32_t)zs_lane();
        w = (uint32_t)__builtin_amdgcn_readfirstlane(zs_wid());
        kcol = w * 32u;
#pragma unroll
        for (int t = 0; t < T; t++) {
            const uint32_t n = t0 + w * T + t;
            tile[t] = n < a.at.tiles ? n : a.at.tiles - 1u;
#pragma unroll
            for (int r = 0; r < RT; r++) acc[t][r] = q4_f4{0.0f, 0.0f, 0.0f, 0.0f};
        }
#pragma unroll
        for (int r = 0; r < RT; r++) {
            const uint32_t row = r0 + r * 16u + (l & 15u);
            x[r] = (const uint16_t*)a.hidden + (row < a.B ? row : a.B - 1u) * a.ld_h + (l >> 4) * 8u;
        }
        sums = a.sums + (w % PER) * a.Bp + r0 + (l < 16u * RT ? l : 16u * RT - 1u);
    }
    // columns 128 b on, to registers and to shared memory at sh (past the last
    // column the last 32 again: the scales there are 0)
    __device__ __forceinline__ void put(uint32_t b, regs& g, tp_lds* sh) const {
#if defined(__HIP_DEVICE_COMPILE__)
        b = b < a.at.blocks ? b : a.at.blocks - 1u;
#pragma unroll
        for (int t = 0; t < T; t++) {
            const uint64_t at = (uint64_t)tile[t] * a.at.blocks + b;
            g.w[t] = zs_gload((const q4_u4*)(a.head + at * 1024u + l * 16u));
            g.s[t] = zs_gload((const hv*)(a.head + a.at.scales + (at * 16u + (l & 15u)) * (PER * 2)));
            if constexpr (MINS) g.m[t] = zs_gload((const hv*)(a.head + a.at.mins + (at * 16u + (l & 15u)) * (PER * 2)));
        }
        uint32_t k = b * 128u + kcol;
        k = k < a.D ? k : a.D - 32u;
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int r = 0; r < RT; r++)
                __builtin_amdgcn_global_load_lds((tp_glb*)(x[r] + p * a.plane + k), sh + ((p * RT + r) * 4 + (int)w) * 1024, 16, 0, 0);
        __builtin_amdgcn_global_load_lds((tp_glb*)(sums + (uint64_t)b * PER * a.Bp), sh + PIECES * 1024 + w * 256u, 4, 0, 0);
#endif
    }
    __device__ __forceinline__ q4_u4 frag(const tp_lds* sh, int p, int r, int k) const {
        return *(const __attribute__((address_space(3))) q4_u4*)(sh + ((p * RT + r) * 4 + k) * 1024 + l * 16u);
    }
    // (the products of a tile are scaled when the next one's are on their way)
    __device__ __forceinline__ void mul(const regs& g, const tp_lds* sh) {
#pragma unroll
        for (int q = 0; q < PER; q++) {
            q4_f4 c0[RT], d[T][RT];
#pragma unroll
            for (int r = 0; r < RT; r++)
                c0[r] = *(const __attribute__((address_space(3))) q4_f4*)(sh + PIECES * 1024 + q * 256 + r * 64 + (l >> 4) * 16u);
            auto scaled = [&](int t) {
                float sf = (float)g.s[t][q];
                asm volatile("" : "+v"(sf));   // (converted once, not in every product)
                const float mf = MINS ? (float)g.m[MINS ? t : 0][q] * -0.0625f : 0.0f;
#pragma unroll
                for (int r = 0; r < RT; r++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        acc[t][r][i] = __builtin_fmaf(sf, d[t][r][i], acc[t][r][i]);
                        if (MINS) acc[t][r][i] = __builtin_fmaf(mf, c0[r][i], acc[t][r][i]);
                    }
            };
#pragma unroll
            for (int k = q * (G / 32); k < (q + 1) * (G / 32); k++) {
                const bool first = k == q * (G / 32), last = k == (q + 1) * (G / 32) - 1;
                q4_u4 f[P][RT];
#pragma unroll
                for (int p = 0; p < P; p++)
#pragma unroll
                    for (int r = 0; r < RT; r++) f[p][r] = frag(sh, p, r, k);
#pragma unroll
                for (int t = 0; t < T; t++) {
                    const q4_u4 op = nm.operand(g.w[t][k]);
#pragma unroll
                    for (int p = 0; p < P; p++)
#pragma unroll
                        for (int r = 0; r < RT; r++) d[t][r] = num::mul(f[p][r], op, first && p == 0 ? c0[r] : d[t][r]);
                    if (last && t > 0) scaled(t - 1);
                }
                if (last) scaled(T - 1);
#if defined(__HIP_DEVICE_COMPILE__)
                if (G > 32) __builtin_amdgcn_sched_barrier(0);   // (the operands of all columns at once do not fit the registers)
#endif
            }
        }
    }
    __device__ __forceinline__ void run() {
        __shared__ char s0_[STAGE], s1_[STAGE], s2_[STAGE];
        tp_lds *s0 = (tp_lds*)s0_, *s1 = (tp_lds*)s1_, *s2 = (tp_lds*)s2_;
        regs g0, g1, g2;
        const uint32_t n = a.at.blocks, whole = n / 3u * 3u;
        put(0, g0, s0);
        tp_in_order();
        put(1, g1, s1);
        tp_in_order();
        for (uint32_t b = 0; b < whole; b += 3u) {
            tp_arrived<LOADS, true>();
            put(b + 2u, g2, s2);
            mul(g0, s0);
            tp_arrived<LOADS, true>();
            put(b + 3u, g0, s0);
            mul(g1, s1);
            tp_arrived<LOADS, true>();
            put(b + 4u, g1, s1);
            mul(g2, s2);
        }
        tp_arrived<0, true>();
        if (n - whole > 0u) mul(g0, s0);
        if (n - whole > 1u) mul(g1, s1);
    }
};
template <int DT, int G, bool MINS, int T, int RT>
__global__ __launch_bounds__(Q4_NT, 2) void zs_k_q4_batch(q4_args a, uint32_t parts) {
    // the parts of the rows next to each other on one XCD, so that a part finds the codes in its L2
    const uint32_t j = blockIdx.x >> 3, t0 = ((j / parts) * 8u + (blockIdx.x & 7u)) * (4 * T), r0 = j % parts * (16 * RT);
    if (t0 >= a.at.tiles) return;
    q4_batch<DT, G, MINS, T, RT> q(a, t0, r0);
    q.run();
#pragma unroll
    for (int t = 0; t < T; t++) {
        const uint32_t id = (t0 + q.w * T + t) * 16u + (q.l & 15u);
        if (id >= a.V) continue;
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t row = r0 + r * 16u + (q.l >> 4) * 4u + i;
                if (row < a.B) a.logits[row * a.ld + id] = DT == ZS_F32 ? ldexpf(q.acc[t][r][i], -a.shift[row]) : q.acc[t][r][i];
            }
    }
}

int q4_pack(const q4_pack_args& a, hipStream_t stream) {
    const uint64_t n = (uint64_t)a.at.tiles * a.at.blocks;
    hipLaunchKernelGGL(zs_k_q4_pack, dim3(n < 65536u ? (uint32_t)n : 65536u), dim3(64), 0, stream, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
int q4_quantize(const q4_pack_args& a, uint32_t dtype, hipStream_t stream) {
    const uint64_t n = ((uint64_t)a.V * (a.D / a.group) + Q4_NT / 64 - 1u) / (Q4_NT / 64);
    const dim3 grid(n < 65536u ? (uint32_t)n : 65536u), wg(Q4_NT);
    if (dtype == ZS_F32) hipLaunchKernelGGL(zs_k_q4_quantize<ZS_F32>, grid, wg, 0, stream, a);
    else if (dtype == ZS_F16) hipLaunchKernelGGL(zs_k_q4_quantize<ZS_F16>, grid, wg, 0, stream, a);
    else hipLaunchKernelGGL(zs_k_q4_quantize<ZS_BF16>, grid, wg, 0, stream, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
template <int DT, int G, bool MINS, int T, int RT>
static void q4_batch_go(const q4_args& a, hipStream_t stream) {
    const uint32_t parts = (a.B + 16u * RT - 1u) / (16u * RT), groups = (a.at.tiles + 4u * T - 1u) / (4u * T);
    hipLaunchKernelGGL((zs_k_q4_batch<DT, G, MINS, T, RT>), dim3((groups + 7u) / 8u * 8u * parts), dim3(Q4_NT), 0, stream, a, parts);
}
template <int DT, int G, bool MINS, int KS>
static void q4_few_go(const q4_args& a, hipStream_t stream) {
    constexpr int T = 4;
    const dim3 grid((a.at.tiles + T - 1u) / T), wg(KS * 64);
    if (a.B <= 4u) hipLaunchKernelGGL((zs_k_q4_logits<DT, G, MINS, T, KS, 1>), grid, wg, 0, stream, a);
    else if (a.B <= 8u) hipLaunchKernelGGL((zs_k_q4_logits<DT, G, MINS, T, KS, 2>), grid, wg, 0, stream, a);
    else hipLaunchKernelGGL((zs_k_q4_logits<DT, G, MINS, T, KS, 4>), grid, wg, 0, stream, a);
}
template <int DT, int G, bool MINS>
static void q4_go(const q4_args& a, hipStream_t stream) {
    if (a.B > 16u) {
        // Tiles of ids a wave: as many as let all workgroups find room at once, two a CU
        // (one, where a workgroup a CU is all there is). us, 64 bf16 rows of 4096, groups
        // of 32, by 1, 2, 3, 4 and 5 tiles: 16000 ids 29 and 37; 32000 ids 46, 40 and (4)
        // 55; 90000 ids (2) 75, 70 and 84; 128256 ids (2) 117 and (4) 102; 151936 ids (2)
        // 139, (4) 136 and 122. Up to 32 rows, of which a workgroup has 32 and not 64, two
        // (17 rows by 2 and by as many as find room: 90000 ids 47 and 57, 128256 ids 66 and
        // 68, 151936 ids 83 and 92; by 64 rows a workgroup 78, 95 and 126). Beyond 64 rows a
        // part of the rows finds another's codes in the L2, and 4 serve. Of larger groups or
        // with minima 5 do not fit the registers (of groups of 128 with minima 4 do but for
        // 6 registers, which are spilled).
        uint32_t t = (a.at.tiles + 2047u) / 2048u;
        t = a.at.tiles <= 1024u ? 1u : t < 2u ? 2u : t;
        if (DT == ZS_F32 || a.B <= 32u) q4_batch_go<DT, G, MINS, 2, 2>(a, stream);
        else if constexpr (DT != ZS_F32) {
            if (a.B > 64u || t == 4u || t > (G == 32 && !MINS ? 5u : 4u)) q4_batch_go<DT, G, MINS, 4, 4>(a, stream);
            else if (t == 1u) q4_batch_go<DT, G, MINS, 1, 4>(a, stream);
            else if (t == 2u) q4_batch_go<DT, G, MINS, 2, 4>(a, stream);
            else if (t == 3u) q4_batch_go<DT, G, MINS, 3, 4>(a, stream);
            else if constexpr (G == 32 && !MINS) q4_batch_go<DT, G, MINS, 5, 4>(a, stream);
        }
        return;
    }
    // Waves along the columns where there are few ids: 4 against 1, us, 16 bf16
    // rows of 4096, groups of 32: 32000 ids 19 and 24 (one row 15 and 19), 65536
    // ids 38 and 32 (29 and 26), 151936 ids 83 and 84 (65 and 66)
    if (a.at.tiles < 4096u) q4_few_go<DT, G, MINS, 4>(a, stream);
    else q4_few_go<DT, G, MINS, 1>(a, stream);
}
template <int DT>
static void q4_group(const q4_args& a, uint32_t group, bool mins, hipStream_t stream) {
    if (group == 32u) mins ? q4_go<DT, 32, true>(a, stream) : q4_go<DT, 32, false>(a, stream);
    else if (group == 64u) mins ? q4_go<DT, 64, true>(a, stream) : q4_go<DT, 64, false>(a, stream);
    else mins ? q4_go<DT, 128, true>(a, stream) : q4_go<DT, 128, false>(a, stream);
}
int q4_logits(const q4_args& a, const q4_x_args* x, uint32_t dtype, uint32_t group, bool mins, hipStream_t stream) {
    if (x) {
        const uint64_t n = ((uint64_t)x->B * ((x->D + 127u) / 128u) + Q4_NT / 64 - 1u) / (Q4_NT / 64);
        const dim3 grid(n < 4096u ? (uint32_t)n : 4096u), wg(Q4_NT);
        if (dtype == ZS_F32) hipLaunchKernelGGL(zs_k_q4_rows_f32, dim3(x->B), wg, 0, stream, *x);
        else if (dtype == ZS_F16) hipLaunchKernelGGL(zs_k_q4_rows<ZS_F16>, grid, wg, 0, stream, *x);
        else hipLaunchKernelGGL(zs_k_q4_rows<ZS_BF16>, grid, wg, 0, stream, *x);
    }
    if (dtype == ZS_F32) q4_group<ZS_F32>(a, group, mins, stream);
    else if (dtype == ZS_F16) q4_group<ZS_F16>(a, group, mins, stream);
    else q4_group<ZS_BF16>(a, group, mins, stream);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
