// zs_tile.h -- products of 16-bit matrices by the matrix cores, one tile of the
// result per workgroup: D[m][n] = sum_k A[m][k] B[n][k] in f32.
#pragma once
#include <hip/hip_runtime.h>
#include "zs_internal.h"
#include "zs_dev.h"

// An operand lies k-fast (rows of A or B, k along a row) or k-slow (rows of k,
// m or n along a row). It may have planes: matrices whose sum it is.
struct tp_mat {
    const uint16_t* p[3];
    uint64_t ld;          // elements from row to row, a multiple of 8, at most TP_LD
    uint32_t rows;        // m or n there are: what a tile reads past them is the last's
    uint32_t k;           // k there are: what is read past them is the last eight's (k-fast) or the last's (k-slow), for
                          // the other operand's zeros there
};
#define TP_LD (1u << 22)
#define TP_KSTEP 32       // k of a step

typedef __attribute__((address_space(3))) char tp_lds;
typedef __attribute__((address_space(1))) const char tp_glb;
typedef float tp_acc __attribute__((ext_vector_type(16)));
typedef short tp_s4 __attribute__((ext_vector_type(4)));
typedef short tp_s8 __attribute__((ext_vector_type(8)));

template <int KIND>
__device__ __forceinline__ tp_acc tp_mfma(tp_s8 a, tp_s8 b, tp_acc c) {
#if defined(__HIP_DEVICE_COMPILE__)
    if constexpr (KIND == ZS_F16 || KIND == 3 || KIND == 5) {
        typedef _Float16 h8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    } else {
        typedef __bf16 b8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    }
#else
    return c;
#endif
}

// All but the last N of a lane's loads are there, in every wave, and (READ) what
// the waves have read of shared memory is in their registers. (The wait's fields:
// vector memory N, its two upper bits apart; LDS; the others are not waited for.)
template <int N, bool READ = false>
__device__ __forceinline__ void tp_arrived() {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | (READ ? 0x0070 : 0x0f70));
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#endif
}
// Loads are counted: those in front of it are issued before those behind it.
__device__ __forceinline__ void tp_in_order() {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_sched_barrier(0);
#endif
}

// One operand of a tile of X rows (m or n): what a lane loads to shared memory
// and what it reads from there. A step's X x 32 values lie in shared memory as
// the loads write them, 16 bytes a lane one behind the other; which 16 bytes a
// lane fetches is permuted so that the reads spread over the banks.
//   k-fast: row r's four 16-byte pieces at r * 64 B, piece c in place c ^ s(r)
//   k-slow: row k's X / 8 pieces at k * 2 X B, piece c in place c ^ ((k & 3) << 2)
template <int X, bool SLOW>
struct tp_side {
    static constexpr int LOADS = X * 4 / 256;    // of a lane a step
    const char* base;
    uint32_t off[SLOW ? 1 : LOADS];
    uint32_t kb, kmax, ld2, left;
    uint32_t rd[SLOW ? 4 : 2];   // (of rows 32 t on, t < 4; of k 16 s on)

    __device__ __forceinline__ void start(const tp_mat& m, uint32_t x0, uint32_t wx) {
        const uint32_t l = (uint32_t)zs_lane(), w = (uint32_t)__builtin_amdgcn_readfirstlane(zs_wid());
        const uint32_t x1 = first(m, x0);
        ld2 = (uint32_t)m.ld * 2u;
        if constexpr (!SLOW) {
            const uint32_t r = l >> 2;
            kb = ((l & 3u) ^ swz(r)) * 16u;
            kmax = m.k * 2u - 16u;
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
                uint32_t row = x0 + (uint32_t)(i * 4) * 16u + w * 16u + r;
                row = row < m.rows ? row : m.rows - 1u;
                off[i] = (row - x1) * ld2;
            }
            const uint32_t rr = l & 31u;
#pragma unroll
            for (int s = 0; s < 2; s++) rd[s] = (wx + rr) * 64u + ((((uint32_t)s * 2u + (l >> 5)) ^ swz(rr)) * 16u);
        } else {
            constexpr uint32_t C = X / 8;        // pieces a row: 16 or 32
            constexpr uint32_t P = 64u / C;      // rows of a wave's load
            const uint32_t r = w * P + l / C;
            uint32_t c = (l % C) ^ ((r & 3u) << 2);
            const uint32_t last = (m.rows >> 3) - 1u - (x1 >> 3);
            c = c < last ? c : last;
            kb = r;
            off[0] = c * 16u;
            left = m.k;
            const uint32_t q = (l & 15u) >> 2, k = (l >> 5) * 8u + q;
            const uint32_t c0 = wx / 8u + ((l >> 4) & 1u) * 2u + ((l & 3u) >> 1);
#pragma unroll
            for (int t = 0; t < 4; t++) rd[t] = k * (2u * X) + ((c0 + (uint32_t)t * 4u) ^ (q << 2)) * 16u + (l & 1u) * 8u;
        }
    }
    static __device__ __forceinline__ uint32_t swz(uint32_t r) { return ((r >> 1) & 3u) ^ ((r >> 3) & 1u); }
    // the tile's first row (m or n), or the last there is where it begins behind that
    static __device__ __forceinline__ uint32_t first(const tp_mat& m, uint32_t x0) {
        const uint32_t end = SLOW ? m.rows - 8u : m.rows - 1u;
        return x0 < end ? x0 : end;
    }
    __device__ __forceinline__ void plane(const tp_mat& m, int p, uint32_t x0) {
        const uint32_t x1 = first(m, x0);
        base = (const char*)m.p[p] + (SLOW ? (uint64_t)x1 * 2u : (uint64_t)x1 * m.ld * 2u);
    }
    // step kt's values to shared memory at s
    __device__ __forceinline__ void load(uint32_t kt, tp_lds* s) const {
#if defined(__HIP_DEVICE_COMPILE__)
        const uint32_t w = (uint32_t)__builtin_amdgcn_readfirstlane(zs_wid());
        if constexpr (!SLOW) {
            uint32_t k = kt * 64u + kb;
            k = k < kmax ? k : kmax;
#pragma unroll
            for (int i = 0; i < LOADS; i++)
                __builtin_amdgcn_global_load_lds((tp_glb*)(base + (off[i] + k)), s + (i * 4096 + w * 1024u), 16, 0, 0);
        } else {
            constexpr uint32_t R = 4u * (64u / (X / 8));   // rows of the workgroup's load
            const uint32_t k0 = kt * 32u < left ? kt * 32u : left - 1u, end = left - 1u - k0;
            const char* b = base + (uint64_t)k0 * ld2;
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
                uint32_t k = kb + (uint32_t)i * R;
                k = k < end ? k : end;
                __builtin_amdgcn_global_load_lds((tp_glb*)(b + (__umul24(k, ld2) + off[0])), s + (i * 4096 + w * 1024u), 16, 0, 0);
            }
        }
#endif
    }
    // the values of 32 rows t and 16 k s for the matrix cores: lane l has row l % 32, k (l / 32) * 8 .. + 7
    __device__ __forceinline__ tp_s8 frag(const tp_lds* s, int t, int ks) const {
#if defined(__HIP_DEVICE_COMPILE__)
        if constexpr (!SLOW) {
            return *(const __attribute__((address_space(3))) tp_s8*)(s + rd[ks] + t * 2048);
        } else {
            typedef __attribute__((address_space(3))) tp_s4 ls4;
            const tp_lds* p = s + rd[t] + ks * (32 * X);
            const tp_s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ls4*)p);
            const tp_s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ls4*)(p + 8 * X));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
#else
        return tp_s8{};
#endif
    }
};

// What operands are: 16-bit numbers (ZS_F16, ZS_BF16), or f32 numbers as planes
// whose products make theirs, the smallest first:
//   TP_TWO    f16 x0 + x1 of x scaled by a power of two (zs_split2): x1 y0, x0 y1,
//             x0 y0. What x0 + x1 leaves of x and the product left out, x1 y1, are
//             each at most 2^-22 of theirs: 3 * 2^-22 |x y| in all. Numbers below
//             2^-18 of the largest have less than 22 bits: half of f16's smallest step,
//             2^-25, is at most 2^-39 of a largest that is 2^14 or more.
//   TP_THREE  bf16 x0 + x1 + x2 (zs_split3), of any size: x2 y0, x0 y2, x1 y1, x1 y0,
//             x0 y1, x0 y0. |x1| is at most 2^-8 |x| and |x2| 2^-17 |x|, so that x1 y2, x2
//             y1 and x2 y2, left out, are 2^-24 (1 + 2^-10) of |x y|.
// or 16-bit numbers A with a B of two planes, B1 what B0 leaves:
//   TP_REST_F16, TP_REST_BF16   x y1, x y0
#define TP_TWO 3
#define TP_THREE 4
#define TP_REST_F16 5
#define TP_REST_BF16 6
template <int KIND> struct tp_planes {
    static constexpr int PAIRS = 1;
    static constexpr uint32_t A = 0, B = 0;   // the planes of pair s at 4 s
};
template <> struct tp_planes<TP_TWO> {
    static constexpr int PAIRS = 3;
    static constexpr uint32_t A = 0x001u, B = 0x010u;
};
template <> struct tp_planes<TP_REST_F16> {
    static constexpr int PAIRS = 2;
    static constexpr uint32_t A = 0x00u, B = 0x01u;
};
template <> struct tp_planes<TP_REST_BF16> : tp_planes<TP_REST_F16> {};
template <> struct tp_planes<TP_THREE> {
    static constexpr int PAIRS = 6;
    static constexpr uint32_t A = 0x001102u, B = 0x010120u;
};

struct tp_none {
    __device__ __forceinline__ void operator()() const {}
};

// A tile of BM x BN = (32 MT WM) x (32 NT WN) by four waves, WM along m.
// 256 x 256 has 128 x 128 a wave, all of its 256 accumulation registers: 16
// instructions of 32 clocks for eight operands of 1 KB, so that the four waves ask
// for 64 of the some 230 bytes a clock that shared memory gives, and memory for 32
// KB in 1024 clocks a CU. Bound by the matrix cores: 8192 x 4096 over 151936 in
// 7250 us, 1407 TFLOP/s (the library's product 1574), the cores busy for 82 % of the
// clocks there are under that load (1.6 to 1.9 GHz). (Of what else is held 16 to 51
// registers are spilled, outside the loop over the steps.) Smaller tiles, two workgroups a
// CU, have one's begin and end beside the other's products, but read more: 256 x 128
// took 5106 us of an evaluation's 4184.
template <int KIND, int MT, int NT, int WM, bool AS, bool BS>
struct tp_tile {
    static constexpr int M = MT, N = NT, WN = 4 / WM, BM = 32 * MT * WM, BN = 32 * NT * WN;
    static constexpr int SA = BM * 64, STAGE = (BM + BN) * 64;
    typedef tp_planes<KIND> planes_of;
    static constexpr int PAIRS = planes_of::PAIRS;
    typedef tp_side<BM, AS> A;
    typedef tp_side<BN, BS> B;
    static constexpr int LOADS = A::LOADS + B::LOADS;
    const tp_mat &ma, &mb;
    A a;
    B b;
    uint32_t m0, n0, kt, ka, kz;    // the step that is loaded next, of ka .. kz - 1
    int pair;

    __device__ __forceinline__ static uint32_t wm() { return (uint32_t)__builtin_amdgcn_readfirstlane(zs_wid()) % WM; }
    __device__ __forceinline__ static uint32_t wn() { return (uint32_t)__builtin_amdgcn_readfirstlane(zs_wid()) / WM; }
    // m and n of a lane's values: n by j, m by i and q, four of them from c[i][j][4 q]
    __device__ __forceinline__ uint32_t n_of(int j) const { return n0 + wn() * (32 * NT) + (uint32_t)j * 32u + ((uint32_t)zs_lane() & 31u); }
    __device__ __forceinline__ uint32_t m_of(int i, int q) const {
        return m0 + wm() * (32 * MT) + (uint32_t)i * 32u + (uint32_t)q * 8u + ((uint32_t)zs_lane() >> 5) * 4u;
    }

    __device__ __forceinline__ tp_tile(const tp_mat& ma_, const tp_mat& mb_, uint32_t m, uint32_t n) : ma(ma_), mb(mb_), m0(m * BM), n0(n * BN) {
        a.start(ma, m0, wm() * (32 * MT));
        b.start(mb, n0, wn() * (32 * NT));
    }
    // Three steps' values in shared memory: one that the waves read, two on their
    // way. (Arrays of their own: the compiler tells from them that a read does not
    // wait for the later steps' loads.)
    __device__ __forceinline__ static tp_lds* stage(uint32_t i) {
        __shared__ char s0_[STAGE], s1_[STAGE], s2_[STAGE];
        return i == 0u ? (tp_lds*)s0_ : i == 1u ? (tp_lds*)s1_ : (tp_lds*)s2_;
    }
    struct regs {   // operands of half a step, 16 k
        tp_s8 a[MT], b[NT];
    };
    __device__ __forceinline__ void get(const tp_lds* s, int ks, regs& r) const {
#pragma unroll
        for (int i = 0; i < MT; i++) r.a[i] = a.frag(s, i, ks);
#pragma unroll
        for (int i = 0; i < NT; i++) r.b[i] = b.frag(s + SA, i, ks);
    }
    __device__ __forceinline__ static void mul(const regs& r, tp_acc (&c)[MT][NT]) {
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NT; j++) c[i][j] = tp_mfma<KIND>(r.a[i], r.b[j], c[i][j]);
    }
    // the next step's values; past the last the last again, which nobody reads
    __device__ __forceinline__ void put(tp_lds* s) {
        a.load(kt, s);
        b.load(kt, s + SA);
        if (++kt == kz) {
            kt = kz - 1u;
            if (PAIRS > 1 && pair + 1 < PAIRS) {
                pair++;
                kt = ka;
                planes();
            }
        }
    }
    __device__ __forceinline__ void planes() {
        a.plane(ma, (int)(planes_of::A >> (4 * pair)) & 15, m0);
        b.plane(mb, (int)(planes_of::B >> (4 * pair)) & 15, n0);
    }
    // c += A B over steps k0 .. k0 + n - 1; beside() is called while the first are on their way
    template <class F = tp_none>
    __device__ __forceinline__ void run(uint32_t k0, uint32_t n, tp_acc (&c)[MT][NT], const F& beside = F()) {
        tp_lds* const s[3] = {stage(0), stage(1), stage(2)};
        if (n == 0u) return;
        regs r0, r1;
        kt = ka = k0;
        kz = k0 + n;
        pair = 0;
        planes();
        put(s[0]);
        tp_in_order();
        put(s[1]);
        tp_in_order();
        put(s[2]);
        tp_in_order();
        beside();
        tp_arrived<2 * LOADS>();
        get(s[0], 0, r0);
        // A step: its first half's products while the second's operands are read;
        // then the next step's values have arrived and this one's memory is free.
        auto step = [&](tp_lds* now, tp_lds* next) {
            get(now, 1, r1);
            mul(r0, c);
            sched<0>();
            tp_arrived<LOADS, true>();
            put(now);
            get(next, 0, r0);
            mul(r1, c);
            sched<LOADS>();
        };
        const uint32_t all = n * PAIRS, whole = all / 3u * 3u;
        for (uint32_t k = 0; k < whole; k += 3u) {
            step(s[0], s[1]);
            step(s[1], s[2]);
            step(s[2], s[0]);
        }
        if (all - whole > 0u) step(s[0], s[1]);
        if (all - whole > 1u) step(s[1], s[2]);
        tp_arrived<0, true>();
    }
    // A wave's values as 16-bit numbers, whole rows n at a time. A lane has four
    // values of each of its rows, so written from there a row's 256 bytes would go
    // out in 16-byte pieces. begin(j) and end(j) come before and behind the values
    // of 32 rows; put(i, j, q) gives the two words of four values.
    template <class P>
    __device__ __forceinline__ void turn(tp_lds* s, int j, const P& put) const {
        typedef uint32_t u2 __attribute__((ext_vector_type(2)));
        typedef __attribute__((address_space(3))) u2 l2;
        const uint32_t l = (uint32_t)zs_lane(), n = l & 31u;
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const uint2 v = put(i, j, q);
                const uint32_t c = i * 4u + q;
                *(l2*)(s + n * (64 * MT) + (c ^ (n & (4u * MT - 1u))) * 16u + (l >> 5) * 8u) = u2{v.x, v.y};
            }
    }
    __device__ __forceinline__ static tp_lds* mine() {   // the wave's share of the memory, room for 32 rows
        static_assert(32 * 64 * MT <= STAGE / 2 && 32 * 128 <= STAGE / 2, "32 rows of a wave's values fit its share of the memory");
        const uint32_t w = (uint32_t)__builtin_amdgcn_readfirstlane(zs_wid());
        return stage(w >> 1) + (w & 1u) * (STAGE / 2);
    }
    // row(r, m, v) takes eight values of the wave's row r from its column m on
    template <class J, class P, class E, class R>
    __device__ __forceinline__ void rows(const J& begin, const P& put, const E& end, const R& row) const {
        constexpr uint32_t C = 4 * MT;   // 16-byte pieces of a row
        typedef uint32_t u4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) u4 l4;
        tp_lds* s = mine();
        const uint32_t l = (uint32_t)zs_lane();
#pragma unroll
        for (int j = 0; j < NT; j++) {
            begin(j);
            turn(s, j, put);
            end(j);
#pragma unroll
            for (uint32_t t = 0; t < 32u; t += 64u / C) {
                const uint32_t r = t + l / C, c = l % C;
                row(j * 32u + r, c * 8u, *(const l4*)(s + r * (64 * MT) + (c ^ (r & (C - 1u))) * 16u));
            }
        }
    }
    // The same of f32 numbers, 32 x 32 at a time: get(i, j, q) gives four values,
    // at(r) is where the wave's row r goes with its `count` columns, NULL for nowhere;
    // PAST: past the caches (of two stores at run time the compiler makes an ordinary one).
    // (One f32 row's gradient of 58134 x 3456 weights, from the lanes as they have the
    // values and so: 337 and 241 us.)
    template <bool PAST, class P, class R>
    __device__ __forceinline__ void words(const P& get, const R& at, uint32_t count) const {
        typedef float f4 __attribute__((ext_vector_type(4)));
        typedef float f4a __attribute__((ext_vector_type(4), aligned(4)));   // (a row may begin at any number)
        typedef __attribute__((address_space(3))) f4 l4;
        tp_lds* s = mine();
        const uint32_t l = (uint32_t)zs_lane(), n = l & 31u;
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int i = 0; i < MT; i++) {
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const float4 v = get(i, j, q);
                    *(l4*)(s + n * 128u + (((uint32_t)q * 2u + (l >> 5)) ^ (n & 7u)) * 16u) = f4{v.x, v.y, v.z, v.w};
                }
#pragma unroll
                for (uint32_t t = 0; t < 4u; t++) {
                    const uint32_t r = t * 8u + (l >> 3), c = l & 7u, m = (uint32_t)i * 32u + c * 4u;
                    float* p = at((uint32_t)j * 32u + r);
                    const f4 v = *(const l4*)(s + r * 128u + (c ^ (r & 7u)) * 16u);
                    if (!p) continue;
                    if (m + 4u <= count) {
                        if constexpr (PAST) __builtin_nontemporal_store((f4a)v, (f4a*)(p + m));
                        else *(f4a*)(p + m) = v;
                    } else
                        for (uint32_t k = 0; m + k < count; k++) p[m + k] = v[k];
                }
            }
    }
    // the order of half a step's instructions: reads and V loads evenly between the products
    template <int V, int I = 0>
    __device__ __forceinline__ static void sched() {
#if defined(__HIP_DEVICE_COMPILE__)
        constexpr int M = MT * NT, D = MT * (AS ? 2 : 1) + NT * (BS ? 2 : 1);
        constexpr int d = (I + 1) * D / M - I * D / M, v = (I + 1) * V / M - I * V / M;
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if constexpr (d > 0) __builtin_amdgcn_sched_group_barrier(0x100, d, 0);
        if constexpr (v > 0) __builtin_amdgcn_sched_group_barrier(0x020, v, 0);
        if constexpr (I + 1 < M) sched<V, I + 1>();
#endif
    }
};

// x within bf16's range (what is past it, or no number, shows in what is left of x)
__device__ __forceinline__ float tp_bf16_below(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
    const float m = __uint_as_float(0x7f7f0000u);
    return __builtin_amdgcn_fmed3f(x, -m, m);
#else
    return x;
#endif
}

// The same product with an f32 A that lies in memory as it is (ANY: its rows at any
// number, fetched one by one, not by 16 bytes) and three planes of B: 128 x 64 a
// workgroup, each wave's 32 rows of A split into planes in its registers (52
// instructions for 16 columns of 32 rows, beside 12 products of them). Where there
// are few n: nothing of A is written and read again. ld, k and rows of A's tp_mat
// count f32 numbers.
template <bool SLOW, bool ANY>
struct tp_raw_tile {
    static constexpr int M = 1, N = 2, BM = 128, BN = 64;
    static constexpr int SA = BM * 128, SB = BN * 64, STAGE = SA + 3 * SB;
    typedef tp_side<BN, false> B;
    const tp_mat &ma, &mb;
    B b;
    const char* base;
    static constexpr int L = ANY ? 16 : 4, G = ANY ? 4 : 16;   // a lane's loads of A a step, bytes of each
    uint32_t m0, n0, off[SLOW && ANY ? 2 : SLOW ? 4 : L], ka, kmax, ld4, rd;

    __device__ __forceinline__ static uint32_t wm() { return (uint32_t)__builtin_amdgcn_readfirstlane(zs_wid()); }
    __device__ __forceinline__ static uint32_t wn() { return 0; }
    __device__ __forceinline__ uint32_t n_of(int j) const { return n0 + (uint32_t)j * 32u + ((uint32_t)zs_lane() & 31u); }
    __device__ __forceinline__ uint32_t m_of(int i, int q) const {
        return m0 + wm() * 32u + (uint32_t)i * 32u + (uint32_t)q * 8u + ((uint32_t)zs_lane() >> 5) * 4u;
    }
    __device__ __forceinline__ tp_raw_tile(const tp_mat& ma_, const tp_mat& mb_, uint32_t m, uint32_t n) : ma(ma_), mb(mb_), m0(m * BM), n0(n * BN) {
        const uint32_t l = (uint32_t)zs_lane(), w = wm(), r = l & 31u, h = l >> 5;
        b.start(mb, n0, 0);
        ld4 = (uint32_t)ma.ld * 4u;
        if constexpr (!SLOW) {
            // row r's eight 16-byte pieces at r * 128 B, piece c in place c ^ (r & 7)
            const uint32_t x = m0 < ma.rows ? m0 : ma.rows - 1u;
            base = (const char*)ma.p[0] + (uint64_t)x * ld4;
            // load i of wave w fetches rows from (i * 4 + w) * R on, R a load
            constexpr uint32_t R = 64u * G / 128u, PER = 64u / R;
            kmax = ma.k * 4u - G;
            const uint32_t rl = l / PER;
            // (a row's place among eight, the same for all i)
            const uint32_t r7 = ANY ? (w * 2u + rl) & 7u : rl & 7u;
            ka = ANY ? ((((l & 31u) >> 2) ^ r7) * 4u + (l & 3u)) * 4u : ((l & 7u) ^ r7) * 16u;
#pragma unroll
            for (int i = 0; i < L; i++) {
                uint32_t row = m0 + ((uint32_t)i * 4u + w) * R + rl;
                row = row < ma.rows ? row : ma.rows - 1u;
                off[i] = (row - x) * ld4;
            }
            rd = (w * 32u + r) * 128u + (r & 7u) * 16u;      // (place of piece 0; piece c's is that ^ 16 c)
        } else {
            // row k's 32 pieces at k * 512 B, piece c in place c ^ (k & 8)
            base = (const char*)ma.p[0] + (uint64_t)m0 * 4u;
            if constexpr (!ANY) {
                const uint32_t last = (ma.rows >> 2) - 1u - (m0 >> 2);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t k = (uint32_t)i * 8u + w * 2u + h;
                    const uint32_t c = (l & 31u) ^ (k & 8u);
                    off[i] = (c < last ? c : last) * 16u;
                }
            } else {
                // a load: half of a row, k = (i * 4 + w) / 2; pieces moved by 8 are the other 32 numbers of the half
                const uint32_t last = ma.rows - 1u - m0;
#pragma unroll
                for (int z = 0; z < 2; z++) {
                    const uint32_t e = ((w & 1u) * 64u + l) ^ (uint32_t)z * 32u;
                    off[z] = (e < last ? e : last) * 4u;
                }
            }
            ka = ANY ? w >> 1 : w * 2u + h;
            kmax = ma.k;
            rd = h * 8u * 512u + ((w * 32u + r) * 4u ^ h * 128u);
        }
    }
    __device__ __forceinline__ static tp_lds* stage(uint32_t i) {
        __shared__ char s0_[STAGE], s1_[STAGE];
        return i == 0u ? (tp_lds*)s0_ : (tp_lds*)s1_;
    }
    __device__ __forceinline__ static void fetch(const char* p, tp_lds* s) {
#if defined(__HIP_DEVICE_COMPILE__)
        // (the size has to be a number as it stands)
        if constexpr (ANY) __builtin_amdgcn_global_load_lds((tp_glb*)p, s, 4, 0, 0);
        else __builtin_amdgcn_global_load_lds((tp_glb*)p, s, 16, 0, 0);
#endif
    }
    __device__ __forceinline__ void put(uint32_t kt, tp_lds* s) {
#if defined(__HIP_DEVICE_COMPILE__)
        const uint32_t w = wm();
        if constexpr (!SLOW) {
            uint32_t k = kt * 128u + ka;
            k = k < kmax ? k : kmax;
#pragma unroll
            for (int i = 0; i < L; i++) fetch(base + (off[i] + k), s + (i * 256 * G + w * 64u * G));
        } else {
            const uint32_t k0 = kt * 32u < kmax ? kt * 32u : kmax - 1u, end = kmax - 1u - k0;
            const char* p = base + (uint64_t)k0 * ld4;
#pragma unroll
            for (int i = 0; i < L; i++) {
                uint32_t k = ka + (uint32_t)i * (ANY ? 2u : 8u);
                // (a row's number is that of its place: the clamped one's pieces stay where the row's own would)
                const uint32_t o = ANY ? off[(i >> 2) & 1] : off[i & 3];
                k = k < end ? k : end;
                fetch(p + (uint64_t)k * ld4 + o, s + (i * 256 * G + w * 64u * G));
            }
        }
#pragma unroll
        for (int q = 0; q < 3; q++) {
            b.plane(mb, q, n0);
            b.load(kt, s + SA + q * SB);
        }
#endif
    }
    // 16 columns ks of the wave's rows as planes: lane l has row l % 32, k (l / 32) * 8 on
    __device__ __forceinline__ void split(const tp_lds* s, int ks, tp_s8 (&p)[3]) const {
        typedef float f4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) f4 l4;
        typedef __attribute__((address_space(3))) float l1;
        float x[8];
        if constexpr (!SLOW) {
            const uint32_t h = (uint32_t)zs_lane() >> 5;
            const uint32_t c = (uint32_t)ks * 4u + h * 2u;
            const f4 u = *(const l4*)(s + (rd ^ (c * 16u))), v = *(const l4*)(s + (rd ^ ((c + 1u) * 16u)));
#pragma unroll
            for (int k = 0; k < 4; k++) x[k] = u[k], x[k + 4] = v[k];
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) x[k] = *(const l1*)(s + rd + (ks * 16 + k) * 512);
        }
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        typedef uint32_t u4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int q = 0; q < 3; q++) {
            u4 o;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                // (the first: of a number that bf16 would make infinite the one below it)
                const b2 v = {(__bf16)(q ? x[2 * k] : tp_bf16_below(x[2 * k])), (__bf16)(q ? x[2 * k + 1] : tp_bf16_below(x[2 * k + 1]))};
                o[k] = __builtin_bit_cast(uint32_t, v);
                if (q < 2) {
                    x[2 * k] -= __uint_as_float(o[k] << 16);
                    x[2 * k + 1] -= __uint_as_float(o[k] & 0xffff0000u);
                }
            }
            p[q] = __builtin_bit_cast(tp_s8, o);
        }
    }
    __device__ __forceinline__ void mul(const tp_lds* s, tp_acc (&c)[1][2]) const {
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            tp_s8 x[3];
            split(s, ks, x);
#pragma unroll
            for (int e = 0; e < 6; e++) {
                constexpr uint32_t A = tp_planes<TP_THREE>::A, P = tp_planes<TP_THREE>::B;
                const int pa = (int)(A >> (4 * e)) & 15, pb = (int)(P >> (4 * e)) & 15;
#pragma unroll
                for (int j = 0; j < 2; j++) c[0][j] = tp_mfma<TP_THREE>(x[pa], b.frag(s + SA + pb * SB, j, ks), c[0][j]);
            }
        }
    }
    template <class F = tp_none>
    __device__ __forceinline__ void run(uint32_t k0, uint32_t n, tp_acc (&c)[1][2], const F& beside = F()) {
        tp_lds *s0 = stage(0), *s1 = stage(1);
        if (n == 0u) return;
        put(k0, s0);
        beside();
        uint32_t k = 1u;
        for (; k < n; k += 2u) {
            tp_arrived<0, true>();
            put(k0 + k, s1);
            mul(s0, c);
            tp_arrived<0, true>();
            if (k + 1u < n) put(k0 + k + 1u, s0);
            mul(s1, c);
        }
        if (k == n) {
            tp_arrived<0, true>();
            mul(s0, c);
        }
        tp_arrived<0, true>();
    }
};

// Workgroup id's place among n pieces of work (~0: none). Workgroups id, id + 8,
// ... run on one XCD: each XCD has a run of pieces of its own.
__device__ __forceinline__ uint32_t tp_place(uint32_t id, uint32_t n) {
    const uint32_t per = (n + 7u) >> 3, t = (id & 7u) * per + (id >> 3);
    return (id >> 3) >= per || t >= n ? ~0u : t;
}
inline uint32_t tp_places(uint32_t n) { return (n + 7u) / 8u * 8u; }
// Tile t of mt x nt, in groups of four along m, n by n, so that the tiles in an
// XCD's CUs share their operands in its L2.
__device__ __forceinline__ uint2 tp_order(uint32_t t, uint32_t mt, uint32_t nt) {
    const uint32_t g = t / (4u * nt), gm = mt - g * 4u < 4u ? mt - g * 4u : 4u, r = t - g * 4u * nt;
    return make_uint2(g * 4u + r % gm, r / gm);
}
