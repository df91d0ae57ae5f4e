// zs_head.hip -- the head of a row of logits: its K largest values with their
// ids and its log-normaliser, for a teacher's lists (zs_teacher_topk) and for
// the beam step (zs_beam.hip).
//
// One pass over the logits (zs_k_head_scan, the whole GPU): every wave takes
// 2048 values into registers, leaves the largest value of each group of 2^gs
// of them and its own maximum m with sum exp((x - m) / T). Then one workgroup
// a row (zs_k_head_pick): ln sum from the waves' records, and a key that at
// least K groups reach, so that the K largest values lie in the groups whose
// maximum reaches it, a few more than K, whose values are read again, listed
// and sorted.
#include "zs_head.h"
#include "zs_select.h"
#include "zs_beam_merge.h"

// ---------------------------------------------------------------------------
// the pass
// ---------------------------------------------------------------------------
#define HS_NT 256

// A value's key for maxima: 0 for what is not above -inf, after hs_cut.
__device__ __forceinline__ uint32_t hs_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ (uint32_t)((int)b >> 31 | (int)0x80000000);
}
__device__ __forceinline__ uint32_t hs_cut(uint32_t k) { return k > 0x007fffffu ? k : 0u; }   // (-inf's)
// Maximum over LG neighbouring lanes (of integers: the move is part of the
// maximum's instruction; of floats it takes two more).
template <int LG>
__device__ __forceinline__ uint32_t hs_max(uint32_t k) {
    k = zs_group_max<LG < 16 ? LG : 16>(k);
    if constexpr (LG >= 32) k = max(k, zs_lane_xor<16>(k));
    if constexpr (LG >= 64) k = max(k, zs_lane_xor<32>(k));
    return k;
}

// LG: lanes of a group. The exponentials and what goes with them bound the
// pass over 16-bit values, not their bytes: a value takes one shift or mask,
// half a maximum, one fma, one exponential (a quarter of the rate) and one
// addition; sums are relative to each thread's own maximum. 2048 x 151936 bf16:
// 102 us, 6.1 TB/s, the vector units busy for 85 % of them; over f32 they are for
// half, and memory bounds the pass: 1024 x 151936 100 us, 6.2 TB/s (a large read
// reaches 7.2).
template <int DT, int LG, bool MASK>
__global__ __launch_bounds__(HS_NT) void zs_k_head_scan(hd_args a, uint64_t r0) {
    constexpr int E = hd_elem<DT>::E, U = HD_WAVE / 64 / E;
    const uint32_t n = zs_quot(blockIdx.x, a.by_chunks), chunk = blockIdx.x - n * a.chunks;
    const uint64_t r = r0 + n;
    if (a.count && chunk == 0 && threadIdx.x == 0) {
        const uint32_t g = zs_quot((uint32_t)r, a.by_width);
        if (g * a.width == (uint32_t)r) a.count[g] = 0;
    }
    if (!hd_live(a, r)) return;
    const hd_row<DT> row(a.logits, a.ld, r, a.V);
    const uint32_t t = threadIdx.x, lane = (uint32_t)zs_lane();
    const uint32_t first = chunk * (U * HS_NT), j0 = first + t;
    if (first >= row.nvec) return;
    uint32_t g[U];
    float m, s;
    auto pass = [&](bool clean) {
        float x[U][E];
        {
            hd_u4 v[U];
            row.take(j0, HS_NT, row.inside(first) && row.inside(first + U * HS_NT - 1u), v);
            uint32_t b[U];
            if (MASK) {
                const uint32_t* allow = a.allow + r * a.allow_words;
#pragma unroll
                for (int u = 0; u < U; u++) b[u] = hd_allow<E>(allow, a.allow_words, row.id0(j0 + (uint32_t)u * HS_NT));
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                hd_unpack<DT>(v[u], x[u]);
#pragma unroll
                for (int q = 0; q < E; q++) {
                    if (MASK) x[u][q] = b[u] >> q & 1u ? x[u][q] : -INFINITY;
                    if (clean) x[u][q] = hd_clean(x[u][q]);
                }
            }
        }
        m = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; u++) {
            float vm = x[u][0];
#pragma unroll
            for (int q = 1; q < E; q++) vm = fmaxf(vm, x[u][q]);
            m = fmaxf(m, vm);
            g[u] = hs_key(vm);
        }
        // 2^(x c - mc): one fma a value; mc's rounding is a factor of all of them
        const float mr = m > -INFINITY ? m : 0.0f, c = hd_factor(mr, a.c), mc = mr * c;
        s = 0.0f;
#pragma unroll
        for (int u = 0; u < U; u++) {
            float e[E];
#pragma unroll
            for (int q = 0; q < E; q++) e[q] = __builtin_amdgcn_exp2f(fmaf(x[u][q], c, -mc));
            s += hd_sum(e);
        }
        const float M = wave_max_f(m), Mr = M > -INFINITY ? M : 0.0f, cM = hd_factor(Mr, a.c), Mc = Mr * cM;
        s *= m == M ? 1.0f : m > -INFINITY && c == cM ? __builtin_amdgcn_exp2f(mc - Mc) : 0.0f;
        m = M;
        s = zs_wave_reduce(s, [](float p, float q) { return p + q; }) * __builtin_amdgcn_exp2f(-fmaf(Mr, cM, -Mc));
    };
    pass(false);
    if (!(s < INFINITY)) pass(true);   // NaN or +inf among the values
    if (lane == 0) a.rec[r * a.recs + chunk * (HD_CHUNK / HD_WAVE) + (uint32_t)zs_wid()] = make_float2(m, s);
    // a group's lanes store their vectors' groups in turn
    uint32_t* gmax = a.gmax + r * a.gstride;
    constexpr int ST = LG < U ? LG : U;
    const uint32_t i = lane & (uint32_t)(LG - 1);
#pragma unroll
    for (int u = 0; u < U; u++) g[u] = hs_max<LG>(g[u]);
#pragma unroll
    for (int u = 0; u < U; u += ST) {
        uint32_t k = g[u];
#pragma unroll
        for (int w = 1; w < ST; w++) k = i == (uint32_t)w ? g[u + w] : k;
        const uint32_t j = j0 + ((uint32_t)u + i) * HS_NT;
        if (i < (uint32_t)ST && j - i < row.nvec) gmax[j / LG] = hs_cut(k);
    }
}

// ---------------------------------------------------------------------------
// the pick
// ---------------------------------------------------------------------------
// Bound by a chain of waits, not by what it moves: the groups' maxima (0.5 us),
// their sort and threshold (0.5), the list of groups (0.6), their values from
// memory (1.2), the places (1): 4 us of a row; the kernel of a row alone takes 5
// to 6 (K = 16 of 50257 f32; K = 64 of 151936 bf16 11), of 2048 rows 29, of which
// a third is the wait for the groups' values; the normaliser's exponentials and
// logarithm are taken beside it by the last wave.
#define HP_NT 256
#define HP_GPT (HD_GROUPS / HP_NT)   // groups per thread at most
#define HP_GL 512                    // listed groups at most (rows in no order: K + 20 to K + 80, of K = 128 up to 270;
                                     // K = 128 of 2048 rows of 50257 f32: 110 us, with 256 of them 126)
#define HP_LIST 1024                 // listed values at most

// Places of the set bits (place t + e * HP_NT for bit e) in ascending order.
template <int E>
__device__ __forceinline__ uint32_t hp_places(uint32_t bits, uint32_t* out, uint32_t* cnt) {
    constexpr uint32_t NW = HP_NT / 64;
    const uint32_t lane = (uint32_t)zs_lane(), wid = (uint32_t)zs_wid();
#pragma unroll
    for (int e = 0; e < E; e++) {
        const uint32_t n = (uint32_t)__popcll(__ballot(bits >> e & 1u));
        if (lane == 0) cnt[(uint32_t)e * NW + wid] = n;
    }
    __syncthreads();
    uint32_t run = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const unsigned long long m = __ballot(bits >> e & 1u);
        uint32_t before = run;
#pragma unroll
        for (uint32_t w = 0; w < NW; w++) {
            const uint32_t c = cnt[(uint32_t)e * NW + w];
            before += w < wid ? c : 0u;
            run += c;
        }
        if (bits >> e & 1u) out[before + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u))] =
            threadIdx.x + (uint32_t)e * HP_NT;
    }
    __syncthreads();
    return run;
}

template <int DT, bool MASK>
__device__ __forceinline__ void hp_pick(const hd_args& a, uint64_t r, uint32_t lgs) {
    constexpr int E = hd_elem<DT>::E;
    constexpr uint32_t NW = HP_NT / 64;
    __shared__ unsigned long long list[HP_LIST];
    __shared__ uint32_t gl[HP_GL], pl[ZS_TEACHER_KMAX];
    __shared__ uint32_t hist[256], u[4], wthr[NW];
    __shared__ hd_norm norm;
    const hd_row<DT> row(a.logits, a.ld, r, a.V);
    const uint32_t* allow = MASK ? a.allow + r * a.allow_words : nullptr;
    const uint32_t t = threadIdx.x, lane = (uint32_t)zs_lane(), wid = (uint32_t)zs_wid(), K = a.K;
    const uint32_t ng = (row.nvec + (1u << lgs) - 1u) >> lgs;
    const uint32_t* gm = a.gmax + r * a.gstride;
    // thread t of wave w holds groups 4 lane + w + 256 e: the groups of a short
    // row fall on all waves alike
    uint32_t k[HP_GPT], tm = 0;
#pragma unroll
    for (int e = 0; e < HP_GPT; e++) {
        const uint32_t g = NW * lane + wid + (uint32_t)e * HP_NT;
        k[e] = (uint32_t)e * HP_NT < ng ? zs_gload(gm + min(g, ng - 1u)) : 0u;
        if (g >= ng) k[e] = 0u;
    }
    // The row's normaliser, by the last wave: its records are read here (two a
    // lane at once: rows of 262144 ids; longer ones take turns), and summed where
    // that wave has nothing else to do (in front of the list the others waited for it).
    const uint32_t recs = (row.nvec * E + HD_CHUNK - 1u) / HD_CHUNK * (HD_CHUNK / HD_WAVE);
    const float2* rec = a.rec + r * a.recs;
    float2 v[2];
#pragma unroll
    for (int w = 0; w < 2; w++) {
        const uint32_t i = lane + 64u * (uint32_t)w;
        v[w] = wid == NW - 1u && i < recs ? rec[i] : make_float2(-INFINITY, 0.0f);
    }
    auto normalise = [&]() {
        if (wid != NW - 1u) return;
        float m = fmaxf(v[0].x, v[1].x);
        for (uint32_t i = lane + 128u; i < recs; i += 64u) m = fmaxf(m, rec[i].x);
        m = wave_max_f(m);
        double s = 0.0;
        auto add = [&](float2 o) { if (o.x > -INFINITY) s += (double)o.y * exp(((double)o.x - (double)m) * a.inv_t); };
        add(v[0]);
        add(v[1]);
        for (uint32_t i = lane + 128u; i < recs; i += 64u) add(rec[i]);
        s = wave_sum_d(s);
        if (lane == 0) norm = {(double)m, log(s)};
    };
#pragma unroll
    for (int e = 0; e < HP_GPT; e++) {
        if ((uint32_t)e * HP_NT >= ng) break;
        tm = max(tm, k[e]);
    }
    if (t < 4) u[t] = 0;
    // theta: in every wave the ceil(K / waves)-th largest thread maximum; the
    // smallest of them is reached by K groups (1: too few hold a candidate, all
    // are listed then)
    const uint32_t srt = wave_sort_u32(tm);
    const uint32_t wt = zs_readlane_u(srt, 64u - (K + NW - 1u) / NW);
    if (lane == 0) wthr[wid] = wt;
    __syncthreads();
    uint32_t theta = wthr[0];
#pragma unroll
    for (uint32_t w = 1; w < NW; w++) theta = min(theta, wthr[w]);
    theta = max(theta, 1u);
    uint32_t reach = 0;
#pragma unroll
    for (int e = 0; e < HP_GPT; e++) {
        if ((uint32_t)e * HP_NT >= ng) break;
        reach |= k[e] >= theta ? 1u << e : 0u;
    }
    if (reach) {
        uint32_t p = atomicAdd(&u[0], (uint32_t)__popc(reach));
        for (; reach; reach &= reach - 1u, p++)
            if (p < HP_GL) gl[p] = NW * lane + wid + ((uint32_t)__ffs((int)reach) - 1u) * HP_NT;
    }
    __syncthreads();
    const uint32_t n_gl = u[0], lm = (1u << lgs) - 1u;
    const float theta_f = theta > 1u ? zs_key_to_float(theta) : -__FLT_MAX__;
    auto keys_of = [&](const float (&x)[E], uint32_t j, uint32_t (&kq)[E]) {
        uint32_t b = ~0u;
        if (MASK) b = hd_allow<E>(allow, a.allow_words, row.id0(j));
#pragma unroll
        for (int q = 0; q < E; q++) kq[q] = b >> q & 1u ? hd_key(hd_clean(x[q])) : 0u;
    };
    auto keys = [&](uint32_t j, uint32_t (&kq)[E]) {
        float x[E];
        row.get(j, x, -INFINITY);
        keys_of(x, j, kq);
    };
    auto entry = [&](uint32_t key, uint32_t j, int q) {
        return ((unsigned long long)(~key) << 32) | (uint32_t)(row.id0(j) + q);
    };
    if (n_gl <= HP_GL) {
        const uint32_t nit = n_gl << lgs;
        // four vectors a thread in flight; those at the row's ends, and all of
        // a row that has no others, are read by `keys`
        constexpr int NU = 4;
        const bool wide = row.nvec >= 3u;
        for (uint32_t i0 = 0; i0 < nit; i0 += NU * HP_NT) {
            hd_u4 v[NU];
            uint32_t jv[NU];
#pragma unroll
            for (int w = 0; w < NU; w++) {
                const uint32_t i = i0 + t + (uint32_t)w * HP_NT;
                jv[w] = i < nit ? (gl[i >> lgs] << lgs) + (i & lm) : row.nvec;
                if (wide) v[w] = row.load(row.inside(jv[w]) ? jv[w] : 1u);
            }
#pragma unroll
            for (int w = 0; w < NU; w++) {
                if (i0 + (uint32_t)w * HP_NT >= nit) break;
                const uint32_t j = jv[w];
                float x[E];
                if (wide && row.inside(j)) hd_unpack<DT>(v[w], x);
                else if (j < row.nvec) row.get(j, x, -INFINITY);
                else {
#pragma unroll
                    for (int q = 0; q < E; q++) x[q] = -INFINITY;
                }
                if (MASK) {
                    const uint32_t b = j < row.nvec ? hd_allow<E>(allow, a.allow_words, row.id0(j)) : 0u;
#pragma unroll
                    for (int q = 0; q < E; q++) x[q] = b >> q & 1u ? x[q] : -INFINITY;
                }
                // (one atomic a wave: one a lane is served lane by lane; NaN reaches nothing)
                uint32_t p = 0, n = 0;
#pragma unroll
                for (int q = 0; q < E; q++) {
                    const unsigned long long m = __ballot(x[q] >= theta_f);
                    p = __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, p));
                    n += (uint32_t)__popcll(m);
                }
                if (!n) continue;
                uint32_t p0 = 0;
                if (lane == 0) p0 = atomicAdd(&u[1], n);
                p += (uint32_t)__builtin_amdgcn_readfirstlane((int)p0);
#pragma unroll
                for (int q = 0; q < E; q++) {
                    if (!(x[q] >= theta_f)) continue;
                    if (p < HP_LIST) list[p] = entry(hd_key(hd_clean(x[q])), j, q);
                    p++;
                }
            }
        }
    }
    __syncthreads();
    uint32_t n = u[1];
    if (n_gl > HP_GL || n > HP_LIST) {
        // Many groups or values reach theta (sorted rows, equal values). The
        // first K values lie in the first K groups by (maximum descending,
        // group ascending): K groups in front of another hold K values in front
        // of any of its. The same holds of the groups' parts, down to single
        // vectors: level by level, 16 parts of a group at most.
        __syncthreads();
#pragma unroll
        for (int e = 0; e < HP_GPT; e++) {   // (places in group order here)
            const uint32_t g = t + (uint32_t)e * HP_NT;
            k[e] = g < ng ? zs_gload(gm + g) : 0u;
        }
        uint32_t ngl = hp_places<HP_GPT>(zs_first<HP_NT, HP_GPT>(k, K, hist, u), gl, hist);
        constexpr int NP = ZS_TEACHER_KMAX * 16 / HP_NT;
        for (uint32_t lg = lgs; lg > 0;) {
            const uint32_t lp = lg > 4u ? 4u : lg;
            lg -= lp;
            const uint32_t lm = (1u << lp) - 1u;
            uint32_t pk[NP];
#pragma unroll
            for (int w = 0; w < NP; w++) {
                const uint32_t i = t + (uint32_t)w * HP_NT;
                pk[w] = 0u;
                if (i >= ngl << lp) continue;
                const uint32_t part = (gl[i >> lp] << lp) + (i & lm);
                for (uint32_t j = part << lg; j < (part + 1u) << lg && j < row.nvec; j++) {
                    uint32_t kq[E];
                    keys(j, kq);
#pragma unroll
                    for (int q = 0; q < E; q++) pk[w] = max(pk[w], kq[q]);
                }
            }
            ngl = hp_places<NP>(zs_first<HP_NT, NP>(pk, K, hist, u), pl, hist);
            const uint32_t part = t < ngl ? (gl[pl[t] >> lp] << lp) + (pl[t] & lm) : 0u;
            __syncthreads();
            if (t < ngl) gl[t] = part;
            __syncthreads();
        }
        if (t < ngl) {
            uint32_t kq[E];
            keys(gl[t], kq);
#pragma unroll
            for (int q = 0; q < E; q++) list[t * E + (uint32_t)q] = kq[q] ? entry(kq[q], gl[t], q) : ~0ull;
        }
        n = ngl * E;
        __syncthreads();
    }
    static_assert(ZS_TEACHER_KMAX * 8 <= HP_LIST && ZS_TEACHER_KMAX <= HP_GL, "the first K groups and their vectors' values fit");
    if (n <= 2u * HP_NT) {
        // an entry's place is the number of entries in front of it; entries of no
        // candidate (~0 all) lie behind the others as they stand. (K = 64 of
        // 256 rows of 20000: 13.5 us, sorted 17.1)
        auto put = [&](uint32_t at) {
            unsigned long long e = ~0ull;
            uint32_t place = at;
            if (at < n) {
                e = list[at];
                place = 0;
                uint32_t i = 0;
                for (; i + 4u <= n; i += 4u) {
#pragma unroll
                    for (int q = 0; q < 4; q++) place += list[i + (uint32_t)q] < e ? 1u : 0u;
                }
                for (; i < n; i++) place += list[i] < e ? 1u : 0u;
                if (e == ~0ull)
                    for (i = 0; i < at; i++) place += list[i] == ~0ull ? 1u : 0u;
            }
            return place | (e == ~0ull ? 1u << 31 : 0u);
        };
        const uint32_t p0 = put(t), p1 = n > HP_NT ? put(t + HP_NT) : 1u << 31;
        normalise();
        __syncthreads();
        hd_put(a, r, p0 & 0x7fffffffu, p0 >> 31 ? ~0ull : list[t], norm);
        if (!(p1 >> 31)) hd_put(a, r, p1, list[t + HP_NT], norm);
        return;
    }
    normalise();
    for (uint32_t i = n + t; i < HP_LIST; i += HP_NT) list[i] = ~0ull;
    __syncthreads();
    block_sort_reg_u64<HP_NT, HP_LIST / HP_NT>(list, HP_LIST);
    hd_put(a, r, t, list[t], norm);
}

// BEAM: the workgroup that is the last of its request's takes the step.
template <int DT, bool MASK, bool BEAM>
__global__ __launch_bounds__(HP_NT, 6) void zs_k_head_pick(hd_args a, bm_args m, uint64_t r0, uint32_t lgs) {
    const uint64_t r = r0 + blockIdx.x;
    if (hd_live(a, r)) hp_pick<DT, MASK>(a, r, lgs);
    if (!BEAM) return;
    __shared__ uint32_t last;
    const uint32_t g = zs_quot((uint32_t)r, a.by_width);
    // The list goes past the L2 (hd_put) and is waited for before the count; a
    // release of the whole L2 by every workgroup took 3 times the pick's time
    // (32 x 32 beams: 93 us instead of 32).
    __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0)
    __syncthreads();
    if (threadIdx.x == 0)
        last = __hip_atomic_fetch_add(&a.count[g], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.width - 1u ? 1u : 0u;
    __syncthreads();
    if (!last) return;
    bm_merge(m, g);
}

int hd_head_launch(const hd_args& a, const bm_args* m, uint32_t dtype, hipStream_t stream) {
    const uint32_t gs = hd_group_shift(a.V, a.K), lgs = gs - (dtype == ZS_F32 ? 2u : 3u);
    const uint64_t per = HD_BLOCKS / a.chunks;
    for (uint64_t r0 = 0; r0 < a.R; r0 += per) {
        const uint32_t n = (uint32_t)(a.R - r0 < per ? a.R - r0 : per);
#define HP_GO(DT, MASK)                                                                                                            \
    if (m) hipLaunchKernelGGL((zs_k_head_pick<DT, MASK, true>), dim3(n), dim3(HP_NT), 0, stream, a, *m, r0, lgs);                   \
    else hipLaunchKernelGGL((zs_k_head_pick<DT, MASK, false>), dim3(n), dim3(HP_NT), 0, stream, a, bm_args{}, r0, lgs);
#define HS_GO(DT, LG)                                                                                                              \
    if (a.allow) {                                                                                                                 \
        hipLaunchKernelGGL((zs_k_head_scan<DT, LG, true>), dim3(n * a.chunks), dim3(HS_NT), 0, stream, a, r0);                     \
        HP_GO(DT, true)                                                                                                            \
    } else {                                                                                                                       \
        hipLaunchKernelGGL((zs_k_head_scan<DT, LG, false>), dim3(n * a.chunks), dim3(HS_NT), 0, stream, a, r0);                    \
        HP_GO(DT, false)                                                                                                           \
    }
#define HS_GS(DT, L4)                                                                                                              \
    if (gs == 4) { HS_GO(DT, L4) } else if (gs == 6) { HS_GO(DT, L4 * 4) } else { HS_GO(DT, L4 * 16) }
        if (dtype == ZS_F32) { HS_GS(ZS_F32, 4) }
        else if (dtype == ZS_F16) { HS_GS(ZS_F16, 2) }
        else { HS_GS(ZS_BF16, 2) }
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
