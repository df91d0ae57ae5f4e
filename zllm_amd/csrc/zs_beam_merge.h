// zs_beam_merge.h -- the step of one request from the heads of its beams' rows.
#pragma once
#include "zs_dev.h"
#include "zs_beam.h"

// ---------------------------------------------------------------------------
// The step of one request by one workgroup. A row needs width + n_eos entries:
// its first `width` that do not end are among them, and so is every EOS id
// among the first `width` overall. Candidates that can matter are those at or
// above a key that at least `width` others reach; as a rule they are few
// (32 beams: 40 to 60 of 1056), and each is placed by the number of candidates
// in front of it. Where they are more than a list holds (equal scores), one wave
// merges the rows' lists, which are sorted, a candidate a turn (a turn takes 600
// cycles: 32 beams took 20000 that way, 5000 as here).
// ---------------------------------------------------------------------------
__device__ __forceinline__ bool bm_is_eos(const bm_args& a, uint32_t id) {
    bool e = false;
#pragma unroll
    for (uint32_t i = 0; i < ZS_BEAM_MAX_EOS; i++) e |= i < a.n_eos && a.eos[i] == id;
    return e;
}

#define BM_NT 256
#define BM_LIST 128   // candidates that are placed by counting at most
__device__ __forceinline__ void bm_merge(const bm_args& a, uint32_t g) {
    constexpr uint32_t NW = BM_NT / 64;
    constexpr int NL = ZS_BEAM_MAX_WIDTH * ((ZS_BEAM_MAX_WIDTH + ZS_BEAM_MAX_EOS + NW - 1) / NW) / 64;   // entries a thread at most
    __shared__ uint2 c_[ZS_BEAM_MAX_WIDTH * (ZS_BEAM_MAX_WIDTH + ZS_BEAM_MAX_EOS)];       // the lists' scores (keys; 0: none) and ids
    __shared__ unsigned long long sel[BM_LIST];
    __shared__ uint32_t cnt[3], thr[NW];   // listed; next beams; finished
    __shared__ float nx_s[ZS_BEAM_MAX_WIDTH];
    __shared__ int nx_p[ZS_BEAM_MAX_WIDTH], nx_t[ZS_BEAM_MAX_WIDTH];
    __shared__ float bs_[ZS_BEAM_MAX_WIDTH];
    __shared__ double bm_[ZS_BEAM_MAX_WIDTH], bl_[ZS_BEAM_MAX_WIDTH];
    __shared__ float fin_s[ZS_BEAM_MAX_WIDTH];
    __shared__ int fin_p[ZS_BEAM_MAX_WIDTH], fin_t[ZS_BEAM_MAX_WIDTH];
    const uint32_t lane = threadIdx.x, W = a.width, K = a.K;
    const size_t at = (size_t)g * W;
    const bool beam = lane < W;
    // all loads at once: what is not needed is dropped afterwards
    const int was = a.done[g], steps = a.steps[g];
    const float score = beam ? a.scores[at + lane] : -INFINITY;
    const double* norm = a.norm + (at + (beam ? lane : 0u)) * 2u;
    const double m = __hip_atomic_load(norm, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const double lns = __hip_atomic_load(norm + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // entry p of a beam is wave p % 4's, neighbouring ones on its neighbouring
    // lanes: a beam that has all that counts is spread over the waves and lanes
    const uint32_t wid = (uint32_t)zs_wid(), wl = (uint32_t)zs_lane(), Kw = (K + NW - 1u) / NW;
    unsigned long long e[NL];
    uint32_t at_[NL];   // b << 8 | p, ~0 for none
#pragma unroll
    for (int k = 0; k < NL; k++) {
        const uint32_t j = wl + (uint32_t)k * 64u, b = zs_quot(j, a.by_kw), p = (j - b * Kw) * NW + wid, i = b * K + p;
        at_[k] = b < W && p < K ? b << 8 | p : ~0u;
        e[k] = at_[k] != ~0u ? __hip_atomic_load(a.list + at * K + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : ~0ull;
    }
    // the pool as it was (threads below W)
    float ps = beam ? a.fin_score[at + lane] : -INFINITY;
    int pl = beam ? a.fin_length[at + lane] : 0, pp = beam ? a.fin_parent[at + lane] : -1, pt = beam ? a.fin_token[at + lane] : -1;
    if (!(ps == ps)) ps = -INFINITY;
    if (beam) {
        // (beams that do not live left no list)
        bs_[lane] = !was && fabsf(score) <= __FLT_MAX__ ? score : -INFINITY;
        bm_[lane] = m;
        bl_[lane] = lns;
        nx_s[lane] = -INFINITY;
        nx_p[lane] = nx_t[lane] = -1;
    }
    if (lane < 3u) cnt[lane] = 0;
    __syncthreads();
    uint32_t key[NL], tm = 0;
#pragma unroll
    for (int k = 0; k < NL; k++) {
        key[k] = 0u;
        if (at_[k] == ~0u) continue;
        const uint32_t b = at_[k] >> 8, id = (uint32_t)e[k];
        const float bs = bs_[b];
        const bool some = bs > -INFINITY && e[k] != ~0ull;
        const float s = some ? (float)((double)bs + (((double)zs_u2f((uint32_t)(e[k] >> 32)) - bm_[b]) - bl_[b])) : -INFINITY;
        const bool eos = bm_is_eos(a, id);
        key[k] = s > -INFINITY ? zs_total_key(s + 0.0f) : 0u;
        if (!eos) tm = max(tm, key[k]);
        c_[b * K + (at_[k] & 255u)] = make_uint2(key[k], id | (eos ? 0x80000000u : 0u));
        // in order: key descending, beam, place in its list; then EOS or not, and the id
        e[k] = (unsigned long long)~key[k] << 32 | b << 27 | (at_[k] & 255u) << 21 | (eos ? 1u << 20 : 0u) | id;
    }
    uint32_t theta = 1u;
    if (W * K > BM_LIST) {   // (as the pick's: every wave has ceil(W / waves) threads that reach its own)
        const uint32_t wt = zs_readlane_u(wave_sort_u32(tm), 64u - (W + NW - 1u) / NW);
        if (wl == 0) thr[wid] = wt;
        __syncthreads();
        theta = thr[0];
#pragma unroll
        for (uint32_t w = 1; w < NW; w++) theta = min(theta, thr[w]);
        theta = max(theta, 1u);
    }
    uint32_t n = 0;
#pragma unroll
    for (int k = 0; k < NL; k++) n += (uint32_t)__popcll(__ballot(key[k] >= theta));
    if (n) {
        uint32_t p = 0;
        if (wl == 0) p = atomicAdd(&cnt[0], n);
        p = (uint32_t)__builtin_amdgcn_readfirstlane((int)p);
#pragma unroll
        for (int k = 0; k < NL; k++) {
            const unsigned long long in = __ballot(key[k] >= theta);
            const uint32_t q = __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, p));
            if (key[k] >= theta && q < BM_LIST) sel[q] = e[k];
            p += (uint32_t)__popcll(in);
        }
    }
    __syncthreads();
    n = cnt[0];
    const bool few = n <= BM_LIST;
    if (few) {
        if (lane < n) {
            const unsigned long long c = sel[lane];
            uint32_t before = 0, ends = 0;
            for (uint32_t i = 0; i < n; i++) {
                const unsigned long long o = sel[i];
                const uint32_t f = o < c ? 1u : 0u;
                before += f;
                ends += f & (uint32_t)o >> 20;
            }
            const uint32_t lo = (uint32_t)c;
            const float cs = zs_key_to_float(~(uint32_t)(c >> 32));
            const int b = (int)(lo >> 27), id = (int)(lo & 0xfffffu);
            if (lo >> 20 & 1u) {
                if (before < W) {
                    fin_s[ends] = cs;
                    fin_p[ends] = b;
                    fin_t[ends] = id;
                    atomicAdd(&cnt[2], 1u);
                }
            } else if (before - ends < W) {
                nx_s[before - ends] = cs;
                nx_p[before - ends] = b;
                nx_t[before - ends] = id;
                atomicAdd(&cnt[1], 1u);
            }
        }
        __syncthreads();
    }
    if (lane >= 64u) return;
    int o_parent = beam ? nx_p[lane] : -1, o_token = beam ? nx_t[lane] : -1;
    float o_score = beam ? nx_s[lane] : -INFINITY;
    uint32_t n_live = cnt[1], n_fin = cnt[2];
    // the beam's next candidate (key 0: none) and the one behind it
    uint2 c = make_uint2(0u, 0u), c2 = c;
    uint32_t next = lane * K;
    const uint32_t end = beam ? next + K : 0u;
    auto step = [&]() {
        c = c2;
        c2 = next < end ? c_[next] : make_uint2(0u, 0u);
        next++;
    };
    step();
    step();
    for (uint32_t rank = 0; !few && n_live < W; rank++) {
        // (beams are in the first 32 lanes: the last lane of the second row has their maximum)
        const uint32_t top = zs_readlane_u(zs_dpp_max<0x142, 0xa>(zs_group_max<16>(c.x)), 31);   // row_bcast:15
        if (!top) break;
        const uint32_t b = (uint32_t)__builtin_ctzll(__ballot(c.x == top));   // the lowest beam of equals
        const float cs = zs_key_to_float(top);
        const uint32_t cid = zs_readlane_u(c.y, b);
        if (cid >> 31) {   // EOS
            if (rank < W) {
                if (lane == 0) { fin_s[n_fin] = cs; fin_p[n_fin] = (int)b; fin_t[n_fin] = (int)(cid & 0x7fffffffu); }
                n_fin++;
            }
        } else {
            if (lane == n_live) { o_parent = (int)b; o_token = (int)cid; o_score = cs; }
            n_live++;
        }
        if (lane == b) step();
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");   // (one wave from here on)
    // the pool and what finished, the pool first among equals: lane i's place
    // is the number of lanes in front of it
    const float len = (float)(steps + 1), div = a.length_penalty == 1.0f ? len : a.length_penalty == 0.0f ? 1.0f : powf(len, a.length_penalty);
    if (lane >= W && lane < W + n_fin && lane < 64u) {
        const uint32_t i = lane - W;
        ps = fin_s[i] / div;
        if (!(ps == ps)) ps = -INFINITY;   // (0 / 0: a length penalty past the floats)
        pl = steps + 1;
        pp = fin_p[i];
        pt = fin_t[i];
    }
    uint32_t place = 0;
    for (uint32_t i = 0; i < W + n_fin; i++) {
        const float o = zs_readlane_f(ps, i);
        place += o > ps || (o == ps && i < lane) ? 1u : 0u;
    }
    const bool stays = lane < W + n_fin && place < W;
    const unsigned long long worst_m = __ballot(stays && place == W - 1u);
    const float worst = worst_m ? zs_readlane_f(ps, (uint32_t)__ffsll((long long)worst_m) - 1u) : -INFINITY;
    const float best = zs_readlane_f(o_score, 0);
    const bool full = worst > -INFINITY;
    const bool done = n_live == 0 || (full && (a.early || worst >= best / div));
    if (stays) {
        const bool some = ps > -INFINITY;
        a.fin_score_o[at + place] = ps;
        a.fin_length_o[at + place] = some ? pl : 0;
        a.fin_parent_o[at + place] = some ? pp : -1;
        a.fin_token_o[at + place] = some ? pt : -1;
    }
    if (beam) {
        a.parent[at + lane] = o_parent;
        a.token[at + lane] = o_token;
        a.score_o[at + lane] = o_score;
    }
    if (lane == 0) {
        a.steps_o[g] = was ? steps : steps + 1;
        a.done_o[g] = was ? was : done ? 1 : 0;
    }
}
