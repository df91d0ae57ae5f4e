// zs_beam_merge.h -- the step of one request from the heads of its beams' rows.
#pragma once
#include "zs_dev.h"
#include "zs_beam.h"

// ---------------------------------------------------------------------------
// The step of one request by one wave, the lists read and scored by four. The
// rows' heads are sorted, so the
// candidates' order is a merge of at most 32 lists (held in LDS): lane b has the
// score of beam b's next candidate, each turn takes the largest (the lowest
// beam of equals). A row needs width + n_eos entries: its first `width` that do not
// end are among them, and so is every EOS id among the first `width` overall.
// ---------------------------------------------------------------------------
__device__ __forceinline__ bool bm_is_eos(const bm_args& a, uint32_t id) {
    bool e = false;
#pragma unroll
    for (uint32_t i = 0; i < ZS_BEAM_MAX_EOS; i++) e |= i < a.n_eos && a.eos[i] == id;
    return e;
}

#define BM_NT 256
__device__ __forceinline__ void bm_merge(const bm_args& a, uint32_t g) {
    constexpr int NL = ZS_BEAM_MAX_WIDTH * (ZS_BEAM_MAX_WIDTH + ZS_BEAM_MAX_EOS) / BM_NT;   // entries a thread at most
    __shared__ uint2 c_[ZS_BEAM_MAX_WIDTH * (ZS_BEAM_MAX_WIDTH + ZS_BEAM_MAX_EOS)];       // the lists' scores (keys; 0: none) and ids
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
    unsigned long long e[NL];
#pragma unroll
    for (int k = 0; k < NL; k++) {
        const uint32_t i = lane + (uint32_t)k * BM_NT;
        e[k] = i < W * K ? __hip_atomic_load(a.list + at * K + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : ~0ull;
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
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NL; k++) {
        const uint32_t i = lane + (uint32_t)k * BM_NT;
        if (i >= W * K) break;
        const uint32_t b = i / K;
        const float bs = bs_[b];
        const bool some = bs > -INFINITY && e[k] != ~0ull;
        const float s = some ? (float)((double)bs + (((double)zs_u2f((uint32_t)(e[k] >> 32)) - bm_[b]) - bl_[b])) : -INFINITY;
        c_[i] = make_uint2(s > -INFINITY ? zs_total_key(s + 0.0f) : 0u, (uint32_t)e[k] | (bm_is_eos(a, (uint32_t)e[k]) ? 0x80000000u : 0u));
    }
    __syncthreads();
    if (lane >= 64u) return;
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
    int o_parent = -1, o_token = -1;
    float o_score = -INFINITY;
    uint32_t n_live = 0, n_fin = 0;
    for (uint32_t rank = 0; n_live < W; rank++) {
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
