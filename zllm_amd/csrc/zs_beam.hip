// zs_beam.hip -- beam search: the step of a group of beams from the heads of
// their rows (zs_head.hip), and the reordering of the beams' states.
#include "zs_head.h"
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
__global__ __launch_bounds__(BM_NT) void zs_k_beam_merge(bm_args a) {
    constexpr int NL = ZS_BEAM_MAX_WIDTH * (ZS_BEAM_MAX_WIDTH + ZS_BEAM_MAX_EOS) / BM_NT;   // entries a thread at most
    __shared__ float cs_[ZS_BEAM_MAX_WIDTH * (ZS_BEAM_MAX_WIDTH + ZS_BEAM_MAX_EOS)];      // the lists' scores and ids
    __shared__ uint32_t ci_[ZS_BEAM_MAX_WIDTH * (ZS_BEAM_MAX_WIDTH + ZS_BEAM_MAX_EOS)];
    __shared__ float bs_[ZS_BEAM_MAX_WIDTH];
    __shared__ double bl_[ZS_BEAM_MAX_WIDTH];
    __shared__ float fin_s[ZS_BEAM_MAX_WIDTH];
    __shared__ int fin_p[ZS_BEAM_MAX_WIDTH], fin_t[ZS_BEAM_MAX_WIDTH];
    const uint32_t g = blockIdx.x, lane = threadIdx.x, W = a.width, K = a.K;
    const size_t at = (size_t)g * W;
    const bool beam = lane < W;
    // all loads at once: what is not needed is dropped afterwards
    const int was = a.done[g], steps = a.steps[g];
    const float score = beam ? a.scores[at + lane] : -INFINITY;
    const double lse = beam ? a.lse[at + lane] : 0.0;
    unsigned long long e[NL];
#pragma unroll
    for (int k = 0; k < NL; k++) {
        const uint32_t i = lane + (uint32_t)k * BM_NT;
        e[k] = i < W * K ? a.list[at * K + i] : ~0ull;
    }
    // the pool as it was (threads below W)
    float ps = beam ? a.fin_score[at + lane] : -INFINITY;
    int pl = beam ? a.fin_length[at + lane] : 0, pp = beam ? a.fin_parent[at + lane] : -1, pt = beam ? a.fin_token[at + lane] : -1;
    if (!(ps == ps)) ps = -INFINITY;
    if (beam) {
        // (beams that do not live left no list)
        bs_[lane] = !was && fabsf(score) <= __FLT_MAX__ ? score : -INFINITY;
        bl_[lane] = lse;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NL; k++) {
        const uint32_t i = lane + (uint32_t)k * BM_NT;
        if (i >= W * K) break;
        const uint32_t b = i / K;
        const float bs = bs_[b];
        const bool some = bs > -INFINITY && e[k] != ~0ull;
        cs_[i] = some ? (float)((double)bs + ((double)zs_u2f((uint32_t)(e[k] >> 32)) - bl_[b])) : -INFINITY;
        ci_[i] = (uint32_t)e[k] | (bm_is_eos(a, (uint32_t)e[k]) ? 0x80000000u : 0u);
    }
    __syncthreads();
    if (lane >= 64u) return;
    // the beam's next candidate and the one behind it
    float s = -INFINITY, s2 = -INFINITY;
    uint32_t id = 0, id2 = 0, next = 0;
    auto ahead = [&]() {
        const bool some = beam && next < K;
        s2 = some ? cs_[lane * K + next] : -INFINITY;
        id2 = some ? ci_[lane * K + next] : 0u;
        next++;
    };
    ahead();
    s = s2;
    id = id2;
    ahead();
    int o_parent = -1, o_token = -1;
    float o_score = -INFINITY;
    uint32_t n_live = 0, n_fin = 0;
    for (uint32_t rank = 0; n_live < W; rank++) {
        const float cs = wave_max_f(s);
        if (!(cs > -INFINITY)) break;
        const uint32_t b = (uint32_t)__ffsll((long long)__ballot(s == cs)) - 1u;   // the lowest beam of equals
        const uint32_t cid = zs_readlane_u(id, b);
        if (cid >> 31) {   // EOS
            if (rank < W) {
                if (lane == 0) { fin_s[n_fin] = cs; fin_p[n_fin] = (int)b; fin_t[n_fin] = (int)(cid & 0x7fffffffu); }
                n_fin++;
            }
        } else {
            if (lane == n_live) { o_parent = (int)b; o_token = (int)cid; o_score = cs; }
            n_live++;
        }
        if (lane == b) {
            s = s2;
            id = id2;
            ahead();
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");   // (one wave from here on)
    // the pool and what finished, the pool first among equals: lane i's place
    // is the number of lanes in front of it
    const float len = (float)(steps + 1), norm = a.length_penalty == 1.0f ? len : a.length_penalty == 0.0f ? 1.0f : powf(len, a.length_penalty);
    if (lane >= W && lane < W + n_fin && lane < 64u) {
        const uint32_t i = lane - W;
        ps = fin_s[i] / norm;
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
    const bool done = n_live == 0 || (full && (a.early || worst >= best / norm));
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

int bm_merge_launch(const bm_args& a, uint32_t groups, hipStream_t stream) {
    hipLaunchKernelGGL(zs_k_beam_merge, dim3(groups), dim3(BM_NT), 0, stream, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

// ---------------------------------------------------------------------------
// Reordering in place. A thread owns one column (16, 4, 2 or 1 bytes at the same
// place of every row) of one group: it loads the parents' values of the rows
// that change, then stores them. No other thread touches the column, so the
// array needs no second copy.
// ---------------------------------------------------------------------------
#define RO_NT 256
// n / d for n < 2^31, from ro_div's multiplier
__device__ __forceinline__ uint32_t ro_quot(uint32_t n, uint32_t mul, uint32_t sh) { return sh >= 32u ? __umulhi(n, mul) >> (sh - 32u) : n; }

template <class T, int W>
__device__ __forceinline__ void ro_column(const bm_state& s, uint64_t col, uint64_t row0, const int (&parent)[W]) {
    uint64_t blk, o;
    if (s.total < 1ull << 31) {
        blk = ro_quot((uint32_t)col, s.mul_cols, s.sh_cols);
        o = ro_quot((uint32_t)blk, s.mul_inner, s.sh_inner);
    } else {
        blk = col / s.cols;
        o = blk / s.n_inner;
    }
    char* base = s.base + o * s.outer_stride + (blk - o * s.n_inner) * s.inner_stride + (col - blk * s.cols) * sizeof(T) +
                 row0 * s.row_stride;
    T v[W];
#pragma unroll
    for (int w = 0; w < W; w++)
        if (parent[w] != w) v[w] = *reinterpret_cast<const T*>(base + (uint32_t)parent[w] * s.row_stride);
#pragma unroll
    for (int w = 0; w < W; w++)
        if (parent[w] != w) *reinterpret_cast<T*>(base + (uint32_t)w * s.row_stride) = v[w];
}

template <int W>
__global__ __launch_bounds__(RO_NT) void zs_k_beam_reorder(ro_args a_) {
    // the arrays are indexed where the launch left them: a local copy would
    // be put into scratch or LDS (16.5 KB a workgroup)
#if defined(__HIP_DEVICE_COMPILE__)
    const auto* a = (const __attribute__((address_space(4))) ro_args*)__builtin_amdgcn_kernarg_segment_ptr();
#else
    const ro_args* a = &a_;
#endif
    typedef uint32_t ro_u4 __attribute__((ext_vector_type(4)));
    const uint32_t g = blockIdx.y, width = a->width;
    int parent[W];   // (the same for the whole workgroup: scalar registers)
#pragma unroll
    for (int w = 0; w < W; w++) {
        const int q = (uint32_t)w < width ? a->parent[(size_t)g * width + (uint32_t)w] : w;
        parent[w] = q >= 0 && q < (int)width ? q : w;
    }
    uint32_t i = 0;
    while (i + 1 < a->n && blockIdx.x >= a->s[i + 1].first) i++;
    bm_state s;
    s.base = a->s[i].base;
    s.row_stride = a->s[i].row_stride;
    s.outer_stride = a->s[i].outer_stride;
    s.inner_stride = a->s[i].inner_stride;
    s.cols = a->s[i].cols;
    s.total = a->s[i].total;
    s.n_inner = a->s[i].n_inner;
    s.mul_cols = a->s[i].mul_cols;
    s.sh_cols = a->s[i].sh_cols;
    s.mul_inner = a->s[i].mul_inner;
    s.sh_inner = a->s[i].sh_inner;
    const uint32_t first = a->s[i].first, blocks = a->s[i].blocks, unit = a->s[i].unit;
    const uint64_t row0 = (uint64_t)g * width;
    for (uint64_t col = (uint64_t)(blockIdx.x - first) * RO_NT + threadIdx.x; col < s.total; col += (uint64_t)blocks * RO_NT) {
        if (unit == 16) ro_column<ro_u4, W>(s, col, row0, parent);
        else if (unit == 4) ro_column<uint32_t, W>(s, col, row0, parent);
        else if (unit == 2) ro_column<uint16_t, W>(s, col, row0, parent);
        else ro_column<uint8_t, W>(s, col, row0, parent);
    }
}

int ro_launch(const ro_args& a, uint32_t blocks, uint32_t groups, hipStream_t stream) {
    for (uint32_t g0 = 0; g0 < groups; g0 += 65535u) {
        ro_args b = a;
        const uint32_t n = groups - g0 < 65535u ? groups - g0 : 65535u;
        b.parent += (size_t)g0 * a.width;
        for (uint32_t i = 0; i < b.n; i++) b.s[i].base += (uint64_t)g0 * a.width * b.s[i].row_stride;
        const dim3 grid(blocks, n);
        if (a.width <= 4) hipLaunchKernelGGL(zs_k_beam_reorder<4>, grid, dim3(RO_NT), 0, stream, b);
        else if (a.width <= 8) hipLaunchKernelGGL(zs_k_beam_reorder<8>, grid, dim3(RO_NT), 0, stream, b);
        else if (a.width <= 16) hipLaunchKernelGGL(zs_k_beam_reorder<16>, grid, dim3(RO_NT), 0, stream, b);
        else hipLaunchKernelGGL(zs_k_beam_reorder<32>, grid, dim3(RO_NT), 0, stream, b);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
