// zs_beam.hip -- beam search: the step of a group of beams from the heads of
// their rows (zs_head.hip), and the reordering of the beams' states.
#include "zs_head.h"
#include "zs_beam.h"

// ---------------------------------------------------------------------------
// The step of one request by one wave. The rows' heads are sorted, so the
// candidates' order is a merge of at most 32 lists: lane b holds the score of
// beam b's next candidate, each turn takes the largest (the lowest beam of
// equals). A row needs width + n_eos entries: its first `width` that do not
// end are among them, and so is every EOS id among the first `width` overall.
// ---------------------------------------------------------------------------
__device__ __forceinline__ bool bm_is_eos(const bm_args& a, uint32_t id) {
    bool e = false;
#pragma unroll
    for (uint32_t i = 0; i < ZS_BEAM_MAX_EOS; i++) e |= i < a.n_eos && a.eos[i] == id;
    return e;
}

__global__ __launch_bounds__(64) void zs_k_beam_merge(bm_args a) {
    __shared__ float fin_s[ZS_BEAM_MAX_WIDTH];
    __shared__ int fin_p[ZS_BEAM_MAX_WIDTH], fin_t[ZS_BEAM_MAX_WIDTH];
    const uint32_t g = blockIdx.x, lane = (uint32_t)zs_lane(), W = a.width, K = a.K;
    const size_t at = (size_t)g * W;
    const bool was = a.done[g] != 0;
    const int steps = a.steps[g];
    const bool beam = lane < W;
    // the pool as it was (lanes below W)
    float ps = beam ? a.fin_score[at + lane] : -INFINITY;
    int pl = beam ? a.fin_length[at + lane] : 0, pp = beam ? a.fin_parent[at + lane] : -1, pt = beam ? a.fin_token[at + lane] : -1;
    if (!(ps == ps)) ps = -INFINITY;
    const float score = beam ? a.scores[at + lane] : -INFINITY;
    const bool live = !was && fabsf(score) <= __FLT_MAX__;
    const unsigned long long* list = a.list + (at + lane) * K;
    const double lse = live ? a.lse[at + lane] : 0.0;
    uint32_t next = 0, id = 0;
    float s = -INFINITY;
    auto take = [&]() {   // the beam's next candidate
        s = -INFINITY;
        if (!live || next >= K) return;
        const unsigned long long e = list[next++];
        if (e == ~0ull) { next = K; return; }
        id = (uint32_t)e;
        s = (float)((double)score + ((double)zs_u2f((uint32_t)(e >> 32)) - lse));
    };
    take();
    int o_parent = -1, o_token = -1;
    float o_score = -INFINITY;
    uint32_t n_live = 0, n_fin = 0;
    for (uint32_t rank = 0; n_live < W; rank++) {
        // larger score, then lower beam; 0: none is left
        unsigned long long key = s > -INFINITY ? ((unsigned long long)zs_total_key(s + 0.0f) << 32) | (63u - lane) : 0ull;
        key = zs_wave_reduce(key, [](unsigned long long x, unsigned long long y) { return x > y ? x : y; });
        if (!key) break;
        const uint32_t b = 63u - (uint32_t)(key & 63u);
        const uint32_t cid = zs_readlane_u(id, b);
        const float cs = zs_readlane_f(s, b);
        if (bm_is_eos(a, cid)) {
            if (rank < W) {
                if (lane == 0) { fin_s[n_fin] = cs; fin_p[n_fin] = (int)b; fin_t[n_fin] = (int)cid; }
                n_fin++;
            }
        } else {
            if (lane == n_live) { o_parent = (int)b; o_token = (int)cid; o_score = cs; }
            n_live++;
        }
        if (lane == b) take();
    }
    __syncthreads();
    // the pool and what finished, the pool first among equals: lane i's place
    // is the number of lanes in front of it
    const double norm = pow((double)(steps + 1), (double)a.length_penalty);
    if (lane >= W && lane < W + n_fin && lane < 64u) {
        const uint32_t i = lane - W;
        ps = (float)((double)fin_s[i] / norm);
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
    const bool done = n_live == 0 || (full && (a.early || worst >= (float)((double)best / norm)));
    if (stays) {
        const bool some = ps > -INFINITY;
        a.fin_score_o[at + place] = some || was ? ps : -INFINITY;
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
        a.done_o[g] = was ? a.done[g] : (done ? 1 : 0);
    }
}

int bm_merge_launch(const bm_args& a, uint32_t groups, hipStream_t stream) {
    hipLaunchKernelGGL(zs_k_beam_merge, dim3(groups), dim3(64), 0, stream, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

// ---------------------------------------------------------------------------
// Reordering in place. A thread owns one column (16, 4, 2 or 1 bytes at the same
// place of every row) of one group: it loads the parents' values of the rows
// that change, then stores them. No other thread touches the column, so the
// array needs no second copy.
// ---------------------------------------------------------------------------
#define RO_NT 256
template <class T, int W>
__device__ __forceinline__ void ro_column(const bm_state& s, uint64_t col, uint64_t row0, uint32_t width, const int* parent) {
    const uint64_t per = s.cols, blk = col / per, o = blk / s.n_inner, i = blk % s.n_inner;
    char* base = s.base + o * s.outer_stride + i * s.inner_stride + (col % per) * sizeof(T);
    T v[W];
#pragma unroll
    for (int w = 0; w < W; w++)
        if ((uint32_t)w < width && parent[w] != w) v[w] = *reinterpret_cast<const T*>(base + (row0 + (uint32_t)parent[w]) * s.row_stride);
#pragma unroll
    for (int w = 0; w < W; w++)
        if ((uint32_t)w < width && parent[w] != w) *reinterpret_cast<T*>(base + (row0 + (uint32_t)w) * s.row_stride) = v[w];
}

template <int W>
__global__ __launch_bounds__(RO_NT) void zs_k_beam_reorder(ro_args a) {
    __shared__ int parent[W];
    const uint32_t g = blockIdx.y;
    if (threadIdx.x < (uint32_t)W) {
        int p = (int)threadIdx.x;
        if (threadIdx.x < a.width) {
            const int q = a.parent[(size_t)g * a.width + threadIdx.x];
            if (q >= 0 && q < (int)a.width) p = q;
        }
        parent[threadIdx.x] = p;
    }
    __syncthreads();
    uint32_t i = 0;
    while (i + 1 < a.n && blockIdx.x >= a.s[i + 1].first) i++;
    const bm_state& s = a.s[i];
    const uint64_t row0 = (uint64_t)g * a.width;
    for (uint64_t col = (uint64_t)(blockIdx.x - s.first) * RO_NT + threadIdx.x; col < s.total; col += (uint64_t)s.blocks * RO_NT) {
        if (s.unit == 16) ro_column<uint4, W>(s, col, row0, a.width, parent);
        else if (s.unit == 4) ro_column<uint32_t, W>(s, col, row0, a.width, parent);
        else if (s.unit == 2) ro_column<uint16_t, W>(s, col, row0, a.width, parent);
        else ro_column<uint8_t, W>(s, col, row0, a.width, parent);
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
