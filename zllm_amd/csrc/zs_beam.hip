// zs_beam.hip -- beam search: the states of the beams follow their parents.
// (The step itself ends in zs_head.hip's pick, with zs_beam_merge.h.)
#include <hip/hip_runtime.h>
#include "zs_beam.h"

// ---------------------------------------------------------------------------
// Reordering in place. A thread owns one column (16, 4, 2 or 1 bytes at the same
// place of every row) of one group: it loads the parents' values of the rows
// that change, then stores them. No other thread touches the column, so the
// array needs no second copy. The loads are issued without conditions, those of
// rows that stay from a parent that is loaded anyway: behind a branch each the
// compiler waits for every one by itself (5 beams, 294 MB: 193 us, so 67; 4
// beams, 4058 MB: 660 to 790, so 640 to 740, and in other runs up to 815, by where
// the caches lie; waiting for all before the first store: 675 to 780).
// ---------------------------------------------------------------------------
#define RO_NT 256
#define RO_GLOBAL __attribute__((address_space(1)))
template <class T, int W>
__device__ __forceinline__ void ro_columns(const bm_state& s, uint64_t col, uint64_t step, uint64_t row0, const uint32_t (&src)[W],
                                           uint32_t changed) {
#pragma unroll 1
    for (; col < s.total; col += step) {
        uint64_t blk, o;
        if (s.total < 1ull << 31) {
            blk = zs_quot((uint32_t)col, s.by_cols);
            o = zs_quot((uint32_t)blk, s.by_inner);
        } else {
            blk = col / s.cols;
            o = blk / s.n_inner;
        }
        char* base = s.base + o * s.outer_stride + (blk - o * s.n_inner) * s.inner_stride + (col - blk * s.cols) * sizeof(T) +
                     row0 * s.row_stride;
        T v[W];
#pragma unroll
        for (int w = 0; w < W; w++) v[w] = __builtin_nontemporal_load((const RO_GLOBAL T*)(base + src[w] * s.row_stride));
#pragma unroll
        for (int w = 0; w < W; w++)
            if (changed >> w & 1u) __builtin_nontemporal_store(v[w], (RO_GLOBAL T*)(base + (uint32_t)w * s.row_stride));
    }
}

template <int W>
__global__ __launch_bounds__(RO_NT, W <= 8 ? 6 : W <= 16 ? 4 : 2) void zs_k_beam_reorder(ro_args a_) {
    // the arrays are indexed where the launch left them: a local copy would
    // be put into scratch or LDS (16.5 KB a workgroup)
#if defined(__HIP_DEVICE_COMPILE__)
    const auto* a = (const __attribute__((address_space(4))) ro_args*)__builtin_amdgcn_kernarg_segment_ptr();
#else
    const ro_args* a = &a_;
#endif
    typedef uint32_t ro_u4 __attribute__((ext_vector_type(4)));
    const uint32_t g = blockIdx.y, width = a->width;
    // (the same for the whole workgroup: scalar registers)
    uint32_t src[W], changed = 0, some = 0;
#pragma unroll
    for (int w = 0; w < W; w++) {
        const int q = __builtin_amdgcn_readfirstlane((uint32_t)w < width ? a->parent[(size_t)g * width + (uint32_t)w] : w);
        src[w] = q >= 0 && q < (int)width ? (uint32_t)q : (uint32_t)w;
        if (src[w] != (uint32_t)w) {
            changed |= 1u << w;
            some = src[w];
        }
    }
    if (!changed) return;
#pragma unroll
    for (int w = 0; w < W; w++) src[w] = changed >> w & 1u ? src[w] : some;
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
    s.by_cols.mul = a->s[i].by_cols.mul;
    s.by_cols.sh = a->s[i].by_cols.sh;
    s.by_inner.mul = a->s[i].by_inner.mul;
    s.by_inner.sh = a->s[i].by_inner.sh;
    const uint32_t first = a->s[i].first, blocks = a->s[i].blocks, unit = a->s[i].unit;
    const uint64_t row0 = (uint64_t)g * width;
    const uint64_t col = (uint64_t)(blockIdx.x - first) * RO_NT + threadIdx.x, step = (uint64_t)blocks * RO_NT;
    if (unit == 16) ro_columns<ro_u4, W>(s, col, step, row0, src, changed);
    else if (unit == 4) ro_columns<uint32_t, W>(s, col, step, row0, src, changed);
    else if (unit == 2) ro_columns<uint16_t, W>(s, col, step, row0, src, changed);
    else ro_columns<uint8_t, W>(s, col, step, row0, src, changed);
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
