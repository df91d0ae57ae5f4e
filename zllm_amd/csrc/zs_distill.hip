// zs_distill.hip -- a student's loss against a teacher's list and its gradient.
//
// With z = x / T, m the row's maximum, e_j = exp(z_j - m / T), S = sum e,
// S_out the sum over the ids outside the list, p the teacher's probabilities,
// P = sum p + p_t, and the first distribution at T = 1 (e1, S1) for the label:
//   KL  = sum_k p_k (ln p_k - (z_k - m / T - ln S)) + p_t (ln p_t - ln S_out + ln S)
//   CE  = ln S1 - (x_label - m)
//   dKL / dx_j = (P e_j / S - p_j - [j outside the list] p_t e_j / S_out) / T
//   dCE / dx_j = e1_j / S1 - [j = label]
// S_out is summed over its own ids: S minus the list's share would lose all of
// its digits where the student has learnt the list.
#include "zs_head.h"
#include "zs_distill.h"

#define DS_NT 256
#define DS_K ZS_DISTILL_KMAX

// A row that takes no part: its label is ignore_index.
__device__ __forceinline__ bool ds_skip(const ds_args& a, uint64_t r) { return a.labels && zs_gload(a.labels + r) == a.ignore; }

// The values of a chunk's vectors (-inf where there is none), U a thread.
template <int DT, int U>
__device__ __forceinline__ void ds_load(const hd_row<DT>& row, uint32_t first, float (&x)[U][hd_elem<DT>::E]) {
    constexpr int E = hd_elem<DT>::E;
    const uint32_t j0 = first + threadIdx.x;
    if (row.inside(first) && row.inside(first + U * DS_NT - 1u)) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; u++) v[u] = row.load(j0 + (uint32_t)u * DS_NT);
#pragma unroll
        for (int u = 0; u < U; u++) hd_unpack<DT>(v[u], x[u]);
    } else {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t j = j0 + (uint32_t)u * DS_NT;
            if (j < row.nvec) row.get(j, x[u], -INFINITY);
            else
#pragma unroll
                for (int q = 0; q < E; q++) x[u][q] = -INFINITY;
        }
    }
}

// ---------------------------------------------------------------------------
// the pass of the loss: per wave the maximum and the sums
// ---------------------------------------------------------------------------
template <int DT, bool TAIL, bool TWO>
__global__ __launch_bounds__(DS_NT) void zs_k_distill_scan(ds_args a, uint64_t r0) {
    constexpr int E = hd_elem<DT>::E, U = HD_WAVE / 64 / E;
    __shared__ uint32_t mask[U * DS_NT / 4];   // a byte a vector: its ids in the list
    const uint64_t r = r0 + blockIdx.x / a.chunks;
    const uint32_t chunk = blockIdx.x % a.chunks, t = threadIdx.x;
    const hd_row<DT> row(a.logits, a.ld, r, a.V);
    const uint32_t first = chunk * (U * DS_NT);
    if (first >= row.nvec || ds_skip(a, r)) return;
    float x[U][E];
    uint32_t id = 0xffffffffu;
    float lk = 0.0f;
    if (TAIL && t < a.K) {
        id = zs_gload(a.ids + r * a.K + t);
        lk = zs_gload(a.logp + r * a.K + t);
    }
    ds_load<DT, U>(row, first, x);
    if (TAIL) {
#pragma unroll
        for (int i = 0; i < U / 4; i++) mask[i * DS_NT + t] = 0;
        __syncthreads();
        const uint32_t j = (id + row.shift) / E - first;
        if (id < a.V && lk != -INFINITY && j < U * DS_NT) atomicOr(&mask[j / 4], 1u << (j % 4 * 8 + (id + row.shift) % E));
        __syncthreads();
    }
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int q = 0; q < E; q++) m = fmaxf(m, x[u][q]);
    m = wave_max_f(m);
    const float mr = m > -INFINITY ? m : 0.0f;
    float s, s1 = 0.0f, so = 0.0f;
    // 2^(x c - mc): one fma a value; mc's rounding is a factor of all of them
    auto sums = [&](float c, bool diff, float& s, float& so, bool list) {
        const float mc = mr * c;
        s = so = 0.0f;
#pragma unroll
        for (int u = 0; u < U; u++) {
            float e[E];
#pragma unroll
            for (int q = 0; q < E; q++) e[q] = __builtin_amdgcn_exp2f(diff ? (x[u][q] - mr) * c : fmaf(x[u][q], c, -mc));
            const float v = hd_sum(e);
            s += v;
            if (TAIL && list) {
                const uint32_t in = reinterpret_cast<const uint8_t*>(mask)[u * DS_NT + t];
                if (in) {
#pragma unroll
                    for (int q = 0; q < E; q++) e[q] = in >> q & 1u ? 0.0f : e[q];
                    so += hd_sum(e);
                } else {
                    so += v;
                }
            }
        }
        const auto add = [](float p, float q) { return p + q; };
        const float f = diff ? 1.0f : __builtin_amdgcn_exp2f(-fmaf(mr, c, -mc));
        s = zs_wave_reduce(s, add) * f;
        if (TAIL && list) so = zs_wave_reduce(so, add) * f;
    };
    float none;
    if (fabsf(mr * a.c) < INFINITY) sums(a.c, false, s, so, true);
    else sums(a.c, true, s, so, true);   // (an exponent that no float holds)
    if (TWO) {
        if (fabsf(mr * (float)HD_LOG2E) < INFINITY) sums((float)HD_LOG2E, false, s1, none, false);
        else sums((float)HD_LOG2E, true, s1, none, false);
    }
    if (zs_lane() == 0) a.rec[r * a.recs + chunk * (HD_CHUNK / HD_WAVE) + (uint32_t)zs_wid()] = make_float4(m, s, s1, so);
}

// ---------------------------------------------------------------------------
// a row's end: the list's probabilities, the loss, the gradient's factors
// ---------------------------------------------------------------------------
#define DF_NT 128   // a thread for every entry of the list
template <int DT, int WHAT>
__global__ __launch_bounds__(DF_NT) void zs_k_distill_row(ds_args a, uint64_t r0) {
    __shared__ double shd[DF_NT / 64];
    __shared__ float shf[DF_NT / 64];
    const uint64_t r = r0 + blockIdx.x;
    const uint32_t t = threadIdx.x;
    const int64_t label = a.labels ? a.labels[r] : -1;
    if (a.labels && label == a.ignore) {
        if ((WHAT & DS_LOSS) && t == 0) a.loss[r] = 0.0f;
        if ((WHAT & DS_LOSS) && a.stats && t < 4) a.stats[r * 4 + t] = 0.0f;
        return;
    }
    const hd_row<DT> row(a.logits, a.ld, r, a.V);
    const bool bad_label = a.labels && (label < 0 || label >= (int64_t)a.V);
    double p = 0.0;
    bool there = false;
    float xk = 0.0f, xl = NAN;
    if (t < a.K) {
        const uint32_t id = a.ids[r * a.K + t];
        const float lk = a.logp[r * a.K + t];
        there = id < a.V && lk != -INFINITY;
        if (there) {
            p = exp((double)lk);
            if (WHAT & DS_LOSS) xk = row.at(id);
        }
    }
    if ((WHAT & DS_LOSS) && a.labels && !bad_label) xl = row.at((uint32_t)label);
    double m, S, S1, So;
    if (WHAT & DS_LOSS) {
        constexpr int E = hd_elem<DT>::E;
        const uint32_t recs = (row.nvec * E + HD_CHUNK - 1u) / HD_CHUNK * (HD_CHUNK / HD_WAVE);
        const float4* rec = a.rec + r * a.recs;
        float mf = -INFINITY;
        for (uint32_t i = t; i < recs; i += DF_NT) mf = fmaxf(mf, rec[i].x);
        m = block_max_f<DF_NT>(mf, shf);
        S = S1 = So = 0.0;
        for (uint32_t i = t; i < recs; i += DF_NT) {
            const float4 v = rec[i];
            const double d = v.x == (float)m ? 0.0 : (double)v.x - m, f = exp(d * a.inv_t);
            S += (double)v.y * f;
            if (a.two) S1 += (double)v.z * exp(d);
            So += (double)v.w * f;
        }
        S = block_sum_d<DF_NT>(S, shd);
        if (!(m > -INFINITY)) S = NAN;   // a row of nothing has no distribution
        S1 = a.two ? block_sum_d<DF_NT>(S1, shd) : S;
        So = a.tail ? block_sum_d<DF_NT>(So, shd) : 0.0;
    } else {
        const float4 st = *reinterpret_cast<const float4*>(a.stats + r * 4);
        m = st.x;
        S = st.y;
        S1 = st.z;
        So = st.w;
    }
    const double psum = block_sum_d<DF_NT>(p, shd);
    const double pt = a.tail ? fmax(1.0 - psum, 0.0) : 0.0;
    if (!a.tail && psum > 0.0) p /= psum;
    const double P = a.tail ? psum + pt : (psum > 0.0 ? 1.0 : psum);
    if (WHAT & DS_LOSS) {
        double term = 0.0;
        if (there && p != 0.0) term = p * (log(p) - (((double)xk - m) * a.inv_t - log(S)));   // (NaN stays)
        term = block_sum_d<DF_NT>(term, shd);
        if (t == 0) {
            if (pt > 0.0) term += pt * (log(pt) - (log(So) - log(S)));
            double loss = (double)a.kl * term;
            if (a.labels) loss += (double)a.ce * (log(S1) - ((double)xl - m));
            a.loss[r] = (float)loss;
            if (a.stats) *reinterpret_cast<float4*>(a.stats + r * 4) = make_float4((float)m, (float)S, (float)S1, (float)So);
        }
    }
    if (WHAT & DS_GRAD) {
        if (t < a.K) a.p[r * a.K + t] = (float)p;
        if (t == 0) {
            const double g = bad_label ? (double)NAN : (double)a.row_grad[r * a.row_grad_stride];
            const double kl = g * a.kl * a.inv_t, ce = a.labels ? g * a.ce : 0.0;
            const float mf = (float)m, c1 = (float)HD_LOG2E;
            // e = 2^(x c - mc) has mc's rounding for a factor (none where mc is no number: differences are taken)
            const float mc = mf * a.c, m1 = mf * c1;
            const double f = fabsf(mc) < INFINITY ? exp2(-(double)fmaf(mf, a.c, -mc)) : 1.0;
            const double f1 = fabsf(m1) < INFINITY ? exp2(-(double)fmaf(mf, c1, -m1)) : 1.0;
            const double one = a.labels ? ce / S1 : 0.0;
            const double in = kl * P / S + (a.two ? 0.0 : one);
            ds_coef k;
            k.m = mf;
            k.mc = mc;
            k.m1 = m1;
            k.fi = (float)(in * f);
            k.fo = (float)((in - (a.tail && So > 0.0 ? kl * pt / So : 0.0)) * f);
            k.f1 = (float)(one * f1);
            k.fp = (float)kl;
            k.fc = (float)ce;
            a.coef[r] = k;
        }
    }
}

// ---------------------------------------------------------------------------
// the pass of the gradient
// ---------------------------------------------------------------------------
template <int DT>
__device__ __forceinline__ void ds_store1(void* p, float y) {
    if constexpr (DT == ZS_F32) *(float*)p = y;
    else *(uint16_t*)p = (uint16_t)hd_pack2<DT>(y, 0.0f);
}
template <int DT, bool TWO>
__global__ __launch_bounds__(DS_NT) void zs_k_distill_grad(ds_args a, uint64_t r0) {
    constexpr int E = hd_elem<DT>::E, U = HD_WAVE / 64 / E;
    typedef typename hd_elem<DT>::T T;
    __shared__ uint32_t mask[U * DS_NT / 4];   // a byte a vector: its ids in the list, or the label
    __shared__ uint32_t hid[DS_K], cnt[DS_K / 64];
    __shared__ float hp[DS_K];
    const uint64_t r = r0 + blockIdx.x / a.chunks;
    const uint32_t chunk = blockIdx.x % a.chunks, t = threadIdx.x;
    const hd_row<DT> row(a.logits, a.ld, r, a.V);
    const uint32_t first = chunk * (U * DS_NT);
    if (first >= row.nvec) return;
    T* grad = reinterpret_cast<T*>(a.grad) + r * a.ld_grad;
    const bool aligned = (((uintptr_t)grad ^ (uintptr_t)row.row) & 15u) == 0;
    const bool skip = ds_skip(a, r);
    const int64_t label = a.labels ? zs_gload(a.labels + r) : -1;
    float x[U][E];
    if (!skip) {
        uint32_t id = 0xffffffffu;
        float p = 0.0f;
        if (t < a.K) {
            id = zs_gload(a.ids + r * a.K + t);
            p = zs_gload(a.p + r * a.K + t);
            if (id < a.V && p == 0.0f && zs_gload(a.logp + r * a.K + t) == -INFINITY) id = 0xffffffffu;   // absent
        }
        const ds_coef k = a.coef[r];
        ds_load<DT, U>(row, first, x);
#pragma unroll
        for (int i = 0; i < U / 4; i++) mask[i * DS_NT + t] = 0;
        // the chunk's entries, in the list's order
        const uint32_t pos = id + row.shift, j = pos / E - first;
        const bool hit = id < a.V && j < U * DS_NT;
        const unsigned long long hm = __ballot(hit);
        if (t < DS_K && zs_lane() == 0) cnt[zs_wid()] = (uint32_t)__popcll(hm);
        __syncthreads();
        if (hit) {
            uint32_t at = zs_wid() ? cnt[0] : 0u;
            at = __builtin_amdgcn_mbcnt_hi((uint32_t)(hm >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hm, at));
            hid[at] = id;
            hp[at] = k.fp * p;
            atomicOr(&mask[j / 4], 1u << (j % 4 * 8 + pos % E));
        }
        if (t == DS_K && label >= 0 && label < (int64_t)a.V) {
            const uint32_t lp = (uint32_t)label + row.shift, lj = lp / E - first;
            if (lj < U * DS_NT) atomicOr(&mask[lj / 4], 1u << (lj % 4 * 8 + lp % E));
        }
        __syncthreads();
        const uint32_t hits = cnt[0] + cnt[1];
        const bool diff = !(fabsf(k.mc) < INFINITY), diff1 = !(fabsf(k.m1) < INFINITY);
#pragma unroll
        for (int u = 0; u < U; u++) {
            float e[E], e1[E];
#pragma unroll
            for (int q = 0; q < E; q++) {
                e[q] = __builtin_amdgcn_exp2f(diff ? (x[u][q] - k.m) * a.c : fmaf(x[u][q], a.c, -k.mc));
                const float c1 = (float)HD_LOG2E;
                e1[q] = TWO ? __builtin_amdgcn_exp2f(diff1 ? (x[u][q] - k.m) * c1 : fmaf(x[u][q], c1, -k.m1)) * k.f1 : 0.0f;
            }
            if (reinterpret_cast<const uint8_t*>(mask)[u * DS_NT + t]) {
                const int i0 = row.id0(first + t + (uint32_t)u * DS_NT);
                uint32_t in = 0;
                float sub[E];
#pragma unroll
                for (int q = 0; q < E; q++) sub[q] = (int64_t)(i0 + q) == label ? k.fc : 0.0f;
                for (uint32_t h = 0; h < hits; h++) {
                    const int at = (int)hid[h] - i0;
                    if (at < 0 || at >= E) continue;
                    in |= 1u << at;
#pragma unroll
                    for (int q = 0; q < E; q++) sub[q] += q == at ? hp[h] : 0.0f;
                }
#pragma unroll
                for (int q = 0; q < E; q++) x[u][q] = e[q] * (in >> q & 1u ? k.fi : k.fo) + (e1[q] - sub[q]);
            } else {
#pragma unroll
                for (int q = 0; q < E; q++) x[u][q] = TWO ? e[q] * k.fo + e1[q] : e[q] * k.fo;
            }
        }
    } else {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int q = 0; q < E; q++) x[u][q] = 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t j = first + t + (uint32_t)u * DS_NT;
        const int i0 = row.id0(j);
        if (aligned && row.inside(j)) {
            uint4 v;
            if constexpr (DT == ZS_F32) v = make_uint4(__float_as_uint(x[u][0]), __float_as_uint(x[u][1]), __float_as_uint(x[u][2]), __float_as_uint(x[u][3]));
            else v = make_uint4(hd_pack2<DT>(x[u][0], x[u][1]), hd_pack2<DT>(x[u][2], x[u][3]), hd_pack2<DT>(x[u][E / 2], x[u][E / 2 + 1]), hd_pack2<DT>(x[u][E - 2], x[u][E - 1]));
            *reinterpret_cast<uint4*>(grad + i0) = v;
        } else {
#pragma unroll
            for (int q = 0; q < E; q++)
                if (i0 + q >= 0 && (uint32_t)(i0 + q) < a.V) ds_store1<DT>(grad + i0 + q, x[u][q]);
        }
    }
}

template <int DT>
static void ds_go(const ds_args& a, int what, uint64_t r0, uint32_t n, hipStream_t stream) {
    const dim3 grid(n * a.chunks), wg(DS_NT);
    if (what & DS_LOSS) {
        if (a.tail && a.two) hipLaunchKernelGGL((zs_k_distill_scan<DT, true, true>), grid, wg, 0, stream, a, r0);
        else if (a.tail) hipLaunchKernelGGL((zs_k_distill_scan<DT, true, false>), grid, wg, 0, stream, a, r0);
        else if (a.two) hipLaunchKernelGGL((zs_k_distill_scan<DT, false, true>), grid, wg, 0, stream, a, r0);
        else hipLaunchKernelGGL((zs_k_distill_scan<DT, false, false>), grid, wg, 0, stream, a, r0);
    }
    if (what == DS_LOSS) hipLaunchKernelGGL((zs_k_distill_row<DT, DS_LOSS>), dim3(n), dim3(DF_NT), 0, stream, a, r0);
    else if (what == DS_GRAD) hipLaunchKernelGGL((zs_k_distill_row<DT, DS_GRAD>), dim3(n), dim3(DF_NT), 0, stream, a, r0);
    else hipLaunchKernelGGL((zs_k_distill_row<DT, DS_LOSS | DS_GRAD>), dim3(n), dim3(DF_NT), 0, stream, a, r0);
    if (what & DS_GRAD) {
        if (a.two) hipLaunchKernelGGL((zs_k_distill_grad<DT, true>), grid, wg, 0, stream, a, r0);
        else hipLaunchKernelGGL((zs_k_distill_grad<DT, false>), grid, wg, 0, stream, a, r0);
    }
}
int ds_launch(const ds_args& a, uint32_t dtype, int what, hipStream_t stream) {
    const uint64_t per = HD_BLOCKS / a.chunks;
    for (uint64_t r0 = 0; r0 < a.N; r0 += per) {
        const uint32_t n = (uint32_t)(a.N - r0 < per ? a.N - r0 : per);
        if (dtype == ZS_F32) ds_go<ZS_F32>(a, what, r0, n, stream);
        else if (dtype == ZS_F16) ds_go<ZS_F16>(a, what, r0, n, stream);
        else ds_go<ZS_BF16>(a, what, r0, n, stream);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
