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

#define DS_NT 512
#define DS_K ZS_DISTILL_KMAX

// One workgroup a row.
template <int DT, int WHAT>
__global__ __launch_bounds__(DS_NT) void zs_k_distill_row(ds_args a, uint64_t r0) {
    constexpr int E = hd_elem<DT>::E, NW = DS_NT / 64;
    typedef typename hd_elem<DT>::T T;
    __shared__ uint32_t lid[DS_K];
    __shared__ float lp[DS_K];
    __shared__ uint32_t bits[(ZS_HEAD_MAX_VOCAB / 4 + 1) / 32 + 1];   // vectors that hold an id of the list
    __shared__ float shf[NW];
    __shared__ double shd[NW];
    const uint64_t r = r0 + blockIdx.x;
    const uint32_t t = threadIdx.x;
    const hd_row<DT> row(a.logits, a.ld, r, a.V);
    T* grad = (WHAT & DS_GRAD) ? reinterpret_cast<T*>(a.grad) + r * a.ld_grad : nullptr;
    const int64_t label = a.labels ? a.labels[r] : -1;
    if (a.labels && label == a.ignore) {
        if ((WHAT & DS_LOSS) && t == 0) a.loss[r] = 0.0f;
        if ((WHAT & DS_LOSS) && a.stats && t < 4) a.stats[r * 4 + t] = 0.0f;
        if (WHAT & DS_GRAD)
            for (uint32_t i = t; i < a.V; i += DS_NT) grad[i] = (T)0;
        return;
    }
    const bool bad_label = a.labels && (label < 0 || label >= (int64_t)a.V);
    // the list: probabilities, the tail's, the vectors that it touches
    for (uint32_t i = t; i < (row.nvec + 31) / 32; i += DS_NT) bits[i] = 0;
    double p = 0.0;
    bool there = false;
    uint32_t id = 0xffffffffu;
    float lk = -INFINITY;
    if (t < a.K) {
        id = a.ids[r * a.K + t];
        lk = a.logp[r * a.K + t];
        there = id < a.V && lk != -INFINITY;
        p = there ? exp((double)lk) : 0.0;
        if (!there) id = 0xffffffffu;
    }
    const double psum = block_sum_d<DS_NT>(p, shd);
    const double pt = a.tail ? fmax(1.0 - psum, 0.0) : 0.0;
    if (!a.tail && psum > 0.0) p /= psum;
    const double P = a.tail ? psum + pt : (psum > 0.0 ? 1.0 : psum);
    if (t < a.K) {
        lid[t] = id;
        lp[t] = (float)p;
        if (there) atomicOr(&bits[(id + row.shift) / E / 32], 1u << ((id + row.shift) / E % 32));
    }
    if (t == 0 && a.labels && !bad_label) atomicOr(&bits[((uint32_t)label + row.shift) / E / 32], 1u << (((uint32_t)label + row.shift) / E % 32));
    __syncthreads();
    auto listed = [&](uint32_t j) { return (bits[j / 32] >> (j % 32)) & 1u; };
    float m, xk = 0.0f, xl = 0.0f;
    double S, S1, So;
    if (WHAT & DS_LOSS) {
        m = -INFINITY;
        float x[E];
        for (uint32_t j = t; j < row.nvec; j += DS_NT) {
            row.get(j, x, -INFINITY);
#pragma unroll
            for (int q = 0; q < E; q++) m = fmaxf(m, x[q]);
        }
        m = block_max_f<DS_NT>(m, shf);
        float s = 0.0f, s1 = 0.0f, so = 0.0f;
        for (uint32_t j = t; j < row.nvec; j += DS_NT) {
            row.get(j, x, -INFINITY);
            uint32_t in = 0;
            if (a.tail && listed(j))
                for (uint32_t k = 0; k < a.K; k++)
                    if (lid[k] != 0xffffffffu && (lid[k] + row.shift) / E == j) in |= 1u << ((lid[k] + row.shift) % E);
            const int i0 = row.id0(j);
            float e[E], e1[E], eo[E];
#pragma unroll
            for (int q = 0; q < E; q++) {
                const bool no_id = i0 + q < 0 || (uint32_t)(i0 + q) >= a.V;   // (where m is -inf too)
                const float d = x[q] - m;
                e[q] = no_id ? 0.0f : __builtin_amdgcn_exp2f(d * a.c);
                e1[q] = no_id || !a.two ? 0.0f : __builtin_amdgcn_exp2f(d * (float)HD_LOG2E);
                eo[q] = in >> q & 1u ? 0.0f : e[q];
            }
            s += hd_sum(e);
            s1 += hd_sum(e1);
            so += hd_sum(eo);
        }
        S = block_sum_d<DS_NT>((double)s, shd);
        S1 = a.two ? block_sum_d<DS_NT>((double)s1, shd) : S;
        So = a.tail ? block_sum_d<DS_NT>((double)so, shd) : 0.0;
        if (there) xk = row.at(id);
        double term = there && p > 0.0 ? p * (log(p) - (((double)xk - (double)m) * a.inv_t - log(S))) : (p != p ? p : 0.0);
        double loss = (double)a.kl * block_sum_d<DS_NT>(term, shd);
        if (t == 0) {
            if (pt > 0.0 || pt != pt) loss += (double)a.kl * pt * (log(pt) - (log(So) - log(S)));
            if (a.labels) {
                xl = bad_label ? NAN : row.at((uint32_t)label);
                loss += (double)a.ce * (log(S1) - ((double)xl - (double)m));
            }
            a.loss[r] = (float)loss;
            if (a.stats) {
                float* st = a.stats + r * 4;
                st[0] = m;
                st[1] = (float)S;
                st[2] = (float)S1;
                st[3] = (float)So;
            }
        }
        __syncthreads();   // the list's logits are read before the row is written
    } else {
        const float* st = a.stats + r * 4;
        m = st[0];
        S = st[1];
        S1 = st[2];
        So = st[3];
    }
    if (!(WHAT & DS_GRAD)) return;
    const double g = (double)a.row_grad[r * a.row_grad_stride] * (bad_label ? (double)NAN : 1.0);
    const double kl = g * a.kl * a.inv_t, ce = a.labels ? g * a.ce : 0.0;
    // e's factor inside and outside the list, e1's, and of p and the label
    const double f_in = kl * P / S, f_out = f_in - (a.tail && So > 0.0 ? kl * pt / So : 0.0), f1 = a.labels ? ce / S1 : 0.0;
    const float fi = (float)(f_in + (a.two ? 0.0 : f1)), fo = (float)(f_out + (a.two ? 0.0 : f1)), fl = (float)f1;
    const float fp = (float)kl, fc = (float)ce;
    for (uint32_t j = t; j < row.nvec; j += DS_NT) {
        float x[E], y[E];
        row.get(j, x, -INFINITY);
        uint32_t in = 0;
        float sub[E];
#pragma unroll
        for (int q = 0; q < E; q++) sub[q] = 0.0f;
        const int i0 = row.id0(j);
        if (listed(j)) {
            for (uint32_t k = 0; k < a.K; k++) {
                const int q = (int)lid[k] - i0;
                if (lid[k] == 0xffffffffu || q < 0 || q >= E) continue;
                in |= 1u << q;
#pragma unroll
                for (int w = 0; w < E; w++) sub[w] += w == q ? fp * lp[k] : 0.0f;
            }
            if (a.labels) {
#pragma unroll
                for (int w = 0; w < E; w++) sub[w] += (int64_t)(i0 + w) == label ? fc : 0.0f;
            }
        }
#pragma unroll
        for (int q = 0; q < E; q++) {
            const float d = x[q] - m;
            y[q] = __builtin_amdgcn_exp2f(d * a.c) * ((in >> q & 1u) || !a.tail ? fi : fo) - sub[q];
            if (a.two) y[q] += __builtin_amdgcn_exp2f(d * (float)HD_LOG2E) * fl;
        }
#pragma unroll
        for (int q = 0; q < E; q++) {
            const int i = i0 + q;
            if (i < 0 || (uint32_t)i >= a.V) continue;
            if constexpr (DT == ZS_F32) grad[i] = y[q];
            else if constexpr (DT == ZS_F16) grad[i] = (_Float16)y[q];
            else grad[i] = (uint16_t)hd_pack2<DT>(y[q], 0.0f);
        }
    }
}

int ds_launch(const ds_args& a, uint32_t dtype, int what, hipStream_t stream) {
    for (uint64_t r0 = 0; r0 < a.N; r0 += HD_BLOCKS) {
        const dim3 grid((uint32_t)(a.N - r0 < HD_BLOCKS ? a.N - r0 : HD_BLOCKS));
#define DS_GO(DT)                                                                                                      \
    if (what == DS_LOSS) hipLaunchKernelGGL((zs_k_distill_row<DT, DS_LOSS>), grid, dim3(DS_NT), 0, stream, a, r0);     \
    else if (what == DS_GRAD) hipLaunchKernelGGL((zs_k_distill_row<DT, DS_GRAD>), grid, dim3(DS_NT), 0, stream, a, r0); \
    else hipLaunchKernelGGL((zs_k_distill_row<DT, DS_LOSS | DS_GRAD>), grid, dim3(DS_NT), 0, stream, a, r0)
        if (dtype == ZS_F32) { DS_GO(ZS_F32); }
        else if (dtype == ZS_F16) { DS_GO(ZS_F16); }
        else { DS_GO(ZS_BF16); }
#undef DS_GO
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
