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
// its digits where the student has learnt the list. Where it is less than 2^-64
// of the row's largest term, its terms leave the floats (e below 2^-126 is 0, and
// p_t / S_out times it 0 times infinity): such a row is read once more for the
// sum relative to the outside ids' own maximum (ds_outside), and those ids'
// gradient is formed with that maximum too.
#include "zs_head.h"
#include "zs_distill.h"

#define DS_NT 256
#define DS_K ZS_DISTILL_KMAX
#define DS_FUSED_VOCAB 4096    // (rows have whole vectors, and a batch of them)
#define DS_FUSED_SHORT 32768   // rows up to here by one workgroup each, were there one row,
#define DS_FUSED_ROWS 96       // longer ones from this many on
#define DS_FUSED_LDS (160 * 1024 - 6400)   // what the kernel's own shared memory leaves

// A row that takes no part: its label is ignore_index.
__device__ __forceinline__ bool ds_skip(const ds_args& a, uint64_t r) { return a.labels && zs_gload(a.labels + r) == a.ignore; }

// The values of a chunk's vectors (-inf where there is none), U a thread.
template <int DT, int U>
__device__ __forceinline__ void ds_load(const hd_row<DT>& row, uint32_t first, float (&x)[U][hd_elem<DT>::E]) {
    constexpr int E = hd_elem<DT>::E;
    hd_u4 v[U];
    row.take(first + threadIdx.x, DS_NT, row.inside(first) && row.inside(first + U * DS_NT - 1u), v);
#pragma unroll
    for (int u = 0; u < U; u++) hd_unpack<DT>(v[u], x[u]);
}

// ---------------------------------------------------------------------------
// the pass of the loss: per wave the maximum and the sums
// ---------------------------------------------------------------------------
template <int DT, bool TAIL, bool TWO>
__global__ __launch_bounds__(DS_NT) void zs_k_distill_scan(ds_args a, uint64_t r0) {
    constexpr int E = hd_elem<DT>::E, U = DS_WAVE / 64 / E;
    __shared__ uint32_t mask[U * DS_NT / 4];   // a byte a vector: its ids in the list
    const uint32_t n = zs_quot(blockIdx.x, a.by_chunks), chunk = blockIdx.x - n * a.chunks, t = threadIdx.x;
    const uint64_t r = r0 + n;
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
    auto sums = [&](float c0, float& s, float& so, bool list) {
        const float c = hd_factor(mr, c0), mc = mr * c;
        s = so = 0.0f;
#pragma unroll
        for (int u = 0; u < U; u++) {
            float e[E];
#pragma unroll
            for (int q = 0; q < E; q++) e[q] = __builtin_amdgcn_exp2f(fmaf(x[u][q], c, -mc));
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
        const float f = __builtin_amdgcn_exp2f(-fmaf(mr, c, -mc));
        s = zs_wave_reduce(s, add) * f;
        if (TAIL && list) so = zs_wave_reduce(so, add) * f;
    };
    float none;
    sums(a.c, s, so, true);
    if (TWO) sums((float)HD_LOG2E, s1, none, false);
    if (zs_lane() == 0) a.rec[r * a.recs + chunk * (HD_CHUNK / DS_WAVE) + (uint32_t)zs_wid()] = make_float4(m, s, s1, so);
}

// ---------------------------------------------------------------------------
// a row's end: the list's probabilities, the loss, the gradient's factors
// ---------------------------------------------------------------------------
// The list of a row, an entry a thread (t < K), and its probabilities.
struct ds_entry {
    uint32_t id;
    bool there;
    double p;       // normalised without the tail
    double pt, P;   // the tail's, and of all outcomes (the same on every thread)
};
template <int NT>
__device__ __forceinline__ ds_entry ds_list(const ds_args& a, uint64_t r, double* shd) {
    ds_entry o;
    o.id = 0xffffffffu;
    o.there = false;
    o.p = 0.0;
    if (threadIdx.x < a.K) {
        o.id = a.ids[r * a.K + threadIdx.x];
        const float lk = a.logp[r * a.K + threadIdx.x];
        o.there = o.id < a.V && lk != -INFINITY;
        if (o.there) o.p = exp((double)lk);
    }
    const double psum = block_sum_d<NT>(o.p, shd);
    o.pt = a.tail ? fmax(1.0 - psum, 0.0) : 0.0;
    if (!a.tail && psum > 0.0) o.p /= psum;
    o.P = a.tail ? psum + o.pt : (psum > 0.0 ? 1.0 : psum);
    return o;
}
// The probability of the entry's id, of all entries that name it: what the
// gradient takes off there. Called by every thread.
#define DS_HASH 256   // twice the entries: a free slot is near
struct ds_ids {
    uint32_t slot[DS_HASH], ids[DS_K], dup;
    float ps[DS_K];
};
template <int NT>
__device__ __forceinline__ float ds_of_id(const ds_entry& l, uint32_t K, ds_ids& d) {
    const uint32_t t = threadIdx.x;
    for (uint32_t i = t; i < DS_HASH; i += NT) d.slot[i] = 0xffffffffu;
    if (t == 0) d.dup = 0;
    if (t < DS_K) {
        d.ids[t] = l.there ? l.id : 0xffffffffu;
        d.ps[t] = l.there ? (float)l.p : 0.0f;
    }
    __syncthreads();
    if (l.there) {
        for (uint32_t s = l.id * 2654435761u >> 24;; s = (s + 1u) % DS_HASH) {
            const uint32_t was = atomicCAS(&d.slot[s], 0xffffffffu, l.id);
            if (was == 0xffffffffu) break;
            if (was == l.id) { d.dup = 1; break; }
        }
    }
    __syncthreads();
    float p = (float)l.p;
    if (d.dup && l.there) {
        p = 0.0f;
        for (uint32_t k = 0; k < K; k++) p += d.ids[k] == l.id ? d.ps[k] : 0.0f;
    }
    return p;
}
// 2^-d of the rounding d of a product
__device__ __forceinline__ double df_undo(float m, float c) {
    const double d = (double)fmaf(m, c, -(m * c));
    if (fabs(d) < 0x1p-8) {   // (three terms: within 2^-36)
        const double y = d * 0.6931471805599453;
        return fma(y, fma(y, fma(y, -1.0 / 6.0, 0.5), -1.0), 1.0);
    }
    return exp2(-d);
}
// The sum of exp((x - m) / T) over the ids outside the list, and its m: the
// row's maximum, or that of those ids.
struct ds_out {
    double s, m;
};
// Is it wanted relative to their own? The terms that a sum relative to the row's
// maximum has lost are less than 2^-106 in all, 2^-42 of it at 2^-64. (w: the
// weight of the tail's term; the second test keeps w pt / s a float.) The same
// on every thread of the workgroup.
__device__ __forceinline__ bool ds_far(const ds_args& a, double pt, double s, float w) {
    const float sf = (float)s, pf = (float)pt;
    const bool far = a.kl != 0.0f && pf > 0.0f && (sf < 0x1p-64f || fabsf(w) * pf > sf * 0x1p100f);
    return __builtin_amdgcn_readfirstlane(far);
}
// The factor from sums relative to 2^(m c) to those relative to 2^(M c), m <= M.
__device__ __forceinline__ float ds_join(float m, float M, float c0) {
    const float Mr = M > -INFINITY ? M : 0.0f, c = hd_factor(Mr, c0);
    return m == M ? 1.0f : m > -INFINITY && hd_factor(m, c0) == c ? __builtin_amdgcn_exp2f(m * c - Mr * c) : 0.0f;
}
// begin(j0): called by every thread, vectors from j0 on are next; in(j): bits of
// vector j's ids that are in the list. Called by every thread.
template <int DT, int NT, int U, class Begin, class In>
__device__ __forceinline__ ds_out ds_outside(const ds_args& a, const hd_row<DT>& row, double m_row, double* shd, Begin begin, In in) {
    constexpr int E = hd_elem<DT>::E;
    float m = -INFINITY, s = 0.0f;
#pragma unroll 1
    for (uint32_t j0 = 0; j0 < row.nvec; j0 += U * NT) {
        hd_u4 v[U];
        row.take(j0 + threadIdx.x, NT, row.inside(j0) && row.inside(j0 + U * NT - 1u), v);
        begin(j0);
        float x[U][E], M = m;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t b = in(j0 + threadIdx.x + (uint32_t)(u * NT));
            hd_unpack<DT>(v[u], x[u]);
#pragma unroll
            for (int q = 0; q < E; q++) {
                x[u][q] = b >> q & 1u ? -INFINITY : x[u][q];
                M = fmaxf(M, x[u][q]);
            }
        }
        const float Mr = M > -INFINITY ? M : 0.0f, c = hd_factor(Mr, a.c), Mc = Mr * c;
        s *= ds_join(m, M, a.c);
        m = M;
#pragma unroll
        for (int u = 0; u < U; u++) {
            float e[E];
#pragma unroll
            for (int q = 0; q < E; q++) e[q] = __builtin_amdgcn_exp2f(fmaf(x[u][q], c, -Mc));
            s += hd_sum(e);
        }
    }
    const float M = block_max_f<NT>(m, reinterpret_cast<float*>(shd));
    const double S = block_sum_d<NT>((double)(s * ds_join(m, M, a.c)), shd);
    if (!(M > -INFINITY)) return {0.0, m_row};   // nothing is outside
    return {S * df_undo(M, hd_factor(M, a.c)), (double)M};
}
// The row's loss (and what the backward pass needs) from its maximum and
// sums; xk: the entry's logit. Called by every thread.
template <int NT>
__device__ __forceinline__ void ds_loss(const ds_args& a, uint64_t r, const ds_entry& l, float xk, int64_t label, float xl,
                                        double m, double S, double S1, ds_out o, double* shd) {
    double term = 0.0;
    if (l.there && l.p != 0.0) term = l.p * (log(l.p) - (((double)xk - m) * a.inv_t - log(S)));   // (NaN stays)
    term = block_sum_d<NT>(term, shd);
    if (threadIdx.x) return;
    // (where the student has nothing outside, the rounding of the list's
    // probabilities is no tail: 128 of them are within 2^-21 of their sum)
    if (l.pt > 0.0 && !(o.s == 0.0 && l.pt < 0x1p-20)) {
        const double d = o.m == m ? 0.0 : (o.m - m) * a.inv_t;
        term += l.pt * (log(l.pt) - (log(o.s) - log(S) + d));
    }
    double loss = a.kl != 0.0f ? (double)a.kl * term : 0.0;
    if (a.labels) loss += a.ce != 0.0f ? (double)a.ce * (log(S1) - ((double)xl - m)) : xl == xl ? 0.0 : NAN;
    a.loss[r] = (float)loss;
    if (a.stats) {
        const double So = o.m == m ? o.s : o.s * exp((o.m - m) * a.inv_t);
        *reinterpret_cast<float4*>(a.stats + r * 4) = make_float4((float)m, (float)S, (float)S1, (float)So);
    }
}
// The gradient's factors; w: the loss's own.
__device__ __forceinline__ ds_coef ds_factors(const ds_args& a, float w, const ds_entry& l, bool bad_label, double m, double S,
                                              double S1, double So) {
    const double g = bad_label ? (double)NAN : (double)w;
    const double kl = g * a.kl * a.inv_t, ce = a.labels ? g * a.ce : 0.0;
    ds_coef k;
    // e = 2^(x c - mc) has mc's rounding for a factor
    const float mf = (float)m;
    k.c = hd_factor(mf, a.c);
    k.mc = mf * k.c;
    k.c1 = hd_factor(mf, (float)HD_LOG2E);
    k.m1 = mf * k.c1;
    const double f = df_undo(mf, k.c), f1 = df_undo(mf, k.c1);
    const double one = a.labels ? ce / S1 : 0.0;
    const double in = kl * l.P / S + (a.two ? 0.0 : one);
    k.fi = (float)(in * f);
    k.fo = (float)((in - (a.tail && So > 0.0 ? kl * l.pt / So : 0.0)) * f);
    k.co = k.c;
    k.mco = k.mc;
    k.f1 = (float)(one * f1);
    k.fp = (float)kl;
    k.fc = (float)ce;
    return k;
}

// Those of the ids outside the list, from a sum relative to their own maximum.
__device__ __forceinline__ void ds_factors_out(const ds_args& a, float w, const ds_entry& l, bool bad_label, double m, double S, ds_out o,
                                               ds_coef& k) {
    if (o.m == m) return;   // (none of them has mass, or the row's maximum is theirs)
    const double g = bad_label ? (double)NAN : (double)w, kl = g * a.kl * a.inv_t, in = kl * l.P / S + (a.labels && !a.two ? g * a.ce / S : 0.0);
    const float mo = (float)o.m;
    k.co = hd_factor(mo, a.c);
    k.mco = mo * k.co;
    k.fo = (float)((in * exp((o.m - m) * a.inv_t) - kl * l.pt / o.s) * df_undo(mo, k.co));
}

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
    const float w = WHAT & DS_GRAD ? a.row_grad[r * a.row_grad_stride] : 0.0f;
    const ds_entry l = ds_list<DF_NT>(a, r, shd);
    double m, S, S1, So;
    float xk = 0.0f, xl = NAN;
    if (WHAT & DS_LOSS) {
        if (l.there) xk = row.at(l.id);
        if (a.labels && !bad_label) xl = row.at((uint32_t)label);
        constexpr int E = hd_elem<DT>::E;
        const uint32_t recs = (row.nvec * E + HD_CHUNK - 1u) / HD_CHUNK * (HD_CHUNK / DS_WAVE);
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
    __shared__ ds_ids ids;
    float p = 0.0f;
    if (WHAT & DS_GRAD) p = ds_of_id<DF_NT>(l, a.K, ids);
    ds_out o = {So, m};
    // (a workgroup a row: where all rows are such, the loss of 512 x 128256 f32
    // takes 114 us for 49, of one bf16 row of 151936 40 for 14, the gradient of
    // 2048 x 50257 bf16 119 for 78. Where none is, 49, 14 and 78 as without it; of
    // 65536 rows of 1000, which are mostly ends, 258 for 247 and the gradient 242
    // for 230)
    const bool far = ds_far(a, l.pt, So, WHAT & DS_GRAD ? w * a.kl * (float)a.inv_t : a.kl);
    if (__builtin_expect(far, 0)) {
        constexpr int E = hd_elem<DT>::E, U = 4;
        __shared__ uint32_t mask[U * DF_NT / 4];   // a byte a vector: its ids in the list
        uint32_t at = 0;
        o = ds_outside<DT, DF_NT, U>(
            a, row, m, shd,
            [&](uint32_t j0) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < U / 4; i++) mask[i * DF_NT + t] = 0;
                __syncthreads();
                const uint32_t pos = l.id + row.shift, j = pos / E - j0;
                if (l.there && j < U * DF_NT) atomicOr(&mask[j / 4], 1u << (j % 4 * 8 + pos % E));
                __syncthreads();
                at = j0;
            },
            [&](uint32_t j) { return (uint32_t) reinterpret_cast<const uint8_t*>(mask)[j - at]; });
    }
    if (WHAT & DS_LOSS) ds_loss<DF_NT>(a, r, l, xk, label, xl, m, S, S1, o, shd);
    if (WHAT & DS_GRAD) {
        if (t < a.K) a.p[r * a.K + t] = l.there ? p : -1.0f;
        const bool listed = __syncthreads_or(l.there && (int64_t)l.id == label);
        if (t == 0) {
            ds_coef k = ds_factors(a, w, l, bad_label, m, S, S1, So);
            if (__builtin_expect(far, 0)) ds_factors_out(a, w, l, bad_label, m, S, o, k);
            k.lone = label < 0 || bad_label || listed ? 0xffffffffu : (uint32_t)label;
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
// e (in the list; outside it eo) and e1 (times its factor) of one value
template <bool TWO>
__device__ __forceinline__ void ds_exps(const ds_coef& k, float x, bool listed, float& e, float& e1) {
    e = __builtin_amdgcn_exp2f(fmaf(x, listed ? k.c : k.co, -(listed ? k.mc : k.mco)));
    e1 = TWO ? __builtin_amdgcn_exp2f(fmaf(x, k.c1, -k.m1)) * k.f1 : 0.0f;
}
// A vector of the gradient to ids i0 .. i0 + E - 1 of the row.
template <int DT>
__device__ __forceinline__ void ds_store(typename hd_elem<DT>::T* grad, uint32_t V, bool whole, int i0, const float (&y)[hd_elem<DT>::E]) {
    constexpr int E = hd_elem<DT>::E;
    if (whole) {
        hd_u4 v;
        if constexpr (DT == ZS_F32) v = hd_u4{__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3])};
        else v = hd_u4{hd_pack2<DT>(y[0], y[1]), hd_pack2<DT>(y[2], y[3]), hd_pack2<DT>(y[E / 2], y[E / 2 + 1]), hd_pack2<DT>(y[E - 2], y[E - 1])};
        *reinterpret_cast<hd_u4*>(grad + i0) = v;
    } else {
#pragma unroll
        for (int q = 0; q < E; q++)
            if ((uint32_t)(i0 + q) < V) ds_store1<DT>(grad + i0 + q, y[q]);
    }
}

// The gradient at an id of the list (p of it; fi) or at the label alone (fo).
template <bool TWO>
__device__ __forceinline__ float ds_at(const ds_coef& k, float x, bool listed, float p, bool label) {
    float e, e1;
    ds_exps<TWO>(k, x, listed, e, e1);
    return e * (listed ? k.fi : k.fo) + (e1 - ((listed ? k.fp * p : 0.0f) + (label ? k.fc : 0.0f)));
}

// Every id's gradient as one outside the list first; those of the list and the
// label are written over it by the wave that wrote their vector, whose stores
// arrive in order: no test per vector, and nothing is waited for.
template <int DT, bool TWO>
__global__ __launch_bounds__(DS_NT) void zs_k_distill_grad(ds_args a, uint64_t r0) {
    constexpr int E = hd_elem<DT>::E, U = DS_WAVE / 64 / E;
    typedef typename hd_elem<DT>::T T;
    __shared__ uint32_t hid[DS_K + 1];
    __shared__ float hy[DS_K + 1];
    __shared__ uint32_t hits;
    const uint32_t n = zs_quot(blockIdx.x, a.by_chunks), chunk = blockIdx.x - n * a.chunks, t = threadIdx.x;
    const uint64_t r = r0 + n;
    const hd_row<DT> row(a.logits, a.ld, r, a.V);
    const uint32_t first = chunk * (U * DS_NT);
    if (first >= row.nvec) return;
    T* grad = reinterpret_cast<T*>(a.grad) + r * a.ld_grad;
    const bool aligned = (((uintptr_t)grad ^ (uintptr_t)row.row) & 15u) == 0;
    float x[U][E];
    const bool skip = ds_skip(a, r);
    if (!skip) {
        const int64_t label = a.labels ? zs_gload(a.labels + r) : -1;
        uint32_t id = 0xffffffffu;
        float p = -1.0f;
        if (t < a.K) {
            id = zs_gload(a.ids + r * a.K + t);
            p = zs_gload(a.p + r * a.K + t);
        }
        const ds_coef k = a.coef[r];
        ds_load<DT, U>(row, first, x);
        if (t == 0) hits = 0;
        // the chunk's entries (p is NaN where the list has one), and the label where they do not have it
        const bool listed = t < a.K && p != -1.0f;
        if (t == DS_K) id = k.lone;
        const bool mine = (listed || t == DS_K) && id < a.V && (id + row.shift) / E - first < U * DS_NT;
        const float xk = mine ? row.at(id) : 0.0f;
        __syncthreads();
        if (mine) {
            const uint32_t h = atomicAdd(&hits, 1u);
            hid[h] = id;
            hy[h] = ds_at<TWO>(k, xk, listed, p, (int64_t)id == label);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int q = 0; q < E; q++) {
                float e, e1;
                ds_exps<TWO>(k, x[u][q], false, e, e1);
                x[u][q] = TWO ? e * k.fo + e1 : e * k.fo;
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
        ds_store<DT>(grad, a.V, aligned && row.inside(j), row.id0(j), x[u]);
    }
    if (skip) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (uint32_t h = (uint32_t)zs_lane(); h < hits; h += 64u)
        if ((((hid[h] + row.shift) / E - first) % DS_NT >> 6) == (uint32_t)zs_wid()) ds_store1<DT>(grad + hid[h], hy[h]);
}

// ---------------------------------------------------------------------------
// loss and gradient by one workgroup a row
// ---------------------------------------------------------------------------
// The row is read once for its sums and passes again, from its end backwards,
// for its gradient: the last two batches are still in registers, the first ones
// in shared memory (with 1024 threads, one workgroup a compute unit: up to two
// batches of 64 KB), what lies between is read again. Loads run a batch ahead of
// their use; they are issued without conditions (vectors at the row's ends are
// clamped to whole ones, the ends themselves read apart), or the compiler waits
// for all of them at every join of the branches. Bound by memory: 4096 rows of
// 151936 bf16, 2.49 GB, 506 us without the tail (4.9 TB/s) and 527 with it (what
// is not hidden: the list's and the row's end). As it was first, 517 and 590,
// against every batch read twice, 578 and 621, 512 threads, two workgroups a
// unit, 635, and passes of their own, 709.
// What is kept of a row's list while the row passes.
struct df_kept {
    double p[DS_K], pt, P;
    float x[DS_K + 1], pid[DS_K];   // logits of the entries (the label's last), probabilities of their ids
};
struct df_wave {
    double s, s1, so;
    float m;
};
template <int DT, bool TAIL, bool TWO, int FU_NT>
__global__ __launch_bounds__(FU_NT, 4) void zs_k_distill_fused(ds_args a, uint64_t r0, uint32_t room) {
    constexpr int E = hd_elem<DT>::E, U = 4, BV = U * FU_NT;   // vectors of a batch
    typedef typename hd_elem<DT>::T T;
    extern __shared__ hd_u4 shared[];   // room batches of the row, then (TAIL) a byte a vector, whole batches: its ids in the list
    __shared__ uint32_t hid[DS_K + 1];
    __shared__ float hy[DS_K + 1];
    __shared__ double shd[FU_NT / 64];
    __shared__ df_wave wv[FU_NT / 64];
    __shared__ df_kept kept;
    __shared__ ds_ids ids;
    const uint64_t r = r0 + blockIdx.x;
    const uint32_t t = threadIdx.x;
    const hd_row<DT> row(a.logits, a.ld, r, a.V);
    T* grad = reinterpret_cast<T*>(a.grad) + r * a.ld_grad;
    const bool aligned = (((uintptr_t)grad ^ (uintptr_t)row.row) & 15u) == 0;
    const int64_t label = a.labels ? a.labels[r] : -1;
    if (a.labels && label == a.ignore) {
        if (t == 0) a.loss[r] = 0.0f;
        const float zero[E] = {};
        for (uint32_t j = t; j < row.nvec; j += FU_NT) ds_store<DT>(grad, a.V, aligned && row.inside(j), row.id0(j), zero);
        return;
    }
    const bool bad_label = a.labels && (label < 0 || label >= (int64_t)a.V);
    const float rg = a.row_grad[r * a.row_grad_stride];   // (long before its use)
    const uint32_t nb = (row.nvec + BV - 1u) / BV;
    // whole vectors lo .. hi (rows of DS_FUSED_VOCAB ids have some); threads 0
    // and 1 have the vectors before and behind them
    const uint32_t lo = row.shift ? 1u : 0u, hi = (a.V + row.shift) / E - 1u;
    const uint32_t edge = t == 0 ? 0u : row.nvec - 1u;
    const bool has_edge = t < 2u && (t == 0 ? lo > 0u : hi + 1u < row.nvec);
    auto fetch = [&](uint32_t b, hd_u4 (&v)[U]) {
#pragma unroll
        for (int u = 0; u < U; u++) v[u] = row.load(min(max(b * BV + t + (uint32_t)u * FU_NT, lo), hi));
    };
    auto unpack = [&](const hd_u4 (&v)[U], uint32_t b, float (&x)[U][E]) {
#pragma unroll
        for (int u = 0; u < U; u++) hd_unpack<DT>(v[u], x[u]);
        if (b * BV < lo || b * BV + BV - 1u > hi) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t j = b * BV + t + (uint32_t)u * FU_NT;
#pragma unroll
                for (int q = 0; q < E; q++) x[u][q] = j >= lo && j <= hi ? x[u][q] : -INFINITY;
            }
        }
    };
    // the last two batches stay in registers, the first ones in shared memory
    const uint32_t keep = min(room, nb > 2u ? nb - 2u : 0u);
    uint32_t* mask = reinterpret_cast<uint32_t*>(shared + room * BV);
    hd_u4 cur[U], nxt[U], was[U];
    fetch(0, cur);
#pragma unroll
    for (int u = 0; u < U; u++) was[u] = cur[u];
    if (TAIL)
        for (uint32_t i = t; i < nb * (BV / 4); i += FU_NT) mask[i] = 0;
    bool listed;
    {
        const ds_entry l = ds_list<FU_NT>(a, r, shd);   // (its barriers order the clearing)
        if (TAIL && l.there) {
            const uint32_t pos = l.id + row.shift, j = pos / E;
            atomicOr(&mask[j / 4], 1u << (j % 4 * 8 + pos % E));
        }
        const float pid = ds_of_id<FU_NT>(l, a.K, ids);
        if (t < DS_K) {
            hid[t] = l.there ? l.id : 0xffffffffu;
            kept.p[t] = l.p;
            kept.pid[t] = pid;
            kept.x[t] = l.there ? row.at(l.id) : 0.0f;
        }
        if (t == DS_K) {
            kept.x[DS_K] = a.labels && !bad_label ? row.at((uint32_t)label) : NAN;
            kept.pt = l.pt;
            kept.P = l.P;
        }
        listed = __syncthreads_or(l.there && (int64_t)l.id == label);
    }
    const uint8_t* in_list = reinterpret_cast<const uint8_t*>(mask);
    // first pass: a maximum and sums per thread, relative to 2^ref
    const float c1 = (float)HD_LOG2E;
    float m = -INFINITY, s = 0.0f, so = 0.0f, s1 = 0.0f, c, ref, ct, ref1;
    auto raise = [&](float bm) {   // to a maximum of at least bm
        const float mr = bm > -INFINITY ? bm : 0.0f;
        c = hd_factor(mr, a.c);
        ref = mr * c;
        ct = TWO ? hd_factor(mr, c1) : c;
        ref1 = mr * ct;
        if (bm > m) {
            // (what came before a maximum whose factor is another has no mass beside it)
            const float f = m > -INFINITY && c == a.c ? __builtin_amdgcn_exp2f(m * c - ref) : 0.0f;
            s *= f;
            if (TAIL) so *= f;
            if (TWO) s1 *= m > -INFINITY && ct == c1 ? __builtin_amdgcn_exp2f(m * ct - ref1) : 0.0f;
            m = bm;
        }
    };
    auto add = [&](const float (&x)[E], uint32_t in) {
        float e[E];
        if (TWO) {
#pragma unroll
            for (int q = 0; q < E; q++) e[q] = __builtin_amdgcn_exp2f(fmaf(x[q], ct, -ref1));
            s1 += hd_sum(e);
        }
#pragma unroll
        for (int q = 0; q < E; q++) e[q] = __builtin_amdgcn_exp2f(fmaf(x[q], c, -ref));
        const float v = hd_sum(e);
        s += v;
        if (TAIL) {
            if (in) {
#pragma unroll
                for (int q = 0; q < E; q++) e[q] = in >> q & 1u ? 0.0f : e[q];
                so += hd_sum(e);
            } else {
                so += v;
            }
        }
    };
    for (uint32_t b = 0; b < nb; b++) {
        // (behind the last batch, the one that the second pass takes third)
        fetch(b + 1u < nb ? b + 1u : nb >= keep + 3u ? nb - 3u : b, nxt);
        if (b < keep) {
#pragma unroll
            for (int u = 0; u < U; u++) shared[b * BV + t + (uint32_t)u * FU_NT] = cur[u];
        }
        float x[U][E], bm = m;
        uint32_t in[U];
#pragma unroll
        for (int u = 0; u < U; u++) in[u] = TAIL ? in_list[b * BV + t + (uint32_t)u * FU_NT] : 0u;
        unpack(cur, b, x);
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int q = 0; q < E; q++) bm = fmaxf(bm, x[u][q]);
        raise(bm);
#pragma unroll
        for (int u = 0; u < U; u++) add(x[u], in[u]);
        if (b + 1u < nb) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                was[u] = cur[u];
                cur[u] = nxt[u];
            }
        }
    }
    if (has_edge) {
        float x[E], bm = m;
        row.get(edge, x, -INFINITY);
#pragma unroll
        for (int q = 0; q < E; q++) bm = fmaxf(bm, x[q]);
        raise(bm);
        add(x, TAIL ? in_list[edge] : 0u);
    }
    // the wave's relative to its maximum, then every wave by itself the row's
    // from theirs: one barrier, and no value from one thread to the others
    const float mw = wave_max_f(m);
    {
        const float f = ds_join(m, mw, a.c);
        df_wave w;
        w.m = mw;
        w.s = wave_sum_d((double)(s * f));
        w.so = TAIL ? wave_sum_d((double)(so * f)) : 0.0;
        w.s1 = TWO ? wave_sum_d((double)(s1 * ds_join(m, mw, c1))) : 0.0;
        if (zs_lane() == 0) wv[zs_wid()] = w;
    }
    __syncthreads();
    df_wave w = {0.0, 0.0, 0.0, -INFINITY};
    if (zs_lane() < FU_NT / 64) w = wv[zs_lane()];
    const float M = wave_max_f(w.m), Mr = M > -INFINITY ? M : 0.0f;
    const double f = (double)ds_join(w.m, M, a.c), u = df_undo(Mr, hd_factor(Mr, a.c));
    double S = wave_sum_d(w.s * f) * u, So = TAIL ? wave_sum_d(w.so * f) * u : 0.0, S1 = S;
    if (TWO) S1 = wave_sum_d(w.s1 * (double)ds_join(w.m, M, c1)) * df_undo(Mr, hd_factor(Mr, c1));
    if (!(M > -INFINITY)) S = S1 = NAN;   // a row of nothing has no distribution
    ds_entry l;
    l.there = t < DS_K && hid[t] < a.V;
    l.pt = kept.pt;
    l.P = kept.P;
    ds_coef k = ds_factors(a, rg, l, bad_label, (double)M, S, S1, So);
    ds_out o = {So, (double)M};
    // (not expected, or every row keeps ready what it needs: 534 us for 527 of
    // 4096 x 151936 bf16; where all rows are such 818)
    if (TAIL && __builtin_expect(ds_far(a, l.pt, So, rg * a.kl * (float)a.inv_t), 0)) {
        o = ds_outside<DT, FU_NT, 1>(a, row, (double)M, shd, [](uint32_t) {}, [&](uint32_t j) { return (uint32_t)in_list[j]; });
        ds_factors_out(a, rg, l, bad_label, (double)M, S, o, k);
    }
    // second pass, from the batch at hand backwards: every id as one outside
    // the list; the others are written over it as in zs_k_distill_grad
    if (t < DS_K) {
        if (l.there) hy[t] = ds_at<TWO>(k, kept.x[t], true, kept.pid[t], (int64_t)hid[t] == label);
    } else if (t == DS_K) {
        hid[DS_K] = label < 0 || bad_label || listed ? 0xffffffffu : (uint32_t)label;
        hy[DS_K] = ds_at<TWO>(k, kept.x[DS_K], false, 0.0f, true);
    }
    __syncthreads();
    auto derive = [&](float (&x)[E]) {   // a vector's gradient in the place of its values
#pragma unroll
        for (int q = 0; q < E; q++) {
            float e, e1;
            ds_exps<TWO>(k, x[q], false, e, e1);
            x[q] = TWO ? e * k.fo + e1 : e * k.fo;
        }
    };
    auto out = [&](uint32_t b, const hd_u4 (&v)[U]) {
        float x[U][E];
        unpack(v, b, x);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t j = b * BV + t + (uint32_t)u * FU_NT;
            derive(x[u]);
            if (j >= lo && j <= hi) ds_store<DT>(grad, a.V, aligned, row.id0(j), x[u]);
        }
    };
    auto next = [&]() {
#pragma unroll
        for (int u = 0; u < U; u++) {
            cur[u] = was[u];
            was[u] = nxt[u];
        }
    };
    uint32_t b = nb;
    while (b > keep + 3u) {
        b--;
        out(b, cur);
        next();
        fetch(b - 3u, nxt);
    }
    while (b > keep) {
        b--;
        out(b, cur);
        next();
    }
    while (b > 0u) {
        b--;
#pragma unroll
        for (int u = 0; u < U; u++) cur[u] = shared[b * BV + t + (uint32_t)u * FU_NT];
        out(b, cur);
    }
    if (has_edge) {
        float x[E];
        row.get(edge, x, -INFINITY);
        derive(x);
        ds_store<DT>(grad, a.V, false, row.id0(edge), x);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (uint32_t h = (uint32_t)zs_lane(); h <= DS_K; h += 64u) {
        const uint32_t id = hid[h], j = (id + row.shift) / E;
        const uint32_t owner = j < lo || j > hi ? 0u : j % FU_NT >> 6;
        if (id < a.V && owner == (uint32_t)zs_wid()) ds_store1<DT>(grad + id, hy[h]);
    }
    // the loss last: its logarithms pass while the stores do
    l.p = l.there ? kept.p[t] : 0.0;
    ds_loss<FU_NT>(a, r, l, t < DS_K ? kept.x[t] : 0.0f, label, kept.x[DS_K], (double)M, S, S1, o, shd);
}

template <int DT, int NT>
static void ds_fused(const ds_args& a, uint64_t r0, uint32_t n, hipStream_t stream) {
    const uint32_t batch = 4u * NT, nb = ((a.V + 7u) / hd_elem<DT>::E + 1u + batch - 1u) / batch;
    const uint32_t mask = a.tail ? nb * batch : 0u;   // a byte a vector, whole batches
    const uint32_t left = NT == 1024 ? (DS_FUSED_LDS - mask) / (batch * 16u) : 0u, room = left < nb ? left : nb, lds = room * batch * 16u + mask;
    if (a.tail && a.two) hipLaunchKernelGGL((zs_k_distill_fused<DT, true, true, NT>), dim3(n), dim3(NT), lds, stream, a, r0, room);
    else if (a.tail) hipLaunchKernelGGL((zs_k_distill_fused<DT, true, false, NT>), dim3(n), dim3(NT), lds, stream, a, r0, room);
    else if (a.two) hipLaunchKernelGGL((zs_k_distill_fused<DT, false, true, NT>), dim3(n), dim3(NT), lds, stream, a, r0, room);
    else hipLaunchKernelGGL((zs_k_distill_fused<DT, false, false, NT>), dim3(n), dim3(NT), lds, stream, a, r0, room);
}
template <int DT>
static void ds_go(const ds_args& a, int what, uint64_t r0, uint32_t n, hipStream_t stream) {
    const dim3 grid(n * a.chunks), wg(DS_NT);
    const uint32_t vec = (a.V + 7u) / hd_elem<DT>::E + 1u;   // vectors of a row at most
    if (what == (DS_LOSS | DS_GRAD) && (a.N >= DS_FUSED_ROWS || a.V <= DS_FUSED_SHORT) && a.V >= DS_FUSED_VOCAB && vec <= 49152u) {
        // against passes of their own (us, one launch against three): bf16 rows
        // of 4096 10 and 14 (16 rows), 30 and 27 (2048); of 32000 14 and 14 (16),
        // 17 and 22 (256), 61 and 91 (2048); of 65536 16 and 13 (16), 18 and 18
        // (96), 19 and 21 (128); of 151936 27 and 15 (16), 31 and 28 (96), 31 and
        // 33 (128), 291 and 351 (2048); f32 rows of 32000 13 and 15 (16), of
        // 151936 38 and 41 (96), 172 and 169 (512), 612 and 681 (2048)
        // 16384 bf16 rows of 32000: 483 us by 256 threads, 544 by 512, 827 by
        // 1024; 8192 of 65536: 540, 478, 571; 4096 of 151936 without the tail: 729, 635, 517
        // (506 now)
        if (vec <= 4u * 1024u) ds_fused<DT, 256>(a, r0, n, stream);
        else if (vec <= 4u * 2048u + 1u) ds_fused<DT, 512>(a, r0, n, stream);
        else ds_fused<DT, 1024>(a, r0, n, stream);
        return;
    }
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
