// zs_ce.h -- kernel arguments of the cross entropy from hidden states and the
// layout of its scratch.
#pragma once
#include <hip/hip_runtime.h>
#include "zs_head_args.h"
#include "zs_tile.h"

#define CE_TILE 256         // ids, rows or columns of a product's tile; of few rows:
#define CE_THIN_M 128       // ids or columns
#define CE_THIN 64          // rows
// f32 weights are multiplied as they lie up to so many rows, and as two planes that
// are made of them once above. us of the loss / of a step as they lie and as planes,
// 3456 x 58134: 1 row 268 / 704 and 628 / 1052, 128 rows 449 / 1291 and 743 / 1500, 192
// rows 618 / 1798 and 714 / 1676, 256 rows 805 / 2399 and 721 / 1843
#define CE_RAW 192u
#define CE_ROOM (4ull << 30)   // bytes of exponentials kept at once (a piece of the rows)

#define CE_DH 1u            // the gradient of the hidden states is wanted
#define CE_DW 2u            // the weight's
#define CE_COPY 4u          // the weight's rows do not begin and end at 16 bytes each: they are copied (f32: only where CE_RAW says so)
#define CE_FAR 8u           // they lie further apart than the products' offsets reach: they are copied
#define CE_E_SHIFT 15.0f
#define CE_E_SCALE 32768.0f // exponentials are kept as f16 of e * 2^15: 11 bits down to 2^-29 of their maximum

struct ce_state {           // what the device finds out
    uint32_t rows;          // that have a label
    uint32_t amax[64];      // bits of the piece's largest factors of a row's gradient, of every 64th row (f16; 1350
                            // rows' atomics on one address took 17 us)
};
struct ce_row {             // of a piece
    float fix;              // the gradient at the label
    uint32_t label;
    float fac, m;           // of an exponential in the gradient, relative to the row's largest logit m
    int32_t sh, sd;         // f32: the powers of two that its hidden state and its gradient of the logits (over the ids' own) are scaled by
};
struct ce_args {
    const void *hidden, *weight;
    uint64_t ld_h, ld_w;
    const int64_t* labels;
    int64_t ignore;
    uint32_t N, V, D, want;
    float zw;
    float *loss, *lse;
    const float* row_grad;
    uint64_t row_grad_stride;
    void *dh, *dw;
    uint64_t ld_dh, ld_dw;
    // the plan
    uint32_t Dp, Vp, R, pieces, sub, subs, thin, raw, units, Dm;   // raw: an f32 weight is multiplied as it lies, 1 by 16 bytes, 2 by 4
    uint32_t lo, first, last;    // the piece at hand: its first row; whether it is the first, the last
    // scratch
    ce_state* st;
    uint32_t* idx;               // [N] the rows with a label in order, behind them the others
    float* own;                  // [R][sub] logits of the `sub` ids that have the label among them
    ce_row* row;                 // [R]
    float2* stat;                // [R][subs] of `sub` ids each: maximum and sum of exponentials
    float* fac;                  // [R][subs] of an exponential in the gradient
    uint16_t* h;                 // [R][Dp] rows with a label, zeros behind them (f32: three planes, the weight's gradient's)
    uint16_t* w;                 // [V][Dp], where the weight itself does not serve (f32: two planes)
    void* e;                     // [R][Vp] f16 (f32: f32) exponentials
    uint16_t* dl;                // [R][Vp] gradient of the logits, in their place (of few rows a second plane; f32: three, the weight's gradient's)
    uint16_t *h2, *dl2;          // f32: the same as two planes of scaled rows, the logits' and the hidden states' gradient's
    int32_t* wsh;                // [Vp] f32: the powers of two that the weight's rows are scaled by
    float* lead;                 // [R][subs] the largest exponential over its id's power of two (the hidden states' gradient is wanted)
    float* part;                 // the hidden states' gradient over parts of the vocabulary (ce_parts)
    float* acc;                  // [V][Dm] the weight's gradient so far (more than one piece)
};
int ce_launch(const ce_args& a, uint32_t dtype, hipStream_t stream);
int ce_clear(void* p, uint32_t rows, uint32_t cols, uint64_t ld, uint32_t dtype, hipStream_t stream);   // zeros, where there are no rows

inline uint64_t ce_up(uint64_t n, uint64_t to) { return (n + to - 1u) / to * to; }
// N, V, D and want (CE_*) given, the plan and the scratch from `work`; the bytes.
inline uint64_t ce_work(ce_args& a, uint32_t dtype, void* work) {
    const bool wide = dtype == ZS_F32, grad = (a.want & (CE_DH | CE_DW)) != 0;
    const uint64_t planes = wide ? 3u : 1u;
    const bool dh = (a.want & CE_DH) != 0, dw = (a.want & CE_DW) != 0;
    a.Dp = (uint32_t)ce_up(a.D, TP_KSTEP);
    a.Vp = (uint32_t)ce_up(a.V, CE_TILE);
    a.Dm = (uint32_t)ce_up(a.D, 4);
    a.raw = !wide || (a.want & CE_FAR) || a.N > CE_RAW ? 0u : a.want & CE_COPY ? 2u : 1u;
    // A tile of 256 rows is 192 of them for nothing where there are 64, but the thin
    // tiles of 65 rows read the weight twice. us of a bf16 loss by thin tiles and by
    // others, 896 x 151936: 64 rows 67 and 118, 128 rows 92 and 118, 160 rows 116 and
    // 121; 4096 x 151936: 271 and 414, 389 and 424, 498 and 415; of a step, whose two
    // other products a tile more costs as much each, 896 x 151936: 64 rows 326 and 351,
    // 65 rows 421 and 357
    a.thin = a.raw || a.N <= (grad ? CE_THIN : 2u * CE_THIN);
    a.sub = a.thin ? 32u : 128u;
    a.subs = a.Vp / a.sub;
    uint64_t R = CE_ROOM / ((uint64_t)a.Vp * (wide ? 4u + (dw ? 6u : 0u) + (dh ? 4u : 0u) : 2u)) / CE_TILE * CE_TILE;
    const uint64_t most = grad ? 65280u : 16384u;   // (a launch's y; 1187 parts of 8 bytes a row at 151936 ids)
    if (!grad || R > most) R = most;
    if (R < CE_TILE) R = CE_TILE;
    a.R = (uint32_t)(R < a.N ? R : ce_up(a.N, CE_TILE));
    a.pieces = (uint32_t)((a.N + (uint64_t)a.R - 1u) / a.R);
    a.units = a.thin ? 512u : 256u;   // workgroups that fill the card
    char* p = (char*)work;
    auto take = [&](uint64_t bytes) { char* at = p; p += hd_pad(bytes); return (void*)at; };
    a.st = (ce_state*)take(sizeof(ce_state));
    a.idx = (uint32_t*)take(a.N * 4ull);
    a.own = (float*)take((uint64_t)a.R * a.sub * 4u);
    a.row = (ce_row*)take(a.R * sizeof(ce_row));
    a.stat = (float2*)take((uint64_t)a.R * a.subs * 8u);
    if (!wide || dw || a.raw) a.h = (uint16_t*)take(planes * a.R * a.Dp * 2u);
    if (wide ? !a.raw : (a.want & (CE_COPY | CE_FAR)) != 0) a.w = (uint16_t*)take((wide ? 2u : 1u) * (uint64_t)a.V * a.Dp * 2u);
    if (wide && !a.raw) {
        a.h2 = (uint16_t*)take(2u * (uint64_t)a.R * a.Dp * 2u);
        a.wsh = (int32_t*)take(a.Vp * 4ull);
    }
    if (grad) {
        a.fac = (float*)take((uint64_t)a.R * a.subs * 4u);
        a.e = take((uint64_t)a.R * a.Vp * (wide || a.thin ? 4u : 2u));   // (thin: a plane more behind it)
        a.dl = !wide ? (uint16_t*)a.e : dw || a.raw ? (uint16_t*)take(planes * a.R * a.Vp * 2u) : nullptr;
        if (wide && dh && !a.raw) {
            a.dl2 = (uint16_t*)take(2u * (uint64_t)a.R * a.Vp * 2u);
            a.lead = (float*)take((uint64_t)a.R * a.subs * 4u);
        }
        if (dh) a.part = (float*)take((uint64_t)a.units * (a.thin ? CE_THIN_M * CE_THIN : CE_TILE * CE_TILE) * 4u);
        if (dw && a.pieces > 1u) a.acc = (float*)take((uint64_t)a.V * a.Dm * 4u);
    }
    return (uint64_t)(p - (char*)work);
}
