// zs_q4.h -- a vocabulary head held in 4 bits: its layout, and kernel arguments.
#pragma once
#include <hip/hip_runtime.h>
#include "zs_head_args.h"

// The head lies in tiles of 16 rows (ids) by 128 columns, one behind the other
// along the columns, 1 KB each: lane l of a wave has row l % 16 and, of each of
// four blocks of 32 columns, the eight from (l / 16) * 8 on, as one 32-bit word.
// Its columns 2 j lie in the four bits from 3 + 4 j on, j < 3, its columns 2 j + 1
// in those from 19 + 4 j on; column 6 has the bits 15 to 18, column 7 the bits 31
// and 0 to 2. (Right by 4 j, at the end around, the pair j then stands at bits 3
// and 19, where a mask makes bf16 operands of it: j = 0 without a shift.)
// Behind the tiles the scales (f16, 128 / group of a row and tile side by side,
// rows next to each other), behind those the minima likewise.
struct q4_layout {
    uint32_t tiles, blocks;      // of rows, of columns
    uint64_t scales, mins, end;  // bytes
};
inline q4_layout q4_of(uint32_t V, uint32_t D, uint32_t group, bool mins) {
    q4_layout q;
    q.tiles = (V + 15u) / 16u;
    q.blocks = (D + 127u) / 128u;
    const uint64_t n = (uint64_t)q.tiles * q.blocks, s = hd_pad(n * 16u * (128u / group) * 2u);
    q.scales = n * 1024u;
    q.mins = q.scales + s;
    q.end = q.mins + (mins ? s : 0u);
    return q;
}
struct q4_args {
    const char* head;
    q4_layout at;
    uint32_t V, D, B;
    const void* hidden;          // rows of 16-bit values at 16 bytes each (planes one behind the other)
    uint64_t ld_h, plane;        // elements
    const float* sums;           // of groups of more than Q4_FEW rows (q4_x_args)
    uint32_t Bp;
    const int32_t* shift;        // f32: of each row (q4_x_args)
    float* logits;
    uint64_t ld;
};
#define Q4_FEW 16u               // rows up to which each wave makes its operands and sums by itself
struct q4_pack_args {
    q4_layout at;
    uint32_t V, D, group;
    uint8_t* codes;              // [V][D / 2]
    uint16_t *scales, *mins;     // [V][D / group] f16
    char* head;
    const void* weight;          // to be quantised
    uint64_t ld_w;
};
struct q4_x_args {               // hidden states to rows the kernels take
    const void* hidden;
    uint64_t ld_h;
    uint32_t B, D, group, Bp;
    float off;                   // what codes are moved by as operands: -24, with minima -16
    int32_t* shift;              // [B] f32: the powers of two the rows are scaled by
    uint16_t* out;               // [planes][B][D], or NULL: they serve as they are
    float* sums;                 // [D / group][Bp], or NULL
};
inline uint32_t q4_bp(uint32_t B) { return (B + 15u) / 16u * 16u + 64u; }   // (a part's last tile of rows may be past B)
inline uint64_t q4_work(q4_x_args& x, uint32_t dtype, bool copy, void* work) {
    char* p = (char*)work;
    const bool wide = dtype == ZS_F32;
    if (copy || wide) {
        x.out = (uint16_t*)p;
        p += hd_pad((uint64_t)x.B * x.D * (wide ? 4u : 2u));
    }
    if (wide) {
        x.shift = (int32_t*)p;
        p += hd_pad(x.B * 4ull);
    }
    if (x.B > Q4_FEW) {
        x.sums = (float*)p;
        p += hd_pad((uint64_t)(x.D / 32u + 4u) * x.Bp * 4u);
    }
    return (uint64_t)(p - (char*)work);
}
int q4_pack(const q4_pack_args& a, hipStream_t stream);
int q4_quantize(const q4_pack_args& a, uint32_t dtype, hipStream_t stream);
int q4_logits(const q4_args& a, const q4_x_args* x, uint32_t dtype, uint32_t group, bool mins, hipStream_t stream);
