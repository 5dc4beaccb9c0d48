// Layout of 4-bit rows, and the decoding that every kernel on them shares.
//
// A row is dim_pad = 128 KS elements in groups of 32; a group is 32 E2M1 codes (0 .5 1 1.5 2 3 4 6 and their negatives, the
// first element in the low bits) and one byte e + 127: element = code * 2^e.  e is the smallest exponent that keeps the
// group's largest magnitude within 7 * 2^e, and each code is the nearest one, ties to the even code -- so nothing in a
// group is off by more than half the step of its top binade, and storing what was read back gives the same codes.
// A group with a NaN or an infinite element gets the byte 255, which reads as NaN.
//
// Rows lie in tiles of 32, as v_mfma_scale_f32_32x32x64_f8f6f4 takes them for its A operand: lane l holds 16 bytes, a group, of
// row l % 32 at each K step.  Which groups make a step is free as long as the B operand agrees, and so a lane's groups of four
// steps are neighbours: line b of a row, 128 bytes, is its groups 8 b .. 8 b + 7, the first four of them lane l < 32's at steps
// 4 b .. 4 b + 3, the others lane l + 32's.  (Two steps are left where KS % 4 is 2: half a line, two groups and two.)  A tile is
// its rows' lines b, for every b, then 64 lanes x SW words of scale bytes, the two lanes of a row together (byte k = step k).
// A row that is re-scored is whole lines; with every step's groups side by side in the tile it was a 16-byte piece out of each
// of its 2 KS lines (1024 queries, 233 rows of 1024 elements each: k_finalize 205 us, so laid out 143).
#pragma once
#include "crag_common.h"

// KS: steps of 64 elements
__host__ __device__ constexpr int crag_fp4_sw(int ks) { return (ks + 3) / 4; }
__host__ __device__ constexpr long long crag_fp4_tile_bytes(int ks) { return 1024ll * ks + 256ll * crag_fp4_sw(ks); }
// The B operand: blocks of 32 columns, ks * pieces operands of 64 lanes x 24 bytes, then 64 lanes x words of scale bytes.
// Wide form: column = query, two pieces.  Narrow form: column c = first piece of query c, 16 + c = its second piece.
__host__ __device__ constexpr int crag_fp4_qsw(int ks, int pieces) { return (ks * pieces + 3) / 4; }
__host__ __device__ constexpr long long crag_fp4_qblock_bytes(int ks, int pieces) { return 64ll * 24 * ks * pieces + 256ll * crag_fp4_qsw(ks, pieces); }

#define CRAG_FP4_EXP_MIN (-125)
#define CRAG_FP4_EXP_MAX 125

// step and half (0: lanes below 32) of a row's group
__host__ __device__ inline void crag_fp4_step(int ks, int grp, int* step, int* half) {
    const int b = grp >> 3;
    if (b * 4 + 4 <= ks) {
        *step = b * 4 + (grp & 3);
        *half = (grp >> 2) & 1;
    } else {
        *step = b * 4 + (grp & 1);
        *half = (grp >> 1) & 1;
    }
}
// where group `grp` of a row lies: its 16 bytes of codes, its scale byte
__host__ __device__ inline void crag_fp4_place(int dim_pad, long long row, int grp, long long* codes, long long* scale) {
    const int ks = dim_pad >> 6, r = (int)(row & 31), b = grp >> 3;
    const long long base = (row >> 5) * crag_fp4_tile_bytes(ks);
    int step, half;
    crag_fp4_step(ks, grp, &step, &half);
    *codes = base + 4096ll * b + r * (b * 4 + 4 <= ks ? 128 : 64) + (grp & 7) * 16;
    *scale = base + 1024ll * ks + (long long)(r * 2 + half) * 4 * crag_fp4_sw(ks) + step;
}
// 2^(b - 127) of a scale byte (>= 2 and <= 252, or 255)
__device__ __forceinline__ float crag_fp4_scale(uint32_t b) { return b == 255u ? __builtin_nanf("") : __builtin_bit_cast(float, b << 23); }
// value of one code
__device__ __forceinline__ float crag_fp4_value(uint32_t c, float scale) {
    const uint32_t t = c & 7u;
    const float m = t < 2u ? 0.5f * (float)t : __builtin_bit_cast(float, ((126u + (t >> 1)) << 23) | ((t & 1u) << 22));
    return (c & 8u ? -m : m) * scale;
}
