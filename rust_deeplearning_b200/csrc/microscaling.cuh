// The microscaling formats the 4-bit weights and the 8-bit rows are held in, and what their kernels share.
//
// A group is 32 consecutive columns of a row with one scale 2^(c - 127), c eight bits (255: the group is NaN).
//   weights  e2m1: 0 0.5 1 1.5 2 3 4 6 and a sign, two codes a byte, the even column in the low half
//   rows     e4m3: the largest value is 448
// c is the smallest code >= 0 with amax <= top * 2^(c - 127), top 6 or 448, so that nothing is cut off; a group that holds an
// infinity or a NaN has c = 255.  Codes are value * 2^(127 - c) rounded to nearest, ties to even.
//
// Columns are padded to whole blocks of 128 (four groups) with zero codes.
//   weights  tiles of 128 rows x 128 columns, one after another along the columns: codes [rows / 128][blocks][128][64 bytes], scales
//            [rows / 128][blocks][32][4][4]: the four scales of row 32 c + l at [l][c], the order a tensor-core product wants.
//            A tile is 8 KB and 512 bytes in one piece.  (Rows in one piece each were read 64 bytes at a time: the output head
//            of the 2B shape took 133 us.)  Rows are padded to 128.  A [gate; up] matrix lays 16 gate rows before the 16 up rows
//            of the same outputs, so that a tile holds both halves of 64 outputs.
//   rows     values [rows padded to 4][padded columns]; scales [blocks][rows padded to 4][4].
#pragma once

#include "common.cuh"

constexpr int MX_GROUP = 32, MX_BLOCK = 128, MX_ROWS = 128, MX_UNIT = 16;
static inline int mx_blocks(int columns) { return (columns + MX_BLOCK - 1) / MX_BLOCK; }

// which row of a weight lies at `place`, or -1: padding; rows: of the matrix, half: outputs of a [gate; up] matrix, 0: not one
__device__ __forceinline__ int mx_row_at(int place, int rows, int half) {
    if (half == 0) return place < rows ? place : -1;
    const int up = place / MX_UNIT & 1, o = place / (2 * MX_UNIT) * MX_UNIT + place % MX_UNIT;
    return o < half ? o + up * half : -1;
}
// bytes from the start of the codes to the one of (place, column), and of the scales to the one of its group
__device__ __forceinline__ long long mx_code_at(int place, int column, int blocks) {
    return (((long long)(place / MX_ROWS) * blocks + column / MX_BLOCK) * MX_ROWS + place % MX_ROWS) * (MX_BLOCK / 2) + column % MX_BLOCK / 2;
}
__device__ __forceinline__ long long mx_scale_at(int place, int column, int blocks) {
    return ((long long)(place / MX_ROWS) * blocks + column / MX_BLOCK) * (MX_ROWS * 4) + place % 32 * 16 + place % MX_ROWS / 32 * 4 + column % MX_BLOCK / MX_GROUP;
}

// The scale code of a group from its largest magnitude; TOP_EXP, TOP_MANT: the format's largest value is 1.TOP_MANT x 2^TOP_EXP.
template <int TOP_EXP, uint32_t TOP_MANT>
__device__ __forceinline__ uint32_t mx_scale_code(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    const int c = (int)(bits >> 23) - TOP_EXP + ((bits & 0x7fffffu) > TOP_MANT ? 1 : 0);
    return bits >= 0x7f800000u ? 255u : (uint32_t)max(c, 0);
}
__device__ __forceinline__ uint32_t mx8_scale_code(float amax) { return mx_scale_code<8, 0x600000u>(amax); }      // 448 = 1.75 x 2^8
__device__ __forceinline__ uint32_t mx4_scale_code(float amax) { return mx_scale_code<2, 0x400000u>(amax); }      // 6 = 1.5 x 2^2
// 2^(127 - c) for the codes the two functions above return (at most 253; 255: NaN, so that every code of the group becomes one)
__device__ __forceinline__ float mx_inverse_scale(uint32_t c) { return __uint_as_float(c == 255u ? 0x7fc00000u : (254u - c) << 23); }
// 2^(c - 127) for every c: 0 is 2^-127 (not normal), 255 is NaN; both are bit 22 beside the shifted code
__device__ __forceinline__ float mx_scale(uint32_t c) { return __uint_as_float((c << 23) | ((((c + 1u) & 0xfeu) == 0u) ? 0x400000u : 0u)); }

// The larger magnitude; a NaN on either side stays (fmaxf would drop it).
__device__ __forceinline__ float mx_larger(float m, float v) {
    const uint32_t a = __float_as_uint(m), b = __float_as_uint(v) & 0x7fffffffu;      // as integers magnitudes are in order, NaN the largest
    return __uint_as_float(a > b ? a : b);
}

// four values, already scaled, to e4m3: value i in byte i
__device__ __forceinline__ uint32_t mx_to_e4m3(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | ((uint32_t)hi << 16);
}
// eight values, already scaled, to e2m1: value i in bits [4 i, 4 i + 4)
__device__ __forceinline__ uint32_t mx_to_e2m1(const float (&v)[8]) {
    uint32_t r;
    asm("{\n.reg .b8 a, b, c, d;\n"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\ncvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        "mov.b32 %0, {a, b, c, d};\n}"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// eight e2m1 codes to four pairs of f16
__device__ __forceinline__ void mx_from_e2m1(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n.reg .b8 a, b, c, d;\nmov.b32 {a, b, c, d}, %4;\n"
        "cvt.rn.f16x2.e2m1x2 %0, a;\ncvt.rn.f16x2.e2m1x2 %1, b;\ncvt.rn.f16x2.e2m1x2 %2, c;\ncvt.rn.f16x2.e2m1x2 %3, d;\n}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
// two e4m3 values (the low half of w)
__device__ __forceinline__ float2 mx_from_e4m3(uint32_t w) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)w));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
