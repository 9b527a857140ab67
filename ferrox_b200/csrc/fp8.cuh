// The 8-bit form of cached keys and values.  A position of a head is head_dim bytes of e4m3 (1 sign, 4 exponent and 3
// mantissa bits, largest value 448, no infinity) and one exponent byte E: element i stands for e4m3(byte i) * 2^(E - 127).
//
//   a = max |x_i|,  e = the smallest whole number with a <= 448 * 2^e, at least FX_FP8_MIN_EXP;  E = e + 127
//   byte i = x_i * 2^-e rounded to nearest, ties to even
//
// Powers of two as scales, because multiplying by them rounds nothing: the one rounding is e4m3's own (half a step, 2^-4 of
// the value), what is read back is exact in bfloat16 (4 significant bits, and 2^(FX_FP8_MIN_EXP - 9) is its smallest
// multiple of a step), and a position's scale can be applied to a score or to a weight instead of to its elements without
// another result.  e4m3 is a floating type: a scale that is not a power of two would buy no precision, only range.
// The largest number held is FX_FP8_MOST: what is nearer to 2^128, which is past the largest number of 32 bits, is held as that.
// A row with an element that is infinite or no number has E = FX_FP8_NAN and bytes of 0; every element of it is NaN.
#pragma once
#include "common.cuh"

constexpr int FX_FP8_MIN_EXP = -119, FX_FP8_MAX_BYTE = 247, FX_FP8_NAN = 255;      // (2^120: the largest scale there is)
#define FX_FP8_MOST __uint_as_float(0x7f700000u)                                   // 240 * 2^120

// Exponent byte of a row whose largest |x| has the bits `amax` (any pattern; 0x7f800000 and above: infinite or no number).
__device__ __forceinline__ int fx_fp8_exponent(uint32_t amax) {
    if (amax >= 0x7f800000u) return FX_FP8_NAN;
    const int e = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u);      // (448 = 1.75 * 2^8)
    return max(e, FX_FP8_MIN_EXP + 127);
}
// What an element is multiplied with before it is rounded: 2^-e (a normal number for every e there is).
__device__ __forceinline__ float fx_fp8_inverse(int exponent) { return __uint_as_float((uint32_t)(254 - exponent) << 23); }
// What a byte's value is multiplied with when it is read: 2^e; NaN for FX_FP8_NAN (its bits: infinity's, times 0 or less).
__device__ __forceinline__ float fx_fp8_scale(int exponent) {
    return exponent == FX_FP8_NAN ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)exponent << 23);
}
__device__ __forceinline__ uint32_t fx_fp8_pack2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// Two bytes (the low half of v) as two 16-bit floating numbers, exactly.
__device__ __forceinline__ uint32_t fx_fp8_unpack2(uint32_t v) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)v));
    return r;
}
__device__ __forceinline__ float2 fx_fp8_float2(uint32_t v) {
    const uint32_t h = fx_fp8_unpack2(v);
    float2 f;
    asm("{.reg .b16 a, b; mov.b32 {a, b}, %2; cvt.f32.f16 %0, a; cvt.f32.f16 %1, b;}" : "=f"(f.x), "=f"(f.y) : "r"(h));
    return f;
}

// Where a request's position lies: its page, or -1 (none, or a position or a page outside the table and the pool).
__device__ __forceinline__ int fx_page_of(const int* table, int table_width, int n_pages, int pos, int page_size) {
    const int at = pos / page_size;
    if (pos < 0 || at >= table_width) return -1;
    const int page = table[at];
    return page < n_pages ? page : -1;
}
