// Rows of keys and values in eight bits: D codes of e4m3 (a sign, four bits of exponent, three of mantissa, 448 at most) and one
// exponent byte b a row; a value is code * 2^(b - 127).
//
// The exponent is n = b - 127 = the smallest with max |x| <= 448 * 2^n, held within -60 .. 60: powers of two, so that x * 2^-n is
// exact, the code's rounding is the only one, and a code times its power is exact in bfloat16 and float32 again.  The limits (values
// beyond 448 * 2^60 become that, those below 2^-70 zeros) keep a score that is summed over codes within 32 bits when it is given
// its power.  A row of zeros has b = 127.  A row with an infinity or a NaN has
// b = 255 and codes of zero, and reads as NaN throughout: no code is ever a NaN itself, so that a row that nobody attends can
// be multiplied by a weight of zero.
#pragma once
#include "common.cuh"

enum : int { LLMX_E4M3 = 2 };     // an element type of caches only (codes, with exponents beside them)

namespace e4m3 {

constexpr int LOWEST = -60, HIGHEST = 60;
constexpr unsigned NOT_NUMBERS = 255;

// The exponent byte of a row whose largest magnitude has the bits `peak` (of a float without its sign).  Magnitudes compare as
// their bits do, infinities and NaN above all numbers.
__device__ __forceinline__ unsigned exponent_byte(unsigned peak) {
    if (peak == 0) return 127;
    if (peak >= 0x7F800000u) return NOT_NUMBERS;
    const int n = (int)(peak >> 23) - 127 - 8 + ((peak & 0x7FFFFFu) > 0x600000u);      // 448 = 1.75 * 2^8
    return (unsigned)(min(max(n, LOWEST), HIGHEST) + 127);
}

// 2^-n, what a row's values are multiplied by before their rounding (of a row that has numbers).
__device__ __forceinline__ float down(unsigned byte) { return __uint_as_float((254u - byte) << 23); }

// 2^n, NaN for a row that is no numbers.  (b = 0, which no row has, counts as zero.)
__device__ __forceinline__ float up(unsigned byte) { return byte == NOT_NUMBERS ? __uint_as_float(0x7FC00000u) : __uint_as_float(byte << 23); }

// Two codes, `lo` in the lower byte; beyond 448 the largest code.
__device__ __forceinline__ unsigned pack2(float lo, float hi) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// Two codes as two halves (every code is one exactly).
__device__ __forceinline__ unsigned halves(unsigned short codes) {
    unsigned r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(codes));
    return r;
}

}  // namespace e4m3
