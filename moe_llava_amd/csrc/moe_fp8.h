// The 8-bit format of the fp8 operators: e4m3 (OCP) elements, one power-of-two scale per block of 128 (1 x 128 for
// activation rows, 128 x 128 for weights), held as an e8m0 exponent byte.
//
// The exponent e is the smallest with max|x| * 2^-e <= 448.  A power of two because (1) scaling then rounds nothing: the
// only rounding is the one to e4m3, and 32- and 64-bit arithmetic agree on it (a generic scale max|x| / 448 puts 16-bit
// inputs on rounding ties of e4m3, which then fall by the last bit of the division); (2) a floating-point element loses
// no precision from it, only part of one binade of range at the small end; (3) v_mfma_scale_f32_16x16x128_f8f6f4 takes
// e8m0 bytes as operands, so the products cost no vector instruction per block of K.
#pragma once
#include "moe_common.h"

namespace moe {

constexpr int QB = 128;               // elements that share a scale along K (and weight rows along N)
constexpr unsigned E8M0_NAN = 255u;   // scale of a block that holds an infinity or a NaN; its elements are all NaN

// |x| as an integer that orders like the magnitude, NaN above infinity: a maximum over it cannot lose a NaN
__device__ __forceinline__ unsigned abs_bits(float x) { return __builtin_bit_cast(unsigned, x) & 0x7fffffffu; }

// e8m0 byte of a block whose largest magnitude has these bits.  448 = 1.75 * 2^8: a mantissa above 1.75 needs the next
// exponent.  Blocks of zeros (and of magnitudes below 2^-118) take the smallest exponent whose inverse is a finite fp32.
__device__ __forceinline__ unsigned scale_byte(unsigned top) {
    if (top >= 0x7f800000u) return E8M0_NAN;
    const int b = (int)((top + 0x1fffffu) >> 23) - 8;
    return (unsigned)(b < 1 ? 1 : b);
}
// 2^-(byte - 127): exact; NaN for the NaN byte, so that every element of such a block becomes NaN
__device__ __forceinline__ float inv_scale(unsigned byte) {
    return __builtin_bit_cast(float, byte == E8M0_NAN ? 0x7fc00000u : (254u - byte) << 23);
}
// four fp32 values -> four e4m3 bytes (round to nearest even; the block's scale keeps them at or below 448)
__device__ __forceinline__ unsigned pack_fp8x4(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}
__device__ __forceinline__ unsigned umax_xor(unsigned v, int mask) {
    const unsigned o = (unsigned)__shfl_xor((int)v, mask, 64);
    return v > o ? v : o;
}

}  // namespace moe
