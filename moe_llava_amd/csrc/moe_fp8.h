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

typedef unsigned char u8;
typedef __attribute__((ext_vector_type(8))) int v8i_t;
typedef __attribute__((ext_vector_type(4))) int v4i_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;

constexpr int QB = 128;               // elements that share a scale along K (and weight rows along N)
constexpr int DIM_MAX = 0x7fffffff - 511;  // rows, and columns of either operand: rounding up to a tile (at most 256) stays in 32 bits
inline bool grid_fits(long long blocks, int threads) { return blocks * threads <= 0xffffffffLL; }  // a launch has 2^32 - 1 threads at most
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

// Activations in fp32: nothing is rounded to 16 bits between the accumulator and the quantisation (that would move ~1 % of
// the elements to a neighbouring e4m3 value).  v_exp_f32 and v_rcp_f32 are good to a unit in the last place each, and the
// rounding of the exponential's argument t (a for silu, 2 u below) makes |t| 2^-23 of it: (|t| + 4) 2^-23 of the result, 2^-19
// at |t| = 12, here and in fast_silu (moe_common.h).  The accumulators under them are good to 2^-16 (moe_fp8.hip), and e4m3's
// half step is 2^-4.
__device__ __forceinline__ float gelu_new_f32(float x) {
    // 0.5 x (1 + tanh u) = x / (1 + 2^(-2u log2 e)), u = sqrt(2 / pi) (x + 0.044715 x^3): the exponent is x (c0 + c1 x^2)
    constexpr float c0 = -2.f * 0.7978845608028654f * 1.4426950408889634f, c1 = c0 * 0.044715f;
    return x * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * fmaf(c1, x * x, c0)));
}

struct Fp8GemmParams {
    const u8 *a;              // rows, e4m3, row stride lda bytes
    long long lda;
    const u8 *a_scale;        // e8m0 [rows, ceil(K/128)], row stride lds_a bytes (a multiple of 4, rows 4-byte aligned)
    long long ld_as;
    const int *gather;
    int gather_shift;
    const u8 *w;              // [experts, N (or 2N), K]
    long long w_expert_stride;
    const u8 *w_scale;        // [experts, blocks of N (or 2x), ceil(K/128)], dense
    long long ws_expert_stride;
    const bf16_t *bias;
    long long bias_expert_stride;
    const int *group_offsets; // NULL: one group, rows [0, max_rows)
    int G, n_experts, max_rows;
    void *out;                // 16-bit [rows, ldo], or e4m3 with out_scale
    long long ldo;
    u8 *out_scale;            // [rows, ceil(N/128)], row stride ld_os
    long long ld_os;
    int K, N_out;
    int b_row_offset;         // gated: weight row of the first 'b' projection row (= N_out)
    int b_blk_offset;         // gated: row of the scales' grid where the 'b' projection starts
    int n_gated;              // gated: columns from here on are not gated; < N_out, or INT_MAX (all are gated)
    int col_tiles, rs;
    int vec_store;            // 16-bit output: rows and pointer allow 16-byte stores
    int zero_tail;            // 16-bit output: rows of [0, max_rows) that belong to no group are set to 0
    int dtype;
    float *splitk_ws;         // K pieces of the 256 x 256 tiles of a last round (Fp8Sched); NULL: tiles stay whole
    int split_max;            // most pieces of a tile
};

// Plain products of few rows (moe_fp8_gemv.hip); fp8_gemm in moe_fp8.hip says when it is taken.
constexpr int FP8_FEW_ROWS = 64;
int launch_fp8_few(const Fp8GemmParams &p, hipStream_t st);

}  // namespace moe
