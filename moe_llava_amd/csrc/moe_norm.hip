// Residual addition + root-mean-square norm in front of an MLP, with 16-bit and / or 8-bit output, and its backward; the
// 8-bit quantisation of rows and of weight blocks, and the transpose of an 8-bit weight (moe_fp8.h has the format).
//
//   s = round(x + r)      the new residual stream, in the rows' own type
//   y = s * rstd * w,  rstd = 1 / sqrt(mean(s^2) + eps)      sums and the product in fp32, one rounding at the output
//   q = e4m3 of the unrounded y, one scale per 128 columns
// backward, with n = s * rstd and g = dy * w:   dx = dr = rstd * (g - n * mean(g * n)) + ds,   dw = sum over rows of dy * n
//
// Bound: HBM (forward 8 bytes per element in 16 bits, + 1 for q; backward 8).  One pass: a row lives in the registers of its
// team (one wave per row for long batches, so no barrier; four or sixteen waves per row for few or very wide rows, where
// latency counts), 8 consecutive elements per lane and load, and the 16 lanes that hold a block of 128 columns agree on its
// maximum by shuffles.  A large copy reaches 5.1 TB/s on the same card (bytes read + written).  Measured, bf16:
//   forward   45056 x 2048: 131 us = 5.6 TB/s     2411 x 2560 with 8-bit rows, fp16: 12.0 us = 4.6 TB/s     1 x 2048: 3.0 us
//   backward  22528 x 2048: 71 us = 5.2 TB/s, and 4.7 us for the join of the 1024 partial weight gradients
//   quantize  rows of 22528 x 2048: 28 us = 4.9 TB/s, of 11264 x 2560: 20 us = 4.3 TB/s
//   transpose 8 x 2048 x 2560 bytes: 19 us = 4.4 TB/s
// With few rows a call costs the host's path (10 us without, 14.5 us with 8-bit rows) and not the kernel.
#include "moe_fp8.h"

namespace moe {

struct NormParams {
    const bf16_t *x, *res;
    long long ldx, ldr;
    const void *w;
    int w_f32;
    float eps;
    int S, M;
    bf16_t *y, *sum;
    long long ldy, lds;
    float *rstd;
    u8 *q, *scale;
    long long ldq, ld_scale;
};

// 8 elements from column c of a row of M; columns behind M read as 0
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const bf16_t *row, int c, int M, float *f) {
    if (VEC) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (c < M) v = *reinterpret_cast<const uint4 *>(row + c);
        unpack8_t<DT>(v, f);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = c + j < M ? Elt<DT>::to_f(row[c + j]) : 0.f;
    }
}
template <int DT, bool VEC>
__device__ __forceinline__ void store8(bf16_t *row, int c, int M, const float *f) {
    if (VEC) {
        if (c < M) *reinterpret_cast<uint4 *>(row + c) = pack8_t<DT>(f);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c + j < M) row[c + j] = Elt<DT>::from_f(f[j]);
    }
}
template <int DT>
__device__ __forceinline__ void load_w8(const void *w, int w_f32, int c, int M, float *f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 0.f;
    if (c >= M) return;
    if (c + 8 <= M && (reinterpret_cast<uintptr_t>(w) & 15) == 0) {
        if (w_f32) {
            const float4 a = *reinterpret_cast<const float4 *>((const float *)w + c);
            const float4 b = *reinterpret_cast<const float4 *>((const float *)w + c + 4);
            f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
        } else {
            unpack8_t<DT>(*reinterpret_cast<const uint4 *>((const bf16_t *)w + c), f);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (c + j < M) f[j] = w_f32 ? ((const float *)w)[c + j] : Elt<DT>::to_f(((const bf16_t *)w)[c + j]);
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m, 64);
    return v;
}
// sum over the TW waves of a team (one team per block when TW > 1); `buf` alternates between calls, so one barrier suffices
template <int TW>
__device__ __forceinline__ float team_sum(float v, float *red, int buf) {
    v = wave_sum(v);
    if (TW == 1) return v;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) red[buf * TW + wave] = v;
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < TW; ++w) t += red[buf * TW + w];
    return t;
}
// quantise 8 elements of a row (all 64 lanes call it together; 16 neighbouring lanes hold a block of 128 columns)
__device__ __forceinline__ void quant8(const float *f, int c, int M, u8 *qrow, u8 *srow) {
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const unsigned u = abs_bits(f[j]);
        top = u > top ? u : top;
    }
    top = umax_xor(umax_xor(umax_xor(umax_xor(top, 1), 2), 4), 8);
    const unsigned sb = scale_byte(top);
    const float inv = inv_scale(sb);
    if (c < M) {  // M % 16 == 0: the 8 columns are valid together
        *reinterpret_cast<uint2 *>(qrow + c) = make_uint2(pack_fp8x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                                                          pack_fp8x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
        if ((c & (QB - 1)) == 0) srow[c / QB] = (u8)sb;
    }
}

template <int DT, int TW, int NCH, bool VEC>
__global__ __launch_bounds__(TW == 1 ? 256 : 64 * TW) void add_rms_norm_kernel(const NormParams p) {
    __shared__ float red[2 * 16];
    constexpr int TPB = TW == 1 ? 4 : 1;
    const int t = TW == 1 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
    const int team = TW == 1 ? (int)(threadIdx.x >> 6) : 0;
    float w[NCH][8];
    bool have_w = false;
    int it = 0;
    for (long long row = (long long)blockIdx.x * TPB + team; row < p.S; row += (long long)gridDim.x * TPB, it ^= 1) {
        float f[NCH][8];
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < NCH; ++i) load8<DT, VEC>(p.x + row * p.ldx, (i * TW * 64 + t) * 8, p.M, f[i]);
        if (p.res) {
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                float r[8];
                load8<DT, VEC>(p.res + row * p.ldr, (i * TW * 64 + t) * 8, p.M, r);
#pragma unroll
                for (int j = 0; j < 8; ++j) f[i][j] = Elt<DT>::round(f[i][j] + r[j]);
            }
        }
        if (!have_w) {  // the weight stays in registers over the rows of a team
#pragma unroll
            for (int i = 0; i < NCH; ++i) load_w8<DT>(p.w, p.w_f32, (i * TW * 64 + t) * 8, p.M, w[i]);
            have_w = true;
        }
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            if (p.sum) store8<DT, VEC>(p.sum + row * p.lds, (i * TW * 64 + t) * 8, p.M, f[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = fmaf(f[i][j], f[i][j], ss);
        }
        ss = team_sum<TW>(ss, red, it);
        const float rstd = 1.0f / sqrtf(ss / (float)p.M + p.eps);
        if (p.rstd && t == 0) p.rstd[row] = rstd;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = (i * TW * 64 + t) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) f[i][j] = f[i][j] * rstd * w[i][j];
            if (p.y) store8<DT, VEC>(p.y + row * p.ldy, c, p.M, f[i]);
            if (p.q) quant8(f[i], c, p.M, p.q + row * p.ldq, p.scale + row * p.ld_scale);
        }
    }
}

struct NormBwdParams {
    const bf16_t *dy, *ds, *sum;
    long long lddy, ldds, lds;
    const void *w;
    int w_f32;
    const float *rstd;
    int S, M;
    bf16_t *dx;
    long long lddx;
    float *part;   // [gridDim.x, M] partial weight gradients
};

// One row per block at a time: a row's gradient and norm, and the block's share of dw, are 32 registers a lane and chunk, so
// a wave per row would leave two waves per SIMD (22528 x 2048: 91 us; four waves per row 70 us = 5.3 TB/s with 1024 blocks, 96
// with 512, 76 with 2048).
template <int DT, int TW, int NCH, bool VEC>
__global__ __launch_bounds__(64 * TW) void add_rms_norm_bwd_kernel(const NormBwdParams p) {
    __shared__ float red[2 * TW];
    const int t = (int)threadIdx.x;
    float w[NCH][8], dw[NCH][8];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        load_w8<DT>(p.w, p.w_f32, (i * TW * 64 + t) * 8, p.M, w[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) dw[i][j] = 0.f;
    }
    int it = 0;
    for (long long row = blockIdx.x; row < p.S; row += gridDim.x, it ^= 1) {
        float n[NCH][8], g[NCH][8];
        const float rstd = p.rstd[row];
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = (i * TW * 64 + t) * 8;
            load8<DT, VEC>(p.sum + row * p.lds, c, p.M, n[i]);
            if (p.dy) {
                load8<DT, VEC>(p.dy + row * p.lddy, c, p.M, g[i]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) g[i][j] = 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                n[i][j] *= rstd;
                dw[i][j] = fmaf(g[i][j], n[i][j], dw[i][j]);
                g[i][j] *= w[i][j];
                dot = fmaf(g[i][j], n[i][j], dot);
            }
        dot = team_sum<TW>(dot, red, it) / (float)p.M;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = (i * TW * 64 + t) * 8;
            float d[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) d[j] = rstd * (g[i][j] - n[i][j] * dot);
            if (p.ds) {
                float e[8];
                load8<DT, VEC>(p.ds + row * p.ldds, c, p.M, e);
#pragma unroll
                for (int j = 0; j < 8; ++j) d[j] += e[j];
            }
            store8<DT, VEC>(p.dx + row * p.lddx, c, p.M, d);
        }
    }
    // one partial row per block (row stride a multiple of 4): no atomics, the same sums every time
    float *out = p.part + (long long)blockIdx.x * ((p.M + 3) & ~3);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int c = (i * TW * 64 + t) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c + j < p.M) out[c + j] = dw[i][j];
    }
}

// dw[m] = sum over the partial rows in a fixed order: 32 columns per block, 4 a thread, 128 row groups joined in LDS
template <int DT>
__global__ __launch_bounds__(1024) void norm_dw_reduce_kernel(const float *part, int P, int M, void *dw, int w_f32) {
    __shared__ f32x4_t red[128][8];
    const int cx = threadIdx.x & 7, ry = threadIdx.x >> 3;
    const int c = blockIdx.x * 32 + cx * 4;
    const long long ld = (M + 3) & ~3;
    f32x4_t a = {0.f, 0.f, 0.f, 0.f};
    if (c < M)
        for (int r = ry; r < P; r += 128) a += *reinterpret_cast<const f32x4_t *>(part + r * ld + c);
    red[ry][cx] = a;
#pragma unroll
    for (int k = 64; k > 0; k >>= 1) {
        __syncthreads();
        if (ry < k) {
            a += red[ry + k][cx];
            red[ry][cx] = a;
        }
    }
    if (ry == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j < M) {
                if (w_f32) ((float *)dw)[c + j] = a[j];
                else ((bf16_t *)dw)[c + j] = Elt<DT>::from_f(a[j]);
            }
    }
}

// rows of 16 bits -> e4m3 + scales; 16 lanes per block of 128 columns
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const bf16_t *x, long long ldx, int S, int M, u8 *q, long long ldq,
                                                            u8 *scale, long long ld_scale) {
    const int kb = (M + QB - 1) / QB;
    const long long n = (long long)S * kb;
    const int l16 = threadIdx.x & 15;
    const long long i = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
    const bool ok = i < n;
    const long long row = ok ? i / kb : 0;
    const int c = ok ? (int)(i - row * kb) * QB + l16 * 8 : M;
    float f[8];
    load8<DT, VEC>(x + row * ldx, c, M, f);
    quant8(f, c, M, q + row * ldq, scale + row * ld_scale);
}

// weights [batch, n, k] in 16 bits -> e4m3 + one scale per 128 x 128; one block of threads per block of the grid
template <int DT>
__global__ __launch_bounds__(256) void quantize_blocks_kernel(const bf16_t *w, int n, int k, u8 *q, u8 *scale) {
    __shared__ unsigned red[4];
    const int nb = (n + QB - 1) / QB, kb = (k + QB - 1) / QB;
    const int bk = blockIdx.x % kb;
    const int bn = (blockIdx.x / kb) % nb;
    const long long b = blockIdx.x / kb / nb;
    const long long base = b * n * (long long)k;
    const int l16 = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    const int c = bk * QB + l16 * 8;
    const int rows = min(QB, n - bn * QB);
    uint4 v[8];
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = i * 16 + r0;
        v[i] = make_uint4(0, 0, 0, 0);
        if (r < rows && c < k) v[i] = *reinterpret_cast<const uint4 *>(w + base + (long long)(bn * QB + r) * k + c);
        float f[8];
        unpack8_t<DT>(v[i], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const unsigned u = abs_bits(f[j]);
            top = u > top ? u : top;
        }
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) top = umax_xor(top, m);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(red[0], red[1]), max(red[2], red[3]));
    const unsigned sb = scale_byte(top);
    const float inv = inv_scale(sb);
    if (threadIdx.x == 0) scale[(b * nb + bn) * kb + bk] = (u8)sb;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = i * 16 + r0;
        if (r < rows && c < k) {
            float f[8];
            unpack8_t<DT>(v[i], f);
            *reinterpret_cast<uint2 *>(q + base + (long long)(bn * QB + r) * k + c) =
                make_uint2(pack_fp8x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                           pack_fp8x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
        }
    }
}

// e4m3 weights [batch, n, k] -> [batch, k, n] (a block of 128 x 128 keeps its scale: only the grid of the scales is
// transposed with it).  64 x 64 bytes per block of threads: 16-byte loads, bytes re-assembled from LDS, 16-byte stores.
__global__ __launch_bounds__(256) void transpose_fp8_kernel(const u8 *w, const u8 *scale, int n, int k, u8 *wt, u8 *scale_t) {
    __shared__ __attribute__((aligned(16))) u8 t[64][64 + 16];
    const int tn = (n + 63) / 64, tk = (k + 63) / 64;
    const int bk = blockIdx.x % tk, bn = (blockIdx.x / tk) % tn;
    const long long b = blockIdx.x / tk / tn;
    const long long base = b * n * (long long)k;
    {
        const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;
        if (bn * 64 + r < n && bk * 64 + c < k)  // k % 16 == 0
            *reinterpret_cast<uint4 *>(&t[r][c]) = *reinterpret_cast<const uint4 *>(w + base + (long long)(bn * 64 + r) * k + bk * 64 + c);
    }
    __syncthreads();
    const int c = threadIdx.x >> 2, r = (threadIdx.x & 3) * 16;
    if (bk * 64 + c < k && bn * 64 + r < n) {    // n % 16 == 0
        unsigned o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            o[i] = (unsigned)t[r + 4 * i][c] | ((unsigned)t[r + 4 * i + 1][c] << 8) | ((unsigned)t[r + 4 * i + 2][c] << 16) |
                   ((unsigned)t[r + 4 * i + 3][c] << 24);
        *reinterpret_cast<uint4 *>(wt + base + (long long)(bk * 64 + c) * n + bn * 64 + r) = make_uint4(o[0], o[1], o[2], o[3]);
    }
    const int nb = (n + QB - 1) / QB, kb = (k + QB - 1) / QB;
    if (threadIdx.x == 0 && (bn & 1) == 0 && (bk & 1) == 0)
        scale_t[b * nb * kb + (long long)(bk / 2) * nb + bn / 2] = scale[b * nb * kb + (long long)(bn / 2) * kb + bk / 2];
}

// waves per row and 8-element chunks per lane.  One wave per row needs >= 4096 rows to fill the chip (256 CUs x 16 waves);
// below that four waves per row halve the latency of a launch (S = 1, M = 2048: one chunk per lane).
struct NormShape { int tw, nch; };
static NormShape norm_shape(int S, int M) {
    const int chunks = (M + 7) / 8;
    auto up = [](int v) { return v <= 1 ? 1 : v <= 2 ? 2 : v <= 4 ? 4 : v <= 5 ? 5 : 8; };
    if (S >= 4096 && chunks <= 64 * 8) return {1, up((chunks + 63) / 64)};
    if (chunks <= 256 * 8) return {4, up((chunks + 255) / 256)};
    return {16, 8};
}
#define NORM_SHAPES(CALL)                                                        \
    if (sh.tw == 1) {                                                            \
        switch (sh.nch) { case 1: CALL(1, 1); break; case 2: CALL(1, 2); break;  \
                          case 4: CALL(1, 4); break; case 5: CALL(1, 5); break; default: CALL(1, 8); } \
    } else NORM_ROW_SHAPES(CALL)
#define NORM_ROW_SHAPES(CALL)                                                    \
    if (sh.tw == 4) {                                                            \
        switch (sh.nch) { case 1: CALL(4, 1); break; case 2: CALL(4, 2); break;  \
                          case 4: CALL(4, 4); break; case 5: CALL(4, 5); break; default: CALL(4, 8); } \
    } else { CALL(16, 8); }

constexpr int NORM_MAX_M = 16 * 64 * 8 * 8;
static int norm_blocks(int S, const NormShape &sh, int most) {
    const int need = sh.tw == 1 ? (S + 3) / 4 : S;
    return need < most ? need : most;
}
static NormShape norm_bwd_shape(int M) { return norm_shape(1, M); }  // never one wave per row
static int norm_bwd_blocks(int S) { return S < 1024 ? S : 1024; }

}  // namespace moe

using namespace moe;

static bool even2(const void *q) { return (reinterpret_cast<uintptr_t>(q) & 1) == 0; }

extern "C" int moe_add_rms_norm_fwd(const void *x, int64_t ldx, const void *residual, int64_t ldr, const void *weight,
                                    int w_dtype, float eps, int S, int M, void *y, int64_t ldy, void *sum, int64_t lds,
                                    float *rstd, void *q, int64_t ldq, void *scale, int64_t ld_scale, int dtype, void *stream) {
    const char *fn = "moe_add_rms_norm_fwd";
    if (!x || !weight || (!y && !q)) return fail(MOE_ERR_ARG, "%s: null pointer", fn);
    if (dtype != MOE_DTYPE_BF16 && dtype != MOE_DTYPE_F16) return fail(MOE_ERR_ARG, "%s: unknown dtype %d", fn, dtype);
    if (w_dtype != MOE_WG_F32 && w_dtype != (dtype == MOE_DTYPE_BF16 ? MOE_WG_BF16 : MOE_WG_F16))
        return fail(MOE_ERR_ARG, "%s: weight type %d: need fp32 or the rows' type", fn, w_dtype);
    if ((!q) != (!scale)) return fail(MOE_ERR_ARG, "%s: q and scale go together", fn);
    if (residual && !sum) return fail(MOE_ERR_ARG, "%s: a residual needs the sum's output", fn);
    if (S < 0 || S > DIM_MAX || M < 1 || M > NORM_MAX_M)
        return fail(MOE_ERR_SHAPE, "%s: need 0 <= S <= %d, 1 <= M <= %d (S=%d M=%d)", fn, DIM_MAX, NORM_MAX_M, S, M);
    if (S > 1 && (ldx < M || (residual && ldr < M) || (y && ldy < M) || (sum && lds < M)))
        return fail(MOE_ERR_SHAPE, "%s: row strides must be >= M", fn);
    if (q && ((M & 15) || (ldq & 7) || ldq < M || ld_scale < (M + QB - 1) / QB))
        return fail(MOE_ERR_SHAPE, "%s: 8-bit output needs M %% 16 == 0, ldq >= M and %% 8 == 0, ld_scale >= ceil(M/128)", fn);
    if (q && (reinterpret_cast<uintptr_t>(q) & 7)) return fail(MOE_ERR_ALIGN, "%s: q must be 8-byte aligned", fn);
    if (!even2(x) || !even2(residual) || !even2(y) || !even2(sum) || !even2(weight) ||
        (w_dtype == MOE_WG_F32 && (reinterpret_cast<uintptr_t>(weight) & 3)))
        return fail(MOE_ERR_ALIGN, "%s: pointers must be aligned to their elements", fn);
    if (S == 0) return 0;
    NormParams p{(const bf16_t *)x, (const bf16_t *)residual, ldx, ldr, weight, w_dtype == MOE_WG_F32, eps, S, M,
                 (bf16_t *)y, (bf16_t *)sum, ldy, lds, rstd, (u8 *)q, (u8 *)scale, ldq, ld_scale};
    const bool vec = (M & 7) == 0 && aligned16(x) && (ldx & 7) == 0 && (!residual || (aligned16(residual) && (ldr & 7) == 0)) &&
                     (!y || (aligned16(y) && (ldy & 7) == 0)) && (!sum || (aligned16(sum) && (lds & 7) == 0));
    const NormShape sh = norm_shape(S, M);
    const dim3 g(norm_blocks(S, sh, 4096)), b(sh.tw == 1 ? 256 : 64 * sh.tw);
    hipStream_t st = (hipStream_t)stream;
#define NORM_CALL(TW_, NCH_)                                                                                       \
    do {                                                                                                           \
        if (dtype == MOE_DTYPE_F16) {                                                                              \
            if (vec) hipLaunchKernelGGL((add_rms_norm_kernel<DT_F16, TW_, NCH_, true>), g, b, 0, st, p);           \
            else hipLaunchKernelGGL((add_rms_norm_kernel<DT_F16, TW_, NCH_, false>), g, b, 0, st, p);              \
        } else {                                                                                                   \
            if (vec) hipLaunchKernelGGL((add_rms_norm_kernel<DT_BF16, TW_, NCH_, true>), g, b, 0, st, p);          \
            else hipLaunchKernelGGL((add_rms_norm_kernel<DT_BF16, TW_, NCH_, false>), g, b, 0, st, p);             \
        }                                                                                                          \
    } while (0)
    NORM_SHAPES(NORM_CALL)
#undef NORM_CALL
    return check_launch("add_rms_norm_kernel");
}

extern "C" size_t moe_add_rms_norm_bwd_workspace_bytes(int S, int M) {
    if (S < 1 || M < 1) return 0;
    return (size_t)norm_bwd_blocks(S) * ((M + 3) & ~3) * sizeof(float);
}

extern "C" int moe_add_rms_norm_bwd(const void *dy, int64_t lddy, const void *dsum, int64_t ldds, const void *sum, int64_t lds,
                                    const void *weight, int w_dtype, const float *rstd, int S, int M, void *dx, int64_t lddx,
                                    void *dweight, void *workspace, size_t ws_bytes, int dtype, void *stream) {
    const char *fn = "moe_add_rms_norm_bwd";
    if (!sum || !weight || !rstd || !dx || !dweight || !workspace) return fail(MOE_ERR_ARG, "%s: null pointer", fn);
    if (dtype != MOE_DTYPE_BF16 && dtype != MOE_DTYPE_F16) return fail(MOE_ERR_ARG, "%s: unknown dtype %d", fn, dtype);
    if (w_dtype != MOE_WG_F32 && w_dtype != (dtype == MOE_DTYPE_BF16 ? MOE_WG_BF16 : MOE_WG_F16))
        return fail(MOE_ERR_ARG, "%s: weight type %d: need fp32 or the rows' type", fn, w_dtype);
    if (S < 1 || S > DIM_MAX || M < 1 || M > NORM_MAX_M)
        return fail(MOE_ERR_SHAPE, "%s: need 1 <= S <= %d, 1 <= M <= %d (S=%d M=%d)", fn, DIM_MAX, NORM_MAX_M, S, M);
    if (S > 1 && ((dy && lddy < M) || (dsum && ldds < M) || lds < M || lddx < M)) return fail(MOE_ERR_SHAPE, "%s: row strides must be >= M", fn);
    if (!even2(dy) || !even2(dsum) || !even2(sum) || !even2(dx) || !even2(weight) || !even2(dweight) ||
        (w_dtype == MOE_WG_F32 && ((reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(dweight)) & 3)) ||
        (reinterpret_cast<uintptr_t>(workspace) & 15))
        return fail(MOE_ERR_ALIGN, "%s: pointers must be aligned to their elements", fn);
    if (ws_bytes < moe_add_rms_norm_bwd_workspace_bytes(S, M)) return fail(MOE_ERR_WORKSPACE, "%s: workspace too small", fn);
    NormBwdParams p{(const bf16_t *)dy, (const bf16_t *)dsum, (const bf16_t *)sum, lddy, ldds, lds, weight,
                    w_dtype == MOE_WG_F32, rstd, S, M, (bf16_t *)dx, lddx, (float *)workspace};
    const bool vec = (M & 7) == 0 && (!dy || (aligned16(dy) && (lddy & 7) == 0)) && (!dsum || (aligned16(dsum) && (ldds & 7) == 0)) &&
                     aligned16(sum) && (lds & 7) == 0 && aligned16(dx) && (lddx & 7) == 0;
    const NormShape sh = norm_bwd_shape(M);
    const int blocks = norm_bwd_blocks(S);
    const dim3 g(blocks), b(64 * sh.tw);
    hipStream_t st = (hipStream_t)stream;
#define NORM_CALL(TW_, NCH_)                                                                                       \
    do {                                                                                                           \
        if (dtype == MOE_DTYPE_F16) {                                                                              \
            if (vec) hipLaunchKernelGGL((add_rms_norm_bwd_kernel<DT_F16, TW_, NCH_, true>), g, b, 0, st, p);       \
            else hipLaunchKernelGGL((add_rms_norm_bwd_kernel<DT_F16, TW_, NCH_, false>), g, b, 0, st, p);          \
        } else {                                                                                                   \
            if (vec) hipLaunchKernelGGL((add_rms_norm_bwd_kernel<DT_BF16, TW_, NCH_, true>), g, b, 0, st, p);      \
            else hipLaunchKernelGGL((add_rms_norm_bwd_kernel<DT_BF16, TW_, NCH_, false>), g, b, 0, st, p);         \
        }                                                                                                          \
    } while (0)
    NORM_ROW_SHAPES(NORM_CALL)
#undef NORM_CALL
    int rc = check_launch("add_rms_norm_bwd_kernel");
    if (rc) return rc;
    const dim3 gr((M + 31) / 32);
    if (dtype == MOE_DTYPE_F16)
        hipLaunchKernelGGL((norm_dw_reduce_kernel<DT_F16>), gr, dim3(1024), 0, st, (const float *)workspace, blocks, M, dweight, p.w_f32);
    else
        hipLaunchKernelGGL((norm_dw_reduce_kernel<DT_BF16>), gr, dim3(1024), 0, st, (const float *)workspace, blocks, M, dweight, p.w_f32);
    return check_launch("norm_dw_reduce_kernel");
}

extern "C" int moe_quantize_rows_fp8(const void *x, int64_t ldx, int S, int M, void *q, int64_t ldq, void *scale,
                                     int64_t ld_scale, int dtype, void *stream) {
    const char *fn = "moe_quantize_rows_fp8";
    if (!x || !q || !scale) return fail(MOE_ERR_ARG, "%s: null pointer", fn);
    if (dtype != MOE_DTYPE_BF16 && dtype != MOE_DTYPE_F16) return fail(MOE_ERR_ARG, "%s: unknown dtype %d", fn, dtype);
    if (S < 0 || M < 16 || (M & 15)) return fail(MOE_ERR_SHAPE, "%s: need S >= 0, M >= 16, M %% 16 == 0 (S=%d M=%d)", fn, S, M);
    if (S > DIM_MAX || M > DIM_MAX) return fail(MOE_ERR_SHAPE, "%s: S=%d, M=%d: at most %d", fn, S, M, DIM_MAX);
    if ((S > 1 && ldx < M) || ldq < M || (ldq & 7) || ld_scale < (M + QB - 1) / QB)
        return fail(MOE_ERR_SHAPE, "%s: row strides too small (or ldq %% 8 != 0)", fn);
    if (!even2(x) || (reinterpret_cast<uintptr_t>(q) & 7)) return fail(MOE_ERR_ALIGN, "%s: x must be 2-byte, q 8-byte aligned", fn);
    if (S == 0) return 0;
    const long long n = ((long long)S * ((M + QB - 1) / QB) + 15) / 16;
    if (!grid_fits(n, 256)) return fail(MOE_ERR_SHAPE, "%s: too many blocks", fn);
    const bool vec = aligned16(x) && (ldx & 7) == 0;
    const dim3 g((unsigned)n), b(256);
    hipStream_t st = (hipStream_t)stream;
#define QR(DT_, V_) hipLaunchKernelGGL((quantize_rows_kernel<DT_, V_>), g, b, 0, st, (const bf16_t *)x, (long long)ldx, S, M, (u8 *)q, (long long)ldq, (u8 *)scale, (long long)ld_scale)
    if (dtype == MOE_DTYPE_F16) { if (vec) QR(DT_F16, true); else QR(DT_F16, false); }
    else { if (vec) QR(DT_BF16, true); else QR(DT_BF16, false); }
#undef QR
    return check_launch("quantize_rows_kernel");
}

extern "C" int moe_quantize_blocks_fp8(const void *w, int batch, int n, int k, void *q, void *scale, int dtype, void *stream) {
    const char *fn = "moe_quantize_blocks_fp8";
    if (!w || !q || !scale) return fail(MOE_ERR_ARG, "%s: null pointer", fn);
    if (dtype != MOE_DTYPE_BF16 && dtype != MOE_DTYPE_F16) return fail(MOE_ERR_ARG, "%s: unknown dtype %d", fn, dtype);
    if (batch < 1 || n < 1 || k < 16 || (k & 15)) return fail(MOE_ERR_SHAPE, "%s: need batch >= 1, n >= 1, k %% 16 == 0 (%d, %d, %d)", fn, batch, n, k);
    if (n > DIM_MAX || k > DIM_MAX) return fail(MOE_ERR_SHAPE, "%s: n=%d, k=%d: at most %d", fn, n, k, DIM_MAX);
    if (!aligned16(w) || (reinterpret_cast<uintptr_t>(q) & 7)) return fail(MOE_ERR_ALIGN, "%s: w must be 16-byte, q 8-byte aligned", fn);
    const long long g = (long long)batch * ((n + QB - 1) / QB) * ((k + QB - 1) / QB);
    if (!grid_fits(g, 256)) return fail(MOE_ERR_SHAPE, "%s: too many blocks", fn);
    if (dtype == MOE_DTYPE_F16)
        hipLaunchKernelGGL((quantize_blocks_kernel<DT_F16>), dim3((unsigned)g), dim3(256), 0, (hipStream_t)stream, (const bf16_t *)w, n, k, (u8 *)q, (u8 *)scale);
    else
        hipLaunchKernelGGL((quantize_blocks_kernel<DT_BF16>), dim3((unsigned)g), dim3(256), 0, (hipStream_t)stream, (const bf16_t *)w, n, k, (u8 *)q, (u8 *)scale);
    return check_launch("quantize_blocks_kernel");
}

extern "C" int moe_transpose_blocks_fp8(const void *w, const void *scale, int batch, int n, int k, void *wt, void *scale_t,
                                        void *stream) {
    const char *fn = "moe_transpose_blocks_fp8";
    if (!w || !scale || !wt || !scale_t) return fail(MOE_ERR_ARG, "%s: null pointer", fn);
    if (batch < 1 || n < 16 || (n & 15) || k < 16 || (k & 15)) return fail(MOE_ERR_SHAPE, "%s: need n %% 16 == 0 and k %% 16 == 0 (%d, %d, %d)", fn, batch, n, k);
    if (n > DIM_MAX || k > DIM_MAX) return fail(MOE_ERR_SHAPE, "%s: n=%d, k=%d: at most %d", fn, n, k, DIM_MAX);
    if (!aligned16(w) || !aligned16(wt)) return fail(MOE_ERR_ALIGN, "%s: weights must be 16-byte aligned", fn);
    const long long g = (long long)batch * ((n + 63) / 64) * ((k + 63) / 64);
    if (!grid_fits(g, 256)) return fail(MOE_ERR_SHAPE, "%s: too many blocks", fn);
    hipLaunchKernelGGL(transpose_fp8_kernel, dim3((unsigned)g), dim3(256), 0, (hipStream_t)stream, (const u8 *)w, (const u8 *)scale, n, k, (u8 *)wt, (u8 *)scale_t);
    return check_launch("transpose_fp8_kernel");
}
