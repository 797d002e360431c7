// Products of few rows on 8-bit weights for gfx950 (decode steps: at most FP8_FEW_ROWS rows in all): weight streaming.
//
// One block owns 16 * NW output columns of one group (gated: their 'a' and 'b' weight rows) and splits K over its waves in
// blocks of 128 columns; weights go global -> registers (two 16-byte loads per lane and fragment: lane (fr, fq) holds the
// chunks fq and fq + 4 of weight row fr), never through LDS; v_mfma_scale_f32_16x16x128_f8f6f4 takes the block's exponent
// bytes; the waves' partial sums meet in LDS in wave order.  Rows are 8-bit rows, or 16-bit rows that are quantised on load:
// the four lanes that hold a row's block of 128 columns agree on its maximum by two shuffles, the same bits as
// moe_quantize_rows_fp8 would give.
// A first product leaves its activation in fp32 (a block of the quantisation spans eight of these blocks); a small launch
// behind quantises it for the second product.
// Bound: HBM, the weights of the groups that hold rows, read once.
#include "moe_fp8.h"

namespace moe {

#ifndef FEW_FRAGS
#define FEW_FRAGS 8
#endif
#ifndef FEW_KS
#define FEW_KS 8
#endif
template <int N>
struct FewInt { static constexpr int value = N; };

template <int DT, int EPI, int NW, bool X16>
struct FewCfg {
    static constexpr bool GATED = EPI == EPI_SWIGLU;
    static constexpr int NACC = GATED ? 2 : 1;
    static constexpr int COLS = 16 * NW;
    static constexpr int U = FEW_FRAGS / (NACC * NW) > 1 ? FEW_FRAGS / (NACC * NW) : 1;
};

template <int DT, int EPI, int NW, bool X16, int RT>
__device__ __forceinline__ void few_body(const Fp8GemmParams &p, int expert, int row_begin, int n_rows, int ctile, float *red) {
    using C = FewCfg<DT, EPI, NW, X16>;
    typedef Elt<DT> E;
    constexpr int NACC = C::NACC, U = C::U;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ks = blockDim.x >> 6;
    const int fr = lane & 15, fq = lane >> 4;
    const int nk = (p.K + QB - 1) / QB;
    const u8 *wr[NACC][NW];
#pragma unroll
    for (int h = 0; h < NACC; ++h)
#pragma unroll
        for (int g = 0; g < NW; ++g) {
            const int c = min(ctile * C::COLS + g * 16 + fr, p.N_out - 1) + h * p.b_row_offset;
            wr[h][g] = p.w + (long long)expert * p.w_expert_stride + (long long)c * p.K;
        }
    const u8 *xr[RT], *xs[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int prow = row_begin + min(t * 16 + fr, n_rows - 1);  // rows behind the last repeat it and are not stored
        const long long srow = p.gather ? (long long)(p.gather[prow] >> p.gather_shift) : (long long)prow;
        if (X16) {
            xr[t] = reinterpret_cast<const u8 *>(p.x16 + srow * p.ldx);
            xs[t] = nullptr;
        } else {
            xr[t] = p.a + srow * p.lda;
            xs[t] = p.a_scale + srow * p.ld_as;
        }
    }
    const int wblk = min(ctile * C::COLS, p.N_out - 1) / QB;  // COLS divides 128: one block of the weights' scales
    const u8 *wsb = p.w_scale + (long long)expert * p.ws_expert_stride + (long long)wblk * nk;
    f32x4_t acc[NACC][NW][RT];
#pragma unroll
    for (int h = 0; h < NACC; ++h)
#pragma unroll
        for (int g = 0; g < NW; ++g)
#pragma unroll
            for (int t = 0; t < RT; ++t) acc[h][g][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    // columns behind K (last block): the address is clamped into the row and the rows' side is zeroed
    auto ldw = [&](const u8 *row, int kb, bool last) {
        int o0 = kb * QB + fq * 16, o1 = o0 + 64;
        if (last) { o0 = min(o0, p.K - 16); o1 = min(o1, p.K - 16); }
        const v4i_t lo = *reinterpret_cast<const v4i_t *>(row + o0), hi = *reinterpret_cast<const v4i_t *>(row + o1);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    struct X { v8i_t q; int s; };
    auto ldx = [&](int t, int kb, bool last) {
        X r;
        int o0 = kb * QB + fq * 16, o1 = o0 + 64;
        const bool ok0 = !last || o0 < p.K, ok1 = !last || o1 < p.K;
        if (last) { o0 = min(o0, p.K - 16); o1 = min(o1, p.K - 16); }
        if constexpr (X16) {
            const uint4 *s0 = reinterpret_cast<const uint4 *>(xr[t] + 2 * o0), *s1 = reinterpret_cast<const uint4 *>(xr[t] + 2 * o1);
            const uint4 z = make_uint4(0, 0, 0, 0);
            const uint4 v[4] = {ok0 ? s0[0] : z, ok0 ? s0[1] : z, ok1 ? s1[0] : z, ok1 ? s1[1] : z};
            float f[32];
            unsigned top = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) unpack8_t<DT>(v[i], f + 8 * i);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const unsigned u = abs_bits(f[i]);
                top = u > top ? u : top;
            }
            top = umax_xor(umax_xor(top, 16), 32);
            r.s = (int)scale_byte(top);
            const float inv = inv_scale((unsigned)r.s);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                r.q[i] = (int)pack_fp8x4(f[4 * i] * inv, f[4 * i + 1] * inv, f[4 * i + 2] * inv, f[4 * i + 3] * inv);
        } else {
            const v4i_t z = {0, 0, 0, 0};
            v4i_t lo = *reinterpret_cast<const v4i_t *>(xr[t] + o0), hi = *reinterpret_cast<const v4i_t *>(xr[t] + o1);
            if (!ok0) lo = z;
            if (!ok1) hi = z;
            r.q = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            r.s = (int)xs[t][kb];
        }
        return r;
    };

    // this wave's blocks of K: [k_lo, k_hi), its exponent bytes 64 at a time in one register per projection
    const int k_lo = (int)((long long)wave * nk / ks), k_hi = (int)((long long)(wave + 1) * nk / ks);
    const bool has_tail = (p.K & (QB - 1)) != 0;
    for (int k0 = k_lo; k0 < k_hi; k0 += 64) {
        const int k1 = min(k0 + 64, k_hi);
        const int mine = min(k0 + lane, nk - 1);
        int wsc[NACC];
#pragma unroll
        for (int h = 0; h < NACC; ++h) wsc[h] = (int)wsb[(long long)h * p.b_blk_offset * nk + mine];
        auto steps = [&](auto u_c, int kb, bool last) {
            constexpr int UU = decltype(u_c)::value;
            v8i_t fw[UU][NACC][NW];
            X fx[UU][RT];
#pragma unroll
            for (int u = 0; u < UU; ++u)
#pragma unroll
                for (int h = 0; h < NACC; ++h)
#pragma unroll
                    for (int g = 0; g < NW; ++g) fw[u][h][g] = ldw(wr[h][g], kb + u, last);
#pragma unroll
            for (int u = 0; u < UU; ++u)
#pragma unroll
                for (int t = 0; t < RT; ++t) fx[u][t] = ldx(t, kb + u, last);
#pragma unroll
            for (int u = 0; u < UU; ++u) {
#pragma unroll
                for (int h = 0; h < NACC; ++h) {
                    const int ws = __builtin_amdgcn_readlane(wsc[h], kb + u - k0);
#pragma unroll
                    for (int g = 0; g < NW; ++g)
#pragma unroll
                        for (int t = 0; t < RT; ++t)
                            acc[h][g][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[u][h][g], fx[u][t].q, acc[h][g][t],
                                                                                           0, 0, 0, ws, 0, fx[u][t].s);
                }
            }
        };
        const int full = (has_tail && k1 == nk) ? k1 - 1 : k1;
        int kb = k0;
        for (; kb + U <= full; kb += U) steps(FewInt<U>{}, kb, false);
        for (; kb < full; ++kb) steps(FewInt<1>{}, kb, false);
        if (kb < k1) steps(FewInt<1>{}, kb, true);
    }

    const bf16_t *bias = p.bias ? p.bias + (long long)expert * p.bias_expert_stride : nullptr;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        __syncthreads();  // the previous row tile's partial sums have been read
#pragma unroll
        for (int h = 0; h < NACC; ++h)
#pragma unroll
            for (int g = 0; g < NW; ++g)
                *reinterpret_cast<f32x4_t *>(red + (((wave * NACC + h) * NW + g) * 64 + lane) * 4) = acc[h][g][t];
        __syncthreads();
        for (int g = wave; g < NW; g += ks) {  // one wave per column group adds the partial sums, in wave order
            f32x4_t a = {0.f, 0.f, 0.f, 0.f}, b = {0.f, 0.f, 0.f, 0.f};
            for (int w = 0; w < ks; ++w) {
                a += *reinterpret_cast<const f32x4_t *>(red + (((w * NACC) * NW + g) * 64 + lane) * 4);
                if (C::GATED) b += *reinterpret_cast<const f32x4_t *>(red + (((w * NACC + NACC - 1) * NW + g) * 64 + lane) * 4);
            }
            const int r = t * 16 + fr;
            const int c0 = ctile * C::COLS + g * 16 + fq * 4;
            if (r < n_rows) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int c = c0 + j;
                    if (c < p.N_out) {
                        const float v = a[j] + (bias ? E::to_f(bias[c]) : 0.f);
                        const long long row = row_begin + r;
                        if constexpr (EPI == EPI_PLAIN) {
                            ((bf16_t *)p.out)[row * p.ldo + c] = E::from_f(v);
                        } else if constexpr (C::GATED) {
                            const float vb = b[j] + (bias ? E::to_f(bias[p.b_row_offset + c]) : 0.f);
                            p.h32[row * p.N_out + c] = (c < p.n_gated ? fast_silu(v) : 1.0f) * vb;
                        } else {
                            p.h32[row * p.N_out + c] = gelu_new_f32(v);
                        }
                    }
                }
            }
        }
    }
}

template <int DT, int EPI, int NW, bool X16>
__global__ __launch_bounds__(512) void fp8_few_kernel(const Fp8GemmParams p) {
    using C = FewCfg<DT, EPI, NW, X16>;
    __shared__ __attribute__((aligned(16))) float red[8 * C::NACC * NW * 256];  // 1 KiB per wave and fragment
    const int ctile = blockIdx.x % p.col_tiles, grp = blockIdx.x / p.col_tiles;
    int b = 0, e = p.max_rows;
    if (p.group_offsets) {
        b = p.group_offsets[grp];
        e = p.group_offsets[grp + 1];
    }
    const int n = e - b;
    if (n <= 0) return;  // a group without rows: its weights are not read
    const int expert = grp % p.n_experts;
    switch ((min(n, FP8_FEW_ROWS) + 15) >> 4) {
        case 1: few_body<DT, EPI, NW, X16, 1>(p, expert, b, min(n, 16), ctile, red); break;
        case 2: few_body<DT, EPI, NW, X16, 2>(p, expert, b, min(n, 32), ctile, red); break;
        case 3: few_body<DT, EPI, NW, X16, 3>(p, expert, b, min(n, 48), ctile, red); break;
        default: few_body<DT, EPI, NW, X16, 4>(p, expert, b, min(n, 64), ctile, red); break;
    }
}

// fp32 activations of few rows -> e4m3 + scales; 16 lanes per block of 128 columns
__global__ __launch_bounds__(256) void quantize_f32_kernel(const float *h, int rows, int I, u8 *q, u8 *scale, long long ld_scale) {
    const int kb = (I + QB - 1) / QB;
    const int i = blockIdx.x * 16 + (threadIdx.x >> 4);
    const bool ok = i < rows * kb;
    const int row = ok ? i / kb : 0;
    const int c = ok ? (i - row * kb) * QB + (threadIdx.x & 15) * 8 : I;
    f32x4_t f[2] = {f32x4_t{0.f, 0.f, 0.f, 0.f}, f32x4_t{0.f, 0.f, 0.f, 0.f}};
    if (c < I) {  // I % 16 == 0
        f[0] = *reinterpret_cast<const f32x4_t *>(h + (long long)row * I + c);
        f[1] = *reinterpret_cast<const f32x4_t *>(h + (long long)row * I + c + 4);
    }
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const unsigned u = abs_bits(f[j >> 2][j & 3]);
        top = u > top ? u : top;
    }
    top = umax_xor(umax_xor(umax_xor(umax_xor(top, 1), 2), 4), 8);
    const unsigned sb = scale_byte(top);
    const float inv = inv_scale(sb);
    if (c < I) {
        *reinterpret_cast<uint2 *>(q + (long long)row * I + c) =
            make_uint2(pack_fp8x4(f[0][0] * inv, f[0][1] * inv, f[0][2] * inv, f[0][3] * inv),
                       pack_fp8x4(f[1][0] * inv, f[1][1] * inv, f[1][2] * inv, f[1][3] * inv));
        if ((c & (QB - 1)) == 0) scale[(long long)row * ld_scale + c / QB] = (u8)sb;
    }
}

int launch_quantize_f32(const float *h, int rows, int I, u8 *q, u8 *scale, long long ld_scale, hipStream_t st) {
    const int n = (rows * ((I + QB - 1) / QB) + 15) / 16;
    hipLaunchKernelGGL(quantize_f32_kernel, dim3(n), dim3(256), 0, st, h, rows, I, q, scale, ld_scale);
    return check_launch("quantize_f32_kernel");
}

int launch_fp8_few(const Fp8GemmParams &p0, int epilogue, hipStream_t st) {
    Fp8GemmParams p = p0;
    const bool gated = epilogue == MOE_EPI_SWIGLU;
    const long long active = p.G < p.max_rows ? p.G : p.max_rows;  // groups that can hold rows
    // column groups per block: 2 share a row fragment, as long as the launch keeps a block for every CU
    const int nw = active * ((p.N_out + 31) / 32) >= 256 ? 2 : 1;
    p.col_tiles = (p.N_out + 16 * nw - 1) / (16 * nw);
    const long long grid = (long long)p.G * p.col_tiles;
    if (grid > 0x7fffffffLL) return fail(MOE_ERR_SHAPE, "fp8 product: grid too large");
    // waves per block: about 16 wave-tasks per CU, at least one block of K each
    const int nk = (p.K + QB - 1) / QB;
    int ks = FEW_KS;
    while (ks > 1 && (active * p.col_tiles * ks > 4096 || ks > nk)) ks >>= 1;
    const dim3 g((unsigned)grid), b(64 * ks);
#define FEW(E_, N_, X_)                                                                                        \
    do {                                                                                                       \
        if (p.dtype == DT_F16) hipLaunchKernelGGL((fp8_few_kernel<DT_F16, E_, N_, X_>), g, b, 0, st, p);        \
        else hipLaunchKernelGGL((fp8_few_kernel<DT_BF16, E_, N_, X_>), g, b, 0, st, p);                         \
    } while (0)
#define FEW_N(E_, X_) do { if (nw == 2) FEW(E_, 2, X_); else FEW(E_, 1, X_); } while (0)
    if (gated) { if (p.x16) FEW_N(EPI_SWIGLU, true); else FEW_N(EPI_SWIGLU, false); }
    else if (epilogue == MOE_EPI_GELU_NEW) { if (p.x16) FEW_N(EPI_GELU_NEW, true); else FEW_N(EPI_GELU_NEW, false); }
    else { if (p.x16) FEW_N(EPI_PLAIN, true); else FEW_N(EPI_PLAIN, false); }
#undef FEW_N
#undef FEW
    return check_launch("fp8_few_kernel");
}

}  // namespace moe
