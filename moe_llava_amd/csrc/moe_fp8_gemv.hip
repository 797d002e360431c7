// Products of few rows on 8-bit weights for gfx950 (the second product of a decode step's experts, single projections):
// weight streaming.
//
// One block owns 16 * NW output columns of one group and splits K over its waves in blocks of 128 columns; weights go
// global -> registers (two 16-byte loads per lane and fragment: lane (fr, fq) holds the chunks fq and fq + 4 of weight row
// fr), never through LDS; v_mfma_scale_f32_16x16x128_f8f6f4 takes the block's exponent bytes; the waves' partial sums meet
// in LDS and are added in wave order.
// Bound: HBM, the weights of the groups that hold rows, read once per 32 rows of a group.  Measured (StableLM width, second
// product, K 5632, N 2048): two active experts 6.9 us = 3.3 TB/s, all four 14.1 us = 3.3 TB/s, of which 3 us are the launch,
// the first misses and the join of the waves; the copy rate is 5.1 TB/s.
//
// Only the plain epilogue exists here.  The first product of an expert MLP stays on the 32-row tiles (moe_fp8.hip) whatever
// its rows: its output is quantised over 128 columns, which eight of these blocks share, and leaving it in fp32 for a
// launch that quantises it cost more than the narrower blocks gained (StableLM width, one token, two active experts: 15.6 +
// 4.5 us against 14; 32 tokens 25 + 4.7 against 20).  Rows come quantised: quantising 16-bit rows on load in every block
// took 2.6 us more at one row of K 2048 and 10 at 64, the launch in front takes 2.3.
#include "moe_fp8.h"

namespace moe {

template <int N>
struct FewInt { static constexpr int value = N; };

template <int DT, int NW, int RT>
__device__ __forceinline__ void few_body(const Fp8GemmParams &p, int expert, int row_begin, int n_rows, int ctile, float *red) {
    typedef Elt<DT> E;
    // blocks of K in flight: 4 weight fragments = 8 loads of 1 KiB per wave (8 and 16 fragments: the registers cost resident
    // waves, which are worth as much as loads in flight)
    constexpr int U = 4 / NW / RT < 1 ? 1 : 4 / NW / RT;
    constexpr int COLS = 16 * NW;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ks = blockDim.x >> 6;
    const int fr = lane & 15, fq = lane >> 4;
    const int nk = (p.K + QB - 1) / QB;
    const u8 *wr[NW];
#pragma unroll
    for (int g = 0; g < NW; ++g)
        wr[g] = p.w + (long long)expert * p.w_expert_stride + (long long)min(ctile * COLS + g * 16 + fr, p.N_out - 1) * p.K;
    const u8 *xr[RT], *xs[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int prow = row_begin + min(t * 16 + fr, n_rows - 1);  // rows behind the last repeat it and are not stored
        const long long srow = p.gather ? (long long)(p.gather[prow] >> p.gather_shift) : (long long)prow;
        xr[t] = p.a + srow * p.lda;
        xs[t] = p.a_scale + srow * p.ld_as;
    }
    // COLS divides 128: the tile lies in one block of the weights' scales
    const u8 *wsb = p.w_scale + (long long)expert * p.ws_expert_stride + (long long)(min(ctile * COLS, p.N_out - 1) / QB) * nk;
    f32x4_t acc[NW][RT];
#pragma unroll
    for (int g = 0; g < NW; ++g)
#pragma unroll
        for (int t = 0; t < RT; ++t) acc[g][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    // columns behind K (last block): the address is clamped into the row and the rows' side is zeroed
    auto ld32 = [&](const u8 *row, int kb, bool last) {
        int o0 = kb * QB + fq * 16, o1 = o0 + 64;
        if (last) { o0 = min(o0, p.K - 16); o1 = min(o1, p.K - 16); }
        const v4i_t lo = *reinterpret_cast<const v4i_t *>(row + o0), hi = *reinterpret_cast<const v4i_t *>(row + o1);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    const int k_lo = (int)((long long)wave * nk / ks), k_hi = (int)((long long)(wave + 1) * nk / ks);  // this wave's blocks of K
    const bool has_tail = (p.K & (QB - 1)) != 0;
    // the exponent bytes of 64 blocks of K sit in one register
    for (int k0 = k_lo; k0 < k_hi; k0 += 64) {
        const int k1 = min(k0 + 64, k_hi);
        const int wsc = (int)wsb[min(k0 + lane, nk - 1)];
        auto steps = [&](auto u_c, int kb, bool last) {
            constexpr int UU = decltype(u_c)::value;
            v8i_t fw[UU][NW], fx[UU][RT];
            int sx[UU][RT];
#pragma unroll
            for (int u = 0; u < UU; ++u) {
#pragma unroll
                for (int g = 0; g < NW; ++g) fw[u][g] = ld32(wr[g], kb + u, last);
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    fx[u][t] = ld32(xr[t], kb + u, last);
                    sx[u][t] = (int)xs[t][kb + u];
                }
            }
            __builtin_amdgcn_sched_barrier(0);  // every load is out before the first is used
#pragma unroll
            for (int u = 0; u < UU; ++u) {
                if (last) {
                    const int o0 = kb * QB + fq * 16;
#pragma unroll
                    for (int t = 0; t < RT; ++t)
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (o0 + (i >> 2) * 64 >= p.K) fx[u][t][i] = 0;
                }
                const int ws = __builtin_amdgcn_readlane(wsc, kb + u - k0);
#pragma unroll
                for (int g = 0; g < NW; ++g)
#pragma unroll
                    for (int t = 0; t < RT; ++t)
                        acc[g][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[u][g], fx[u][t], acc[g][t], 0, 0, 0, ws, 0,
                                                                                    sx[u][t]);
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
        for (int g = 0; g < NW; ++g) *reinterpret_cast<f32x4_t *>(red + ((wave * NW + g) * 64 + lane) * 4) = acc[g][t];
        __syncthreads();
        for (int g = wave; g < NW; g += ks) {  // one wave per column group adds the partial sums, in wave order
            f32x4_t a = {0.f, 0.f, 0.f, 0.f};
            for (int w = 0; w < ks; ++w) a += *reinterpret_cast<const f32x4_t *>(red + ((w * NW + g) * 64 + lane) * 4);
            const int r = t * 16 + fr;
            const int c0 = ctile * COLS + g * 16 + fq * 4;
            if (r < n_rows) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c0 + j < p.N_out)
                        ((bf16_t *)p.out)[(long long)(row_begin + r) * p.ldo + c0 + j] =
                            E::from_f(a[j] + (bias ? E::to_f(bias[c0 + j]) : 0.f));
            }
        }
    }
}

template <int DT, int NW>
__global__ __launch_bounds__(512) void fp8_few_kernel(const Fp8GemmParams p) {
    __shared__ __attribute__((aligned(16))) float red[8 * NW * 256];  // 1 KiB per wave and fragment
    const int ctile = blockIdx.x % p.col_tiles, grp = blockIdx.x / p.col_tiles;
    int b = 0, e = p.max_rows;
    if (p.group_offsets) {
        b = p.group_offsets[grp];
        e = p.group_offsets[grp + 1];
    }
    const int n = e - b;  // a group without rows: its weights are not read
    const int expert = grp % p.n_experts;
    for (int r = 0; r < n; r += 32) {  // more than 32 rows of a group: its weights a second time, from the caches
        if (n - r <= 16) few_body<DT, NW, 1>(p, expert, b + r, n - r, ctile, red);
        else few_body<DT, NW, 2>(p, expert, b + r, min(n - r, 32), ctile, red);
    }
}

int launch_fp8_few(const Fp8GemmParams &p0, hipStream_t st) {
    Fp8GemmParams p = p0;
    const long long active = p.G < p.max_rows ? p.G : p.max_rows;  // groups that can hold rows
    // column groups per block: 2 share a row fragment, as long as the launch keeps a block for every CU
    const int nw = active * ((p.N_out + 31) / 32) >= 256 ? 2 : 1;
    p.col_tiles = (p.N_out + 16 * nw - 1) / (16 * nw);
    const long long grid = (long long)p.G * p.col_tiles;
    if (!grid_fits(grid, 512)) return fail(MOE_ERR_SHAPE, "fp8 product: grid too large");
    // waves per block: about 16 wave-tasks per CU, at least one block of K each
    const int nk = (p.K + QB - 1) / QB;
    int ks = 8;
    while (ks > 1 && (active * p.col_tiles * ks > 4096 || ks > nk)) ks >>= 1;
    const dim3 g((unsigned)grid), b(64 * ks);
    if (p.dtype == DT_F16) {
        if (nw == 2) hipLaunchKernelGGL((fp8_few_kernel<DT_F16, 2>), g, b, 0, st, p);
        else hipLaunchKernelGGL((fp8_few_kernel<DT_F16, 1>), g, b, 0, st, p);
    } else {
        if (nw == 2) hipLaunchKernelGGL((fp8_few_kernel<DT_BF16, 2>), g, b, 0, st, p);
        else hipLaunchKernelGGL((fp8_few_kernel<DT_BF16, 1>), g, b, 0, st, p);
    }
    return check_launch("fp8_few_kernel");
}

}  // namespace moe
