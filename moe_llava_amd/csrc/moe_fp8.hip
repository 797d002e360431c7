// Grouped, variable-length matrix products in 8 bits on MFMA for gfx950: e4m3 operands with a power-of-two scale for every
// 1 x 128 block of the rows and every 128 x 128 block of the weights (moe_fp8.h).
//
//   out[r, n] = sum_b 2^(ea[r, b] + ew[n / 128, b]) * sum_{k in block b} qa[r, k] * qw[n, k]   (+ bias)     fp32 accumulation
//
// plain (16-bit output), or as the first product of an expert MLP: SwiGLU / gelu_new in fp32 on the accumulators, and the
// result quantised again for the second product (the activation never leaves the kernel in more than 8 bits).
//
// Tile BM (rows) x BNW (weight rows) x 128 (K) per 512-thread block, 8 waves as 2 (rows) x 4 (weight rows).  One ring slot
// is one K slice = one block of the scales, so v_mfma_scale_f32_16x16x128_f8f6f4 takes the two exponent bytes of the slice
// as operands and accumulates in place: no vector instruction per block of K.  A slice is 128 bytes of every operand row,
// the geometry of the 16-bit tile (moe_gemm.hip: LDS-DMA fills, XOR swizzle on the source address and on the read, loader
// waves 0-3), at twice the multiplications per byte.  Lane (fr, fq) of a fragment holds the 16-byte chunks fq and fq + 4 of
// its row: any split of the 128 columns over the lanes is right as long as both operands use the same one.
// The scale bytes of a whole tile (rows x K / 128, and two rows of the weights' grid) are put in LDS once per tile by the
// waves that do not load operands.
//
// Precision.  The 8-bit matrix instructions (this one and v_mfma_f32_16x16x32_fp8_fp8 alike) do not add in full fp32: the
// products of 8 columns are aligned to the largest of them with 13 bits below its exponent, and what lies below is cut off.
// On normal data a sum of thousands of columns is off by 1.4e-5 of its value (the bf16 instruction: 1e-8).  A 16-bit output
// does not show it.  The quantised output of the activation does, at its ties: a few 1e-4 of the hidden values go to the
// neighbouring e4m3 value, and the expert MLP's output is 0.0023 (bf16) or 0.0012 (fp16) off the 64-bit result in the 2-norm,
// where fp32 products of the same 8-bit operands give 0.0017 (bf16's own rounding) and 0.0002.  The format's own noise is
// 0.026.  The bf16 instruction on converted operands would be exact at half the rate; the rate is what 8-bit experts are for.
//
// Bound and measured.  A slice of the 256 x 256 tile takes 1.39 us when every fill hits a cache (a timing copy that re-reads two
// slices) and 1.45 to 1.65 with the fills from memory; its matrix instructions take 1.05 at the 1.95 GHz that the card holds
// under them, and so do its LDS accesses (192 KiB read, 64 KiB filled).  So 12 % at 45056 x 5632 x 2048 and 3 % at 8192^3 is what
// the memory side still costs.  The fixed part of a tile (first fills, scales, epilogue: 5 to 6.5 us) is hidden by nothing, as
// one block fills a CU's LDS.  8192 x 8192 x 8192: 2.77 PFLOP/s.
// 22528 x 2048 x 5632 (K 2048: 16 slices a tile): 247 us = 2.10 PFLOP/s; 45056 x 5632 x 2048: 467-490 us = 2.1-2.2; the gated
// product of 45056 x 2048 x 11264: 0.93-1.11 ms = 1.9-2.2 (its epilogue is 3 to 4 us of vector work a tile; bias in the
// accumulators and v_maximum3 for the block maxima: gelu_new 27424 x 2560 x 10240 x 2 1364 -> 1325 us, SwiGLU -1 %).
// Tried without gain: persistent blocks that start the next tile under the epilogue (49 spilled registers; 45056 rows 1.40 ->
// 1.52 ms, 1408 rows 94 -> 106 us for the MLP), an epilogue instance per bias and mask (116 and more spilled registers),
// super-rows of 2 to 16 row tiles (within 2 %, 16: -7 %), 8-bit outputs stored to stay in the caches (0.3 %), 32 x 32 x 64
// fragments for the 256 x 256 tile (plain products 3 % slower, the MLPs 1 %), the same in slices of 64 columns and a ring of four
// (12 % slower), fills issued between the matrix instructions (2 to 5 % slower), weight and row fragments read in other orders
// (1 %), a deeper ring for the 32-row tiles, other read-ahead depths.
#include "moe_fp8.h"

#include <climits>

namespace moe {

constexpr int FTHREADS = 512;
constexpr int FLW = 4;                 // loader waves (one per SIMD)
constexpr int FP8_STRIP = 28672;       // LDS bytes for the rows' scales of a tile
constexpr int FP8_WS_ROW = 512;        // ... and for each of the two rows of the weights' scales: K <= 65536
constexpr int FP8_MAX_K = FP8_WS_ROW * QB;

__device__ const uint4 g_fp8_zero = {0u, 0u, 0u, 0u};  // source of the columns behind K in the last slice

__device__ __forceinline__ void glds16b(const u8 *gsrc, char *lds_wave_base) {
    __builtin_amdgcn_global_load_lds(
        reinterpret_cast<const __attribute__((address_space(1))) void *>(reinterpret_cast<uintptr_t>(gsrc)),
        reinterpret_cast<__attribute__((address_space(3))) void *>(
            static_cast<unsigned>(reinterpret_cast<uintptr_t>(lds_wave_base))),
        16, 0, 0);
}
template <int N>
__device__ __forceinline__ void fwait_vm_barrier() {
    // all but the N youngest of this wave's fills have landed, then everybody's have (a __syncthreads would drain them all)
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(N) : "memory");
}
template <int N>
struct FInt { static constexpr int value = N; };

template <int EPI, int BM, int BNW>
struct FTile {
    static constexpr bool GATED = EPI == EPI_SWIGLU;
    static constexpr bool QOUT = EPI != EPI_PLAIN;            // output quantised for the next product
    static_assert(BM == 256 || BM == 192 || BM == 128 || BM == 64 || BM == 32, "row tile");
    static_assert(BNW == 256 || ((BNW == 128 || BNW == 64) && !GATED), "column tile");
    static_assert(!QOUT || (GATED ? BNW / 2 : BNW) % QB == 0, "an output block lies in one tile");
    static constexpr int SLOT = (BM + BNW) * QB;              // bytes of one K slice
    static constexpr int NS = (131072 / SLOT) > 8 ? 8 : (131072 / SLOT);
    static constexpr int NC = GATED ? BNW / 2 : BNW;          // output columns
    static constexpr int ROWB = (QOUT ? NC : NC * 2) + 16;    // bytes of an image row
    static constexpr int XS = NS * SLOT;                      // offset of the rows' scales
    static constexpr int WS = XS + FP8_STRIP;                 // ... of the weights' scales
    static constexpr int TOP = BM * ROWB;                     // offset of the block maxima (epilogue): [4][BM]
    static constexpr int LDS_K = WS + 2 * FP8_WS_ROW;
    static constexpr int LDS_E = TOP + (QOUT ? 4 * BM * 4 : 0);
    static constexpr int LDS_BYTES = LDS_K > LDS_E ? LDS_K : LDS_E;
    static_assert(NS >= 2 && LDS_BYTES <= 163840, "LDS");
    static constexpr int NF = BNW / 64;                       // 16-row weight fragments per wave
    static constexpr int WNT = BNW / 4;                       // weight rows per wave
};

// The work list of a launch, derived by every block from the device-side group sizes (scalar work).  The eight XCDs (block
// id mod 8) each take one contiguous eighth of the real tiles, in super-rows of rs row tiles: an XCD works on rs x (32 / rs)
// tiles at a time, which share their panels in its L2.
// With a workspace, the Rm < 32 tiles of an XCD's last, partial round are cut along K into s = min(32 / Rm, split_max) pieces
// that fill the round; a launch behind adds a tile's pieces in K order: no atomics, the same bits from call to call.  A cut
// tile differs from a whole one only through the order of the fp32 additions.
constexpr int FP8_XCD_CUS = 32;
template <int BM>
struct Fp8Sched {
    int RT;
    long long T;
    __device__ __forceinline__ explicit Fp8Sched(const Fp8GemmParams &p) {
        RT = 0;
        if (p.group_offsets) {
            for (int g = 0; g < p.G; ++g) RT += (p.group_offsets[g + 1] - p.group_offsets[g] + BM - 1) / BM;
        } else {
            RT = (p.max_rows + BM - 1) / BM;
        }
        T = (long long)RT * p.col_tiles;
    }
    __device__ __forceinline__ int tiles(int x) const { return (int)((T >> 3) + (x < (int)(T & 7) ? 1 : 0)); }
    __device__ __forceinline__ long long start(int x) const {
        const long long q = T >> 3, r = T & 7;
        return x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q;
    }
    // tiles of XCD x that run whole, and how many pieces each of the others is cut into
    __device__ __forceinline__ void cut(const Fp8GemmParams &p, int x, int &full, int &rm, int &s) const {
        const int n = tiles(x);
        full = n / FP8_XCD_CUS * FP8_XCD_CUS;
        rm = n - full;
        s = rm > 0 ? FP8_XCD_CUS / rm : 1;
        if (s > p.split_max) s = p.split_max;
        if (!p.splitk_ws || s < 2) { full = n; rm = 0; s = 1; }
    }
    __device__ __forceinline__ int whole(const Fp8GemmParams &p, int x) const { int f, r, s; cut(p, x, f, r, s); return f; }
    __device__ __forceinline__ int items(const Fp8GemmParams &p, int x) const { int f, r, s; cut(p, x, f, r, s); return f + r * s; }
    __device__ __forceinline__ int most_items(const Fp8GemmParams &p) const {  // of any XCD
        return (int)(T >> 3) + ((T & 7) ? 1 : 0) + (p.splitk_ws ? FP8_XCD_CUS : 0);
    }
    __device__ __forceinline__ bool item(const Fp8GemmParams &p, int x, int i, long long &t, int &piece, int &pieces) const {
        int full, rm, s;
        cut(p, x, full, rm, s);
        piece = 0;
        pieces = 1;
        if (i < full) { t = start(x) + i; return true; }
        const int j = i - full;
        if (j >= rm * s) return false;
        t = start(x) + full + j % rm;
        piece = j / rm;
        pieces = s;
        return true;
    }
    __device__ __forceinline__ void tile(const Fp8GemmParams &p, long long t, int &ct, int &row_begin, int &row_end, int &expert) const {
        const long long per = (long long)p.rs * p.col_tiles;
        const int sr = (int)(t / per), rem = (int)(t - sr * per);
        const int rin = min(p.rs, RT - sr * p.rs);
        ct = rem / rin;
        const int rt = sr * p.rs + (rem - ct * rin);
        row_begin = rt * BM;
        row_end = p.max_rows;
        expert = 0;
        if (!p.group_offsets) return;
        int tile0 = 0;
        for (int g = 0; g < p.G; ++g) {
            const int b = p.group_offsets[g], e = p.group_offsets[g + 1];
            const int nt = (e - b + BM - 1) / BM;
            if (rt < tile0 + nt) {
                row_begin = b + (rt - tile0) * BM;
                row_end = e;
                expert = g % p.n_experts;
                return;
            }
            tile0 += nt;
        }
    }
};

template <int DT, int EPI, int BM, int BNW>
__global__ __launch_bounds__(FTHREADS, 2) void fp8_gemm_kernel(const Fp8GemmParams p) {
    using T = FTile<EPI, BM, BNW>;
    typedef Elt<DT> E;
    constexpr int NS = T::NS, NF = T::NF, WNT = T::WNT, NC = T::NC, ROWB = T::ROWB;
    constexpr bool SPLITS = EPI == EPI_PLAIN && BM == 256 && BNW == 256;  // the tile whose last round is cut along K
    __shared__ __attribute__((aligned(16))) char lds[T::LDS_BYTES];

    // ---- the work item of this block: a tile, or a piece of a tile's K range (Fp8Sched) ----
    const int nk = (p.K + QB - 1) / QB;
    const Fp8Sched<BM> sch(p);
    int ct = 0, row_begin = 0, row_end = 0, expert = 0, k_lo = 0, k_hi = nk, slot = -1;
    {
        const int x = blockIdx.x & 7, i = blockIdx.x >> 3;
        long long t;
        int piece, pieces;
        if (!sch.item(p, x, i, t, piece, pieces)) {
            // surplus block of the worst-case grid.  With zero_tail the grid has at least one more than the items on every
            // XCD: those blocks clear the rows that belong to no group.
            if (!T::QOUT && p.zero_tail) {
                const int per_xcd = (int)(gridDim.x >> 3) - sch.most_items(p), k = i - sch.items(p, x);  // surplus of an XCD, at least
                const int lo = p.group_offsets[0], hi = p.group_offsets[p.G];
                if (k < per_xcd)
                    for (long long r = (long long)k * 8 + x; r < p.max_rows; r += per_xcd * 8)
                        if (r < lo || r >= hi)
                            for (int c = threadIdx.x; c < p.N_out; c += FTHREADS) ((bf16_t *)p.out)[r * p.ldo + c] = 0;
            }
            return;
        }
        sch.tile(p, t, ct, row_begin, row_end, expert);
        if (SPLITS && pieces > 1) {
            k_lo = piece * nk / pieces;
            k_hi = (piece + 1) * nk / pieces;
            slot = x * FP8_XCD_CUS + (i - sch.whole(p, x));
        }
    }

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave & 3, lwave = wave & 3;
    const int tail = p.K - (nk - 1) * QB;  // columns of the last slice (a multiple of 16)
    auto xsw = [](int row) { return (row >> 1) & 7; };
    auto src_row = [&](int prow) -> long long {
        if (prow > row_end - 1) prow = row_end - 1;  // rows behind the group are computed from its last one, never stored
        return p.gather ? (long long)(p.gather[prow] >> p.gather_shift) : (long long)prow;
    };

    // ---- operand fills: one instruction = 8 rows x 128 bytes ----
    constexpr int NPX = BM / 8 / FLW, NPW = BNW / 8 / FLW, PP = NPX + NPW;
    const u8 *a_src[NPX], *w_src[NPW];
    const int lr = lane >> 3, lc = lane & 7;
    auto setup_ptrs = [&]() {
#pragma unroll
        for (int j = 0; j < NPX; ++j) {
            const int row = (lwave * NPX + j) * 8 + lr;
            a_src[j] = p.a + src_row(row_begin + row) * p.lda + (lc ^ xsw(row)) * 16;
        }
        const u8 *wb = p.w + (long long)expert * p.w_expert_stride;
#pragma unroll
        for (int j = 0; j < NPW; ++j) {
            const int row = (lwave * NPW + j) * 8 + lr;
            int wrow;
            if (T::GATED) {
                // wave wq owns rows [wq * WNT, +WNT) of the slot: first the 'a' rows of its columns, then their 'b' rows
                const int wq = row / WNT, within = row % WNT;
                const int col = ct * NC + wq * (WNT / 2) + (within % (WNT / 2));
                wrow = min(col, p.N_out - 1) + (within / (WNT / 2)) * p.b_row_offset;
            } else {
                wrow = min(ct * BNW + row, p.N_out - 1);
            }
            w_src[j] = wb + (long long)wrow * p.K + (lc ^ xsw(row)) * 16;
        }
    };
    auto stage = [&](int buf, int kt) {
        char *slot = lds + buf * T::SLOT;
        if (kt == nk - 1 && tail < QB) {
            const u8 *z = reinterpret_cast<const u8 *>(&g_fp8_zero);
#pragma unroll
            for (int j = 0; j < NPX; ++j) {
                const int cs = lc ^ xsw((lwave * NPX + j) * 8 + lr);
                glds16b(cs * 16 < tail ? a_src[j] + (long long)kt * QB : z, slot + (lwave * NPX + j) * 1024);
            }
#pragma unroll
            for (int j = 0; j < NPW; ++j) {
                const int cs = lc ^ xsw((lwave * NPW + j) * 8 + lr);
                glds16b(cs * 16 < tail ? w_src[j] + (long long)kt * QB : z, slot + BM * QB + (lwave * NPW + j) * 1024);
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < NPX; ++j) glds16b(a_src[j] + (long long)kt * QB, slot + (lwave * NPX + j) * 1024);
#pragma unroll
        for (int j = 0; j < NPW; ++j) glds16b(w_src[j] + (long long)kt * QB, slot + BM * QB + (lwave * NPW + j) * 1024);
    };
    // ---- scales of the tile: waves 4-7.  Rows: dword (4 slices) kq of row r at XS + (kq * BM + r) * 4 ----
    auto load_scales = [&]() {
        const int t2 = tid - 256;
        const int kq_n = (nk + 3) >> 2;
        const int r = t2 % BM;
        const u8 *src = p.a_scale + src_row(row_begin + r) * p.ld_as;
        for (int kq = t2 < 256 / BM * BM ? t2 / BM : kq_n; kq < kq_n; kq += 256 / BM)
            *reinterpret_cast<unsigned *>(lds + T::XS + (kq * BM + r) * 4) = *reinterpret_cast<const unsigned *>(src + kq * 4);
        const u8 *wsb = p.w_scale + (long long)expert * p.ws_expert_stride;
        const int nb = (p.N_out + QB - 1) / QB;
        for (int i = t2; i < 2 * nk; i += 256) {
            const int h = i >= nk ? 1 : 0, kb = i - h * nk;
            int blk;
            if (T::GATED) blk = min(ct * NC / QB, nb - 1) + h * p.b_blk_offset;
            else blk = min(ct * BNW / QB + h, nb - 1);
            lds[T::WS + h * FP8_WS_ROW + kb] = (char)wsb[(long long)blk * nk + kb];
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    };

    const int fr = lane & 15, fq = lane >> 4;
    const int koff0 = (fq ^ xsw(fr)) * 16, koff1 = ((4 + fq) ^ xsw(fr)) * 16;
    const int w_off = BM * QB + (wn * WNT + fr) * QB;

    auto tile_body = [&](auto mfw_c, auto loads_c, const int row_off) {
        constexpr int MFW = decltype(mfw_c)::value;
        constexpr bool LOADS = decltype(loads_c)::value != 0;
        const int x_off = (row_off + fr) * QB;
        f32x4_t acc[NF][MFW];
        // the accumulators start at the bias where the epilogue quantises: no addition per element there
        constexpr int HF = T::GATED ? NF / 2 : NF;             // output fragments of the wave
        constexpr int CW = T::GATED ? WNT / 2 : WNT;           // output columns of the wave
        const bf16_t *bias = p.bias ? p.bias + (long long)expert * p.bias_expert_stride : nullptr;
#pragma unroll
        for (int nf = 0; nf < NF; ++nf) {
            f32x4_t b = {0.f, 0.f, 0.f, 0.f};
            if (T::QOUT && bias) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int c = min(ct * NC + wn * CW + (nf % HF) * 16 + fq * 4 + j, p.N_out - 1);
                    b[j] = E::to_f(bias[nf < HF ? c : p.b_row_offset + c]);
                }
            }
#pragma unroll
            for (int mf = 0; mf < MFW; ++mf) acc[nf][mf] = b;
        }

        if (LOADS) {
#pragma unroll
            for (int s = 0; s < NS - 1; ++s)
                if (k_lo + s < k_hi) stage(s, k_lo + s);
        } else {
            load_scales();
        }
        for (int kt = k_lo; kt < k_hi; ++kt) {
            const int ahead = k_hi - 1 - kt, at = kt - k_lo;
            static_assert((NS - 2) * PP < 64, "vmcnt field");
            switch (ahead < NS - 2 ? ahead : NS - 2) {
                case 0: fwait_vm_barrier<0>(); break;
                case 1: fwait_vm_barrier<PP>(); break;
                case 2: fwait_vm_barrier<(NS > 3 ? 2 : 0) * PP>(); break;
                case 3: fwait_vm_barrier<(NS > 4 ? 3 : 0) * PP>(); break;
                case 4: fwait_vm_barrier<(NS > 5 ? 4 : 0) * PP>(); break;
                case 5: fwait_vm_barrier<(NS > 6 ? 5 : 0) * PP>(); break;
                default: fwait_vm_barrier<(NS > 7 ? 6 : 0) * PP>(); break;
            }
            if (LOADS && kt + NS - 1 < k_hi) stage((at + NS - 1) % NS, kt + NS - 1);
            const char *lb = lds + (at % NS) * T::SLOT;
            const char *xs = lds + T::XS + ((kt >> 2) * BM + row_off + fr) * 4 + (kt & 3);
            constexpr int PD = 2;  // X fragments read ahead
            v8i_t wf[NF], xf[MFW];
            int xsc[MFW], wsc[2];
            auto ld32 = [&](const char *q) {
                const v4i_t lo = *reinterpret_cast<const v4i_t *>(q + koff0), hi = *reinterpret_cast<const v4i_t *>(q + koff1);
                return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            };
            auto ldx = [&](int t) {
                xsc[t] = (int)*reinterpret_cast<const u8 *>(xs + t * 64);
                xf[t] = ld32(lb + x_off + t * 16 * QB);
            };
            // plain: the wave's columns lie in one block of the weights' scales; gated: 'a' fragments in one, 'b' in the other
            wsc[0] = (int)*reinterpret_cast<const u8 *>(lds + T::WS + (T::GATED ? 0 : (wn * WNT) / QB) * FP8_WS_ROW + kt);
            wsc[1] = T::GATED ? (int)*reinterpret_cast<const u8 *>(lds + T::WS + FP8_WS_ROW + kt) : wsc[0];
#pragma unroll
            for (int nf = 0; nf < NF; ++nf) wf[nf] = ld32(lb + w_off + nf * 16 * QB);
#pragma unroll
            for (int t = 0; t < PD && t < MFW; ++t) ldx(t);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int t = 0; t < MFW; ++t) {
                if (t + PD < MFW) ldx(t + PD);
#pragma unroll
                for (int nf = 0; nf < NF; ++nf)
                    acc[nf][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                        wf[nf], xf[t], acc[nf][t], 0, 0, 0, wsc[T::GATED && nf >= NF / 2 ? 1 : 0], 0, xsc[t]);
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
        }
        if (SPLITS && slot >= 0) {
            // a piece: the accumulators as they are, 1 KiB per fragment in (lane, register) order; fp8_fixup_kernel adds the
            // pieces (buffer stores: one register of address, a scalar offset per fragment)
            float *ws = p.splitk_ws + (size_t)slot * (BM * BNW);
            const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(ws, 0, BM * BNW * 4, 0x00020000);
            const int sbase = __builtin_amdgcn_readfirstlane(((row_off / 16) * (BNW / 16) + wn * NF) * 1024);
            typedef unsigned u32x4v_t __attribute__((ext_vector_type(4)));
#pragma unroll
            for (int nf = 0; nf < NF; ++nf)
#pragma unroll
                for (int mf = 0; mf < MFW; ++mf)
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4v_t, acc[nf][mf]), rsrc, lane * 16,
                                                           sbase + (mf * (BNW / 16) + nf) * 1024, 0);
            return;
        }
        __syncthreads();  // every wave is done reading the ring

        auto bias_at = [&](int c) { return c < p.N_out ? E::to_f(bias[c]) : 0.f; };
        if constexpr (!T::QOUT) {
#pragma unroll
            for (int nf = 0; nf < NF; ++nf) {
                const int cl = wn * WNT + nf * 16 + fq * 4, c0 = ct * NC + cl;
                float bv[4] = {0.f, 0.f, 0.f, 0.f};
                if (bias) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) bv[j] = bias_at(c0 + j);
                }
#pragma unroll
                for (int mf = 0; mf < MFW; ++mf) {
                    uint2 o;
                    o.x = E::pack2(acc[nf][mf][0] + bv[0], acc[nf][mf][1] + bv[1]);
                    o.y = E::pack2(acc[nf][mf][2] + bv[2], acc[nf][mf][3] + bv[3]);
                    *reinterpret_cast<uint2 *>(lds + (row_off + mf * 16 + fr) * ROWB + cl * 2) = o;
                }
            }
        } else {
            // activation in fp32, the maximum of every row's block of 128 columns over the four lanes of a row (shuffles) and
            // over the waves of the block (LDS), then e4m3 into the image.  Columns behind N_out repeat the last real one, its
            // gate included (n_gated never lies between the two): they belong to the same block, so its maximum is not
            // changed, and they are not stored.
            constexpr int GW = QB / CW;                        // waves that share a block of 128 columns
            unsigned *const top = reinterpret_cast<unsigned *>(lds + T::TOP);
            float mx[MFW];
#pragma unroll
            for (int mf = 0; mf < MFW; ++mf) mx[mf] = 0.f;
#pragma unroll
            for (int nf = 0; nf < HF; ++nf) {
                const int c0 = ct * NC + wn * CW + nf * 16 + fq * 4;
#pragma unroll
                for (int mf = 0; mf < MFW; ++mf)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float a = acc[nf][mf][j];
                        float h;
                        if constexpr (T::GATED) h = (c0 + j < p.n_gated ? fast_silu(a) : 1.0f) * acc[nf + HF][mf][j];
                        else h = gelu_new_f32(a);
                        acc[nf][mf][j] = h;
                        mx[mf] = __builtin_elementwise_maximum(mx[mf], __builtin_fabsf(h));  // v_maximum3: a NaN stays
                    }
            }
#pragma unroll
            for (int mf = 0; mf < MFW; ++mf) {
                const unsigned m = umax_xor(umax_xor(abs_bits(mx[mf]), 16), 32);
                if (fq == 0) top[wn * BM + row_off + mf * 16 + fr] = m;
            }
            __syncthreads();
            const int g0 = (wn / GW) * GW;
#pragma unroll
            for (int mf = 0; mf < MFW; ++mf) {
                const int r = row_off + mf * 16 + fr;
                unsigned m = 0;
#pragma unroll
                for (int w = 0; w < GW; ++w) {
                    const unsigned o = top[(g0 + w) * BM + r];
                    m = o > m ? o : m;
                }
                const unsigned sb = scale_byte(m);
                const float inv = inv_scale(sb);
                const int blk = (ct * NC + wn * CW) / QB;
                if (wn == g0 && fq == 0 && row_begin + r < row_end && blk * QB < p.N_out)
                    p.out_scale[(long long)(row_begin + r) * p.ld_os + blk] = (u8)sb;
#pragma unroll
                for (int nf = 0; nf < HF; ++nf)
                    *reinterpret_cast<unsigned *>(lds + r * ROWB + wn * CW + nf * 16 + fq * 4) =
                        pack_fp8x4(acc[nf][mf][0] * inv, acc[nf][mf][1] * inv, acc[nf][mf][2] * inv, acc[nf][mf][3] * inv);
            }
        }
        __syncthreads();
    };
    constexpr int TF = BM / 16;
    // 256 x 256: the loader waves own 5 of the 16 row fragments, their SIMD partners 11: a loader wave spends the head of a
    // slice issuing its fills.  Measured (45056 rows, K 5632, N 2048): 473 -> 457 us; 6, 7 within 1 % of 8.
    constexpr int AMF = BM == 256 && BNW == 256 ? 5 : TF / 2;
    if (wave < FLW) {
        setup_ptrs();
        tile_body(FInt<AMF>{}, FInt<1>{}, 0);
    } else {
        tile_body(FInt<TF - AMF>{}, FInt<0>{}, AMF * 16);
    }

    if (SPLITS && slot >= 0) return;
    // ---- image -> global, 16 bytes a lane; 2 bytes a lane (consecutive lanes, consecutive columns) where the output's rows
    //      do not allow that (8 scattered 2-byte stores a lane took 13 us of a 29.5-us launch, 333 rows, K 1008, N 1003) ----
    typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
    if (!T::QOUT && !p.vec_store) {
        const int rows = min(BM, row_end - row_begin), cols = min(NC, p.N_out - ct * NC);
        constexpr int RPI = FTHREADS / 64;
        for (int r = wave; r < rows; r += RPI)
#pragma unroll
            for (int c = lane; c < NC; c += 64)
                if (c < cols)
                    ((bf16_t *)p.out)[(long long)(row_begin + r) * p.ldo + ct * NC + c] = *reinterpret_cast<const bf16_t *>(lds + r * ROWB + c * 2);
        return;
    }
    constexpr int EL = T::QOUT ? 16 : 8;  // elements per 16-byte chunk
    constexpr int CPR = NC / EL, RPI = FTHREADS / CPR;
    const int cc = tid % CPR, r0 = tid / CPR;
    const int col = ct * NC + cc * EL;
    const int left = p.N_out - col;
    if (left <= 0) return;
#pragma unroll 4
    for (int r = r0; r < BM; r += RPI) {
        const int prow = row_begin + r;
        if (prow >= row_end) break;
        const u32x4_t v = *reinterpret_cast<const u32x4_t *>(lds + r * ROWB + cc * 16);
        if constexpr (T::QOUT) {
            __builtin_nontemporal_store(v, reinterpret_cast<u32x4_t *>((u8 *)p.out + (long long)prow * p.ldo + col));
        } else {
            bf16_t *dst = (bf16_t *)p.out + (long long)prow * p.ldo + col;
            if (left >= 8) {
                __builtin_nontemporal_store(v, reinterpret_cast<u32x4_t *>(dst));
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < left) dst[j] = (bf16_t)(v[j >> 1] >> ((j & 1) * 16));
            }
        }
    }
}

// Adds the K pieces of every cut 256 x 256 tile in K order, then bias and the rounding of the plain epilogue.  The waves of a
// fixed grid take (XCD, tile, fragment) items; a fragment's pieces are read as they were stored, 1 KiB at a time.
// HBM-bound: pieces * 256 KiB read (at most 64 MiB); 4 us where the device finds nothing to add.
constexpr int FP8_FIX_BLOCKS = 256, FP8_FIX_THREADS = 1024;
template <int DT>
__global__ __launch_bounds__(FP8_FIX_THREADS) void fp8_fixup_kernel(const Fp8GemmParams p) {
    typedef Elt<DT> E;
    constexpr int BM = 256, FR = 16;  // fragments per row and column of a tile
    const Fp8Sched<BM> sch(p);
    const int lane = threadIdx.x & 63, fr = lane & 15, fq = lane >> 4;
    const int w0 = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * (FP8_FIX_THREADS / 64) + (threadIdx.x >> 6)));
    constexpr int NW = FP8_FIX_BLOCKS * (FP8_FIX_THREADS / 64);
    int base = 0;
    for (int x = 0; x < 8; ++x) {
        int full, rm, s;
        sch.cut(p, x, full, rm, s);
        const int n = rm * FR * FR;
        // items are dealt over all waves across the XCDs: the first item of XCD x goes to wave base % NW
        for (int it = (w0 - base % NW + NW) % NW; it < n; it += NW) {
            const int r = it / (FR * FR), f = it % (FR * FR);
            int ct, row_begin, row_end, expert;
            sch.tile(p, sch.start(x) + full + r, ct, row_begin, row_end, expert);
            const int row = row_begin + (f / FR) * 16 + fr, c0 = ct * 256 + (f % FR) * 16 + fq * 4;
            f32x4_t a = {0.f, 0.f, 0.f, 0.f};
            const float *ws = p.splitk_ws + (size_t)(x * FP8_XCD_CUS + r) * (BM * 256) + f * 256 + lane * 4;
#pragma unroll 4
            for (int k = 0; k < s; ++k) a += *reinterpret_cast<const f32x4_t *>(ws + (size_t)k * rm * (BM * 256));
            if (row >= row_end) continue;
            const bf16_t *bias = p.bias ? p.bias + (long long)expert * p.bias_expert_stride : nullptr;
            bf16_t *dst = (bf16_t *)p.out + (long long)row * p.ldo + c0;
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = a[j] + (bias && c0 + j < p.N_out ? E::to_f(bias[c0 + j]) : 0.f);
            if (p.vec_store && c0 + 4 <= p.N_out) {
                *reinterpret_cast<uint2 *>(dst) = make_uint2(E::pack2(v[0], v[1]), E::pack2(v[2], v[3]));
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c0 + j < p.N_out) dst[j] = E::from_f(v[j]);
            }
        }
        base += n;
    }
}

template <int DT, int EPI, int BM, int BNW>
static int launch_fp8_tile(Fp8GemmParams p, hipStream_t st) {
    using T = FTile<EPI, BM, BNW>;
    p.col_tiles = (p.N_out + T::NC - 1) / T::NC;
    p.rs = p.col_tiles <= 8 ? 3 : 4;
    const long long rt = p.group_offsets ? (long long)p.max_rows / BM + p.G : ((long long)p.max_rows + BM - 1) / BM;
    constexpr bool SPLITS = EPI == EPI_PLAIN && BM == 256 && BNW == 256;
    if (!SPLITS || p.split_max < 2) p.splitk_ws = nullptr;
    const long long grid = (rt * p.col_tiles + 7) / 8 * 8 + (p.zero_tail ? 8 : 0) + (p.splitk_ws ? 8 * FP8_XCD_CUS : 0);
    if (!grid_fits(grid, FTHREADS)) return fail(MOE_ERR_SHAPE, "fp8 product: too many tiles (%lld)", grid);
    hipLaunchKernelGGL((fp8_gemm_kernel<DT, EPI, BM, BNW>), dim3((unsigned)grid), dim3(FTHREADS), 0, st, p);
    int rc = check_launch("fp8_gemm_kernel");
    if (rc || !p.splitk_ws) return rc;
    hipLaunchKernelGGL((fp8_fixup_kernel<DT>), dim3(FP8_FIX_BLOCKS), dim3(FP8_FIX_THREADS), 0, st, p);
    return check_launch("fp8_fixup_kernel");
}

// Tile choice.  One block runs on a CU at a time, so a launch takes rounds of 256 tiles; a round takes slices * step + fixed.
// step is a CU's time per slice with its fills in flight, or, when the round's tiles together ask for more than the caches
// deliver, their (BM + BNW) * 128 bytes per slice at 13 TB/s.  The constants were measured on one-round launches (K = 5632 and
// 10240, one group and four; microseconds).  The smallest estimate is within 5 % of the best of thirteen tiles on 39 of 44
// swept shapes (100 ... 11264 rows, K 1024 ... 10240, N 1024 ... 5632, 1 to 8 groups), 1.6 % off on average and 21 % at worst;
// the 256 x 256 tile alone is up to 3.2 x off there (1408 rows, K 5632, N 2048, 4 groups: 57.9 us against 30.9).
// It ranks tiles; as a time it is low where a launch keeps all CUs busy for long and the clock falls: 4096 x 4096 x 10240 is
// estimated at 110 us and takes 124 (1.39 us a slice, not 1.29), 11264 x 2560 -> 2048 in 8 groups at 62 and takes 68 to 80.
// With a workspace, the 256 x 256 tile's last round may be cut along K (Fp8Sched): its estimate is then the whole rounds, a
// piece of the tail, and the pieces written and read back (0.11 us each at 4.7 TB/s, 5 us for the launch).  6854 rows, K
// 10240, N 2560 (290 tiles on 256 CUs): 264 us whole, 200 + 19 cut; pieces of 12, 20 or 26 slices the same, 40 slower.
struct Fp8Tile { int bm, bn; float step, fixed; };
constexpr Fp8Tile FP8_TILES[] = {{256, 256, 1.15f, 6.5f}, {192, 256, 1.0f, 6.0f}, {128, 256, 0.86f, 5.0f}, {256, 128, 0.85f, 5.0f}, {128, 128, 0.54f, 5.5f},
                                 {64, 256, 0.63f, 4.5f},  {64, 128, 0.40f, 5.5f},  {32, 256, 0.54f, 3.0f},  {32, 128, 0.38f, 5.0f},
                                 {32, 64, 0.31f, 5.0f}};
template <int EPI>
static bool fp8_tile_ok(int bm, int bn, int kq) {
    if (bm * kq > FP8_STRIP) return false;                     // the tile's scales have to fit their LDS
    if (EPI == EPI_SWIGLU) return bn == 256;                   // 128 output columns = one block of the quantisation
    if (EPI == EPI_GELU_NEW) return bn == 256 || bn == 128;
    return true;
}
constexpr int FP8_PIECE_SLICES = 12;  // a piece covers at least this many slices
constexpr size_t FP8_SPLIT_BYTES = (size_t)8 * FP8_XCD_CUS * 256 * 256 * 4;  // one 256 x 256 fp32 tile per CU: 64 MiB
// whether a product could use that workspace at all: K long enough to cut, and about a round of big tiles
static bool fp8_may_split(long long rows, int K, int N) { return K >= 32 * QB && rows / 256 * ((N + 255) / 256) >= 192; }

// the estimate, the tile and (split) the largest number of pieces: 1 = tiles stay whole
template <int EPI>
static const Fp8Tile &choose_fp8_tile(const Fp8GemmParams &p, double *estimate = nullptr, int *split = nullptr) {
    const int nk = (p.K + QB - 1) / QB, kq = (nk + 3) / 4 * 4;
    const double parts = p.max_rows < p.G ? p.max_rows : p.G;  // groups that can hold rows: half a tile of each is lost
    const Fp8Tile *best = nullptr;
    double best_t = 0;
    for (const Fp8Tile &t : FP8_TILES) {
        if (!fp8_tile_ok<EPI>(t.bm, t.bn, kq)) continue;
        const int nc = EPI == EPI_SWIGLU ? t.bn / 2 : t.bn;
        const double rt = p.G == 1 ? (double)((p.max_rows + t.bm - 1) / t.bm) : ((double)p.max_rows / t.bm + 0.5 * parts) * 1.05;
        const double tiles = rt * ((p.N_out + nc - 1) / nc);
        const double slice = (t.bm + t.bn) * 128e-6 / 13.0;    // a tile's fills of a slice at the chip's rate
        auto round_us = [&](double n, double slices) { return slices * (n * slice > t.step ? n * slice : t.step) + t.fixed; };
        const int full = (int)(tiles / 256);
        const double rest = tiles - 256.0 * full;
        double us = full * round_us(256, nk) + (rest > 0 ? round_us(rest, nk) : 0.0);
        int cut = 1;
        if (EPI == EPI_PLAIN && t.bm == 256 && t.bn == 256 && p.splitk_ws && nk >= 32) {
            const int n = (int)(tiles / 8) + 1, rm = n % FP8_XCD_CUS;
            int s = rm ? FP8_XCD_CUS / rm : 1;
            if (s > nk / FP8_PIECE_SLICES) s = nk / FP8_PIECE_SLICES;
            const double cut_us = s >= 2 ? (n / FP8_XCD_CUS) * round_us(256, nk) + round_us(8 * rm * s, (double)nk / s) + 5.0 + 8 * rm * s * 0.11 : us;
            if (cut_us < us) { us = cut_us; cut = s; }
        }
        if (!best || us < best_t) { best = &t; best_t = us; if (split) *split = cut; }
    }
    if (estimate) *estimate = best_t;
    return *best;
}

template <int DT, int EPI>
static int launch_fp8_gemm(Fp8GemmParams p, hipStream_t st) {
    int bm, bn;
    p.split_max = 1;
    const Knobs &k = knobs();
    bool forced = false;                                       // MOE_GEMM_TILE, where it names a tile of this table
    for (const Fp8Tile &t : FP8_TILES) forced |= t.bm == k.tile_bm && t.bn == k.tile_bnw;
    if (forced && fp8_tile_ok<EPI>(k.tile_bm, k.tile_bnw, ((p.K + QB - 1) / QB + 3) / 4 * 4)) {
        bm = k.tile_bm; bn = k.tile_bnw;
        if (bm == 256 && bn == 256) p.split_max = k.splitk;
    } else {
        const Fp8Tile &t = choose_fp8_tile<EPI>(p, nullptr, &p.split_max);
        bm = t.bm; bn = t.bn;
    }
#define FP8_TILE(M_, N_) if (bm == M_ && bn == N_) return launch_fp8_tile<DT, EPI, M_, N_>(p, st);
    FP8_TILE(256, 256) FP8_TILE(192, 256) FP8_TILE(128, 256) FP8_TILE(64, 256) FP8_TILE(32, 256)
    if constexpr (EPI != EPI_SWIGLU) { FP8_TILE(256, 128) FP8_TILE(128, 128) FP8_TILE(64, 128) FP8_TILE(32, 128) }
    if constexpr (EPI == EPI_PLAIN) { FP8_TILE(32, 64) }
#undef FP8_TILE
    return fail(MOE_ERR_ARG, "fp8 product: no tile %d x %d", bm, bn);
}

static int fp8_gemm(Fp8GemmParams p, int epilogue, int dtype, hipStream_t st) {
    p.dtype = dtype;
    if (p.max_rows == 0) return 0;
    // Few rows stream the weights.  The few-row kernel's time is its start and end and the active weights at the HBM rate,
    // more with 17 to 32 rows a group (two row fragments per weight fragment), twice with more (the weights twice); the tiles'
    // is choose_fp8_tile's estimate, or the weights at the rate that their fewer blocks reach.  Measured, us (few / tiles):
    // K 2048, N 5632: 8.0 / 8.8 at 16 rows, 10.0 / 8.9 at 32, 14.6 / 8.9 at 48; K 5632, N 2048: 8.8 / 17.5, 11.6 / 17.6, 17.3 /
    // 17.6; K = N = 1024: 3.9 / 7.1, 4.8 / 7.2, 6.3 / 7.4.  It has no rows to clear: zero_tail launches stay on the tiles.
    if (epilogue == MOE_EPI_PLAIN && p.max_rows <= FP8_FEW_ROWS && !p.zero_tail) {
        const double act = p.max_rows < p.G ? p.max_rows : p.G, mb = act * p.N_out * p.K * 1e-6, per = p.max_rows / act;
        const double few = (5.0 + mb / 5.2) * (per > 32 ? 2.0 : per > 16 ? 1.25 : 1.0);
        double tiles = 0;
        choose_fp8_tile<EPI_PLAIN>(p, &tiles);
        if (few < (tiles > mb / 4.5 ? tiles : mb / 4.5)) return launch_fp8_few(p, st);
    }
#define FP8_EPI(DT_)                                                                   \
    switch (epilogue) {                                                                \
        case MOE_EPI_SWIGLU: return launch_fp8_gemm<DT_, EPI_SWIGLU>(p, st);           \
        case MOE_EPI_GELU_NEW: return launch_fp8_gemm<DT_, EPI_GELU_NEW>(p, st);       \
        default: return launch_fp8_gemm<DT_, EPI_PLAIN>(p, st);                        \
    }
    if (dtype == MOE_DTYPE_F16) { FP8_EPI(DT_F16) }
    FP8_EPI(DT_BF16)
#undef FP8_EPI
}

// shape, stride and alignment rules that every product shares; nothing is launched when one is broken
static int fp8_args_ok(const char *fn, const void *a, int64_t lda, const void *a_scale, int64_t ld_as, int gather_shift,
                       const void *w, const void *w_scale, const void *bias, int G, int n_experts, int max_rows, int K, int N) {
    if (!a || !a_scale || !w || !w_scale) return fail(MOE_ERR_ARG, "%s: null pointer", fn);
    if (K < 16 || (K & 15) || K > FP8_MAX_K) return fail(MOE_ERR_SHAPE, "%s: need K %% 16 == 0, 16 <= K <= %d (K=%d)", fn, FP8_MAX_K, K);
    if (N < 1 || G < 1 || G > 4096 || n_experts < 1 || max_rows < 0 || gather_shift < 0 || gather_shift > 1)
        return fail(MOE_ERR_SHAPE, "%s: need N >= 1, 1 <= G <= 4096, experts >= 1, rows >= 0 (N=%d G=%d experts=%d rows=%d)", fn, N, G, n_experts, max_rows);
    if (N > DIM_MAX || max_rows > DIM_MAX) return fail(MOE_ERR_SHAPE, "%s: N=%d, rows=%d: at most %d", fn, N, max_rows, DIM_MAX);
    if (lda < K || (lda & 15)) return fail(MOE_ERR_SHAPE, "%s: row stride %lld: need >= K and a multiple of 16", fn, (long long)lda);
    const int kb = (K + QB - 1) / QB;
    if (ld_as < kb || (ld_as & 3)) return fail(MOE_ERR_SHAPE, "%s: scale row stride %lld: need >= %d and a multiple of 4", fn, (long long)ld_as, kb);
    if (!aligned16(a) || !aligned16(w)) return fail(MOE_ERR_ALIGN, "%s: operands must be 16-byte aligned", fn);
    if (reinterpret_cast<uintptr_t>(a_scale) & 3) return fail(MOE_ERR_ALIGN, "%s: row scales must be 4-byte aligned", fn);
    if (bias && (reinterpret_cast<uintptr_t>(bias) & 1)) return fail(MOE_ERR_ALIGN, "%s: bias must be 2-byte aligned", fn);
    return 0;
}

static Fp8GemmParams plain_params(const void *a, int64_t lda, const void *a_scale, int64_t ld_as, const int32_t *gather,
                                  int gather_shift, const void *w, const void *w_scale, const void *bias,
                                  const int32_t *group_offsets, int G, int n_experts, int max_rows, int K, int N, int zero_tail,
                                  void *out, int64_t ldo) {
    const int nk = (K + QB - 1) / QB, nb = (N + QB - 1) / QB;
    Fp8GemmParams p{};
    p.a = (const u8 *)a; p.lda = lda; p.a_scale = (const u8 *)a_scale; p.ld_as = ld_as;
    p.gather = gather; p.gather_shift = gather_shift;
    p.w = (const u8 *)w; p.w_expert_stride = (long long)N * K;
    p.w_scale = (const u8 *)w_scale; p.ws_expert_stride = (long long)nb * nk;
    p.bias = (const bf16_t *)bias; p.bias_expert_stride = N;
    p.group_offsets = group_offsets; p.G = G; p.n_experts = n_experts; p.max_rows = max_rows;
    p.out = out; p.ldo = ldo; p.K = K; p.N_out = N; p.n_gated = N;
    p.vec_store = aligned16(out) && (ldo & 7) == 0;
    p.zero_tail = zero_tail != 0 && group_offsets != nullptr;
    return p;
}

}  // namespace moe

using namespace moe;

extern "C" int moe_grouped_gemm_fp8_fwd(const void *a, int64_t lda, const void *a_scale, int64_t ld_as, const int32_t *gather,
                                        int gather_shift, const void *w, const void *w_scale, const void *bias,
                                        const int32_t *group_offsets, int G, int n_experts_local, int max_rows, int K, int N,
                                        int zero_tail, void *out, int64_t ldo, int dtype, void *stream) {
    const char *fn = "moe_grouped_gemm_fp8_fwd";
    if (dtype != MOE_DTYPE_BF16 && dtype != MOE_DTYPE_F16) return fail(MOE_ERR_ARG, "%s: unknown dtype %d", fn, dtype);
    if (!out || (!group_offsets && G != 1)) return fail(MOE_ERR_ARG, "%s: null pointer", fn);
    int rc = fp8_args_ok(fn, a, lda, a_scale, ld_as, gather_shift, w, w_scale, bias, G, n_experts_local, max_rows, K, N);
    if (rc) return rc;
    if (ldo < N) return fail(MOE_ERR_SHAPE, "%s: output row stride %lld < N", fn, (long long)ldo);
    if (reinterpret_cast<uintptr_t>(out) & 1) return fail(MOE_ERR_ALIGN, "%s: out must be 2-byte aligned", fn);
    return fp8_gemm(plain_params(a, lda, a_scale, ld_as, gather, gather_shift, w, w_scale, bias, group_offsets, G, n_experts_local,
                                 max_rows, K, N, zero_tail, out, ldo),
                    MOE_EPI_PLAIN, dtype, (hipStream_t)stream);
}

extern "C" size_t moe_grouped_linear_fp8_workspace_bytes(int rows, int K) {
    if (rows < 0 || K < 1) return 0;
    const size_t q = ((size_t)rows * K + 255) & ~(size_t)255, qs = (size_t)rows * (((K + QB - 1) / QB + 3) / 4 * 4);
    // the K pieces' share: N is not known here, so long K and about a round of big tiles at N = 2048
    return q + (fp8_may_split(rows, K, 2048) ? ((qs + 255) & ~(size_t)255) + FP8_SPLIT_BYTES : qs);
}

extern "C" int moe_grouped_linear_fp8_fwd(const void *x, int64_t ldx, const void *w, const void *w_scale, const void *bias,
                                          const int32_t *group_offsets, int G, int n_experts_local, int rows, int K, int N,
                                          int zero_tail, void *workspace, size_t ws_bytes, void *out, int64_t ldo, int dtype,
                                          void *stream) {
    const char *fn = "moe_grouped_linear_fp8_fwd";
    if (!x || !workspace || !out || (!group_offsets && G != 1)) return fail(MOE_ERR_ARG, "%s: null pointer", fn);
    if (dtype != MOE_DTYPE_BF16 && dtype != MOE_DTYPE_F16) return fail(MOE_ERR_ARG, "%s: unknown dtype %d", fn, dtype);
    const long long ld_as = ((K + QB - 1) / QB + 3) / 4 * 4;
    // the product's own rules first, so that a bad call launches nothing
    int rc = fp8_args_ok(fn, workspace, K, workspace, ld_as, 0, w, w_scale, bias, G, n_experts_local, rows, K, N);
    if (rc) return rc;
    if (ldo < N || (rows > 1 && ldx < K)) return fail(MOE_ERR_SHAPE, "%s: row strides %lld, %lld: need >= K, >= N", fn, (long long)ldx, (long long)ldo);
    if ((reinterpret_cast<uintptr_t>(x) & 1) || (reinterpret_cast<uintptr_t>(out) & 1)) return fail(MOE_ERR_ALIGN, "%s: x and out must be 2-byte aligned", fn);
    if (ws_bytes < moe_grouped_linear_fp8_workspace_bytes(rows, K)) return fail(MOE_ERR_WORKSPACE, "%s: workspace %zu bytes too small", fn, ws_bytes);
    if (rows == 0) return 0;
    u8 *q = (u8 *)workspace, *qs = q + (((size_t)rows * K + 255) & ~(size_t)255);
    Fp8GemmParams p = plain_params(q, K, qs, ld_as, nullptr, 0, w, w_scale, bias, group_offsets, G, n_experts_local, rows, K, N,
                                   zero_tail, out, ldo);
    if ((rc = moe_quantize_rows_fp8(x, ldx, rows, K, q, K, qs, ld_as, dtype, stream))) return rc;
    if (fp8_may_split(rows, K, 2048)) p.splitk_ws = (float *)(qs + (((size_t)rows * ld_as + 255) & ~(size_t)255));
    return fp8_gemm(p, MOE_EPI_PLAIN, dtype, (hipStream_t)stream);
}

namespace {
inline size_t pad256b(size_t b) { return (b + 255) & ~(size_t)255; }
struct FfnWs {
    u8 *hq, *hs, *aq, *as;
    float *split;
    long long ld_hs, ld_as;
    size_t total;
};
FfnWs carve_ffn(void *ws, int src_rows, int max_rows, int M, int I) {
    FfnWs r;
    char *base = (char *)ws;
    size_t off = 0;
    auto take = [&](size_t bytes) { char *q = base + off; off += pad256b(bytes); return (u8 *)q; };
    r.ld_hs = ((I + QB - 1) / QB + 3) / 4 * 4;
    r.ld_as = ((M + QB - 1) / QB + 3) / 4 * 4;
    r.hq = take((size_t)max_rows * I);
    r.hs = take((size_t)max_rows * r.ld_hs);
    r.aq = take((size_t)src_rows * M);
    r.as = take((size_t)src_rows * r.ld_as);
    r.split = fp8_may_split(max_rows, I, M) ? (float *)take(FP8_SPLIT_BYTES) : nullptr;
    r.total = off;
    return r;
}
}  // namespace

extern "C" size_t moe_expert_ffn_fp8_workspace_bytes(int src_rows, int max_rows, int M, int I) {
    if (src_rows < 0 || max_rows < 0 || M < 1 || I < 1) return 0;
    return carve_ffn(nullptr, src_rows, max_rows, M, I).total;
}

extern "C" int moe_expert_ffn_fp8_fwd(int act, const void *x, int64_t ldx, int src_rows, const void *a, int64_t lda,
                                      const void *a_scale, int64_t ld_as, const int32_t *gather, int gather_shift,
                                      const void *w1, const void *w1_scale, const void *b1, const void *w2,
                                      const void *w2_scale, const void *b2, const int32_t *group_offsets, int G,
                                      int n_experts_local, int max_rows, int M, int I, int n_gated, void *workspace,
                                      size_t ws_bytes, void *y, int dtype, void *stream) {
    const char *fn = "moe_expert_ffn_fp8_fwd";
    if (act != MOE_ACT_SWIGLU && act != MOE_ACT_GELU_NEW) return fail(MOE_ERR_ARG, "%s: unknown act %d", fn, act);
    if (dtype != MOE_DTYPE_BF16 && dtype != MOE_DTYPE_F16) return fail(MOE_ERR_ARG, "%s: unknown dtype %d", fn, dtype);
    if ((!x) == (!a)) return fail(MOE_ERR_ARG, "%s: give either 16-bit rows x or 8-bit rows a", fn);
    if (!group_offsets || !workspace || !y) return fail(MOE_ERR_ARG, "%s: null pointer", fn);
    if (src_rows < 0 || max_rows < 0) return fail(MOE_ERR_SHAPE, "%s: negative row count", fn);
    if (M < 16 || (M & 15) || I < 16 || (I & 15)) return fail(MOE_ERR_SHAPE, "%s: need M %% 16 == 0 and I %% 16 == 0 (M=%d I=%d)", fn, M, I);
    if (!aligned16(workspace) || !aligned16(y)) return fail(MOE_ERR_ALIGN, "%s: workspace and y must be 16-byte aligned", fn);
    const FfnWs ws = carve_ffn(workspace, x ? src_rows : 0, max_rows, M, I);
    if (ws_bytes < ws.total) return fail(MOE_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", fn, ws_bytes, ws.total);
    if (x) {
        if (src_rows > 1 && ldx < M) return fail(MOE_ERR_SHAPE, "%s: row stride %lld < M", fn, (long long)ldx);
        if (reinterpret_cast<uintptr_t>(x) & 1) return fail(MOE_ERR_ALIGN, "%s: x must be 2-byte aligned", fn);
        a = max_rows ? ws.aq : workspace; lda = M; a_scale = max_rows ? ws.as : workspace; ld_as = ws.ld_as;
    }
    int rc = fp8_args_ok(fn, a, lda, a_scale, ld_as, gather_shift, w1, w1_scale, b1, G, n_experts_local, max_rows, M, I);
    if (rc) return rc;
    rc = fp8_args_ok(fn, workspace, I, workspace, ws.ld_hs, 0, w2, w2_scale, b2, G, n_experts_local, max_rows, I, M);
    if (rc) return rc;
    if (max_rows == 0) return 0;
    if (x && (rc = moe_quantize_rows_fp8(x, ldx, src_rows, M, ws.aq, M, ws.as, ws.ld_as, dtype, stream))) return rc;
    const bool gated = act == MOE_ACT_SWIGLU;
    const int mb = (M + QB - 1) / QB, ib = (I + QB - 1) / QB;
    Fp8GemmParams p{};
    p.a = (const u8 *)a; p.lda = lda; p.a_scale = (const u8 *)a_scale; p.ld_as = ld_as;
    p.gather = gather; p.gather_shift = gather_shift;
    p.w = (const u8 *)w1; p.w_expert_stride = (long long)(gated ? 2 : 1) * I * M;
    p.w_scale = (const u8 *)w1_scale; p.ws_expert_stride = (long long)(gated ? 2 : 1) * ib * mb;
    p.bias = (const bf16_t *)b1; p.bias_expert_stride = (gated ? 2 : 1) * (long long)I;
    p.group_offsets = group_offsets; p.G = G; p.n_experts = n_experts_local; p.max_rows = max_rows;
    p.out = ws.hq; p.ldo = I; p.out_scale = ws.hs; p.ld_os = ws.ld_hs;
    p.K = M; p.N_out = I; p.b_row_offset = I; p.b_blk_offset = ib;
    // no mask: no column is past it.  The columns behind I that the last tile computes as repeats of column I - 1 count in a
    // block's maximum, so they have to be gated as that column is (with a mask, n_gated < I: both lie behind it).
    p.n_gated = (n_gated < 0 || n_gated >= I) ? INT_MAX : n_gated;
    if ((rc = fp8_gemm(p, gated ? MOE_EPI_SWIGLU : MOE_EPI_GELU_NEW, dtype, (hipStream_t)stream))) return rc;
    p = plain_params(ws.hq, I, ws.hs, ws.ld_hs, nullptr, 0, w2, w2_scale, b2, group_offsets, G, n_experts_local, max_rows, I, M, 0, y, M);
    p.splitk_ws = ws.split;
    return fp8_gemm(p, MOE_EPI_PLAIN, dtype, (hipStream_t)stream);
}
