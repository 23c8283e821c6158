/* w4_tile.h — the matrix-unit kernel of the int4 group-scale products (w4.hip) for many rows, instantiated by
 * w4_tiled.hip, and what the kernel for a few rows (w4_rows.hip) shares with it.
 *
 * A workgroup computes TM rows x TN output channels (GLU: gate and up of TN channels) over a range of K, in steps of
 * KS columns. Rows of x are the A operand of v_mfma_f32_16x16x32_bf16 and weights the B operand, so a lane's four
 * results are four rows of ONE channel and a group's scale is one value per lane.
 *
 * Weights as operands. A nibble q becomes the bf16 value 16 + q by bit operations alone (mantissa bits 3..6 of
 * 2^4: two operations per two weights, exact), and what that adds comes off through the C operand of the group's first
 * matrix instruction: C = -(16 + z) * sum of the row's x over the group, whose sums are made once where x is staged.
 * Products are exact in f32; the group's sum is scaled in f32 and added to the accumulator. (Rounding q * s to bf16
 * instead would cost 2^-9 per weight.) The pairs that come out of a dword are nibbles (i, i + 4): x is staged in the
 * same order inside every 8 columns.
 *
 * Groups. A lane (channel c = lane & 15, quarter q = lane >> 4) reads 16 bytes = 32 columns of its channel per
 * 128-column block: columns 32 q .. Instruction r multiplies dword r of all four quarters, which lie in one group only
 * if G = 128. For G = 64 two and for G = 32 four cross-lane swaps per 16 bytes re-deal the dwords so that instruction r
 * covers columns of one group; w4_koff says which, and the x operand is read accordingly.
 *
 * Staging. Weights and x of the next step are on their way in registers (plain loads, whole 64- or 256-byte runs
 * per row); a step is written to one of two LDS buffers, one barrier per step that orders LDS only. Scales and zero
 * points come CC columns at a time, in runs of up to 64 bytes per row: read step by step, a few bytes of a line each,
 * they cost as many requests as the weights themselves. Columns behind K count as zero, rows and channels that are not
 * there repeat others, so that every step runs whole. */
#ifndef PLOW_MOE_W4_TILE_H
#define PLOW_MOE_W4_TILE_H

#include "common.h"
#include "kernels.h"

/* K split of the dense products: the workgroups of slice z take the steps [z * steps_per, ...) and write f32 sums to
 * part [slices][streams][M][N]; 0 slices = no split */
struct W4Tiles {
    uint32_t slices, steps_per;
    float* part;
};

/* whether the choice behind which a launch of routed experts went out names its form: 0 tiles of 16 rows, 1 of 64 */
__device__ __forceinline__ bool w4_chosen(const GroupW4& g, uint32_t form) {
    return *(const __attribute__((address_space(4))) uint32_t*)g.ws == form; /* written by an earlier kernel: a scalar load */
}

__device__ __forceinline__ float w4_f32(uint32_t h, uint32_t f16) {
    asm("" : "+v"(f16)); /* a select, no branch */
    return f16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)h) : __uint_as_float(h << 16);
}

/* column, inside a 128-column block, of the first of the 8 values that instruction r takes from quarter q */
template <int G>
__device__ __forceinline__ uint32_t w4_koff(uint32_t q, uint32_t r) {
    if (G == 128) return 32u * q + 8u * r;
    if (G == 64) return (q < 2u ? 32u * q : 32u * (q - 2u) + 16u) + 8u * (r & 1u) + 64u * (r >> 1);
    return 32u * r + 8u * q;
}
/* re-deals a lane's four dwords between the quarters so that they fit w4_koff */
template <int G>
__device__ __forceinline__ void w4_deal(uint32_t (&d)[4]) {
    if (G == 128) return;
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const auto s = __builtin_amdgcn_permlane32_swap(d[j], d[j + 2], false, false);
        d[j] = s[0], d[j + 2] = s[1];
    }
    if (G == 64) return;
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
        const auto s = __builtin_amdgcn_permlane16_swap(d[j], d[j + 1], false, false);
        d[j] = s[0], d[j + 1] = s[1];
    }
}
/* 8 nibbles -> 8 bf16 values 16 + q, in the order (0, 4), (1, 5), (2, 6), (3, 7). The two constants are kept from the
 * compiler's sight in registers: as literals they cost an instruction each, since the fused and-or takes no literal. */
struct W4Bits {
    uint32_t mask, base;
};
__device__ __forceinline__ W4Bits w4_bits() {
    W4Bits k = {0x00780078u, 0x41804180u};
    asm("" : "+v"(k.mask), "+s"(k.base));
    return k;
}
__device__ __forceinline__ v8bf w4_unpack(uint32_t w, const W4Bits& k) {
    v4i r;
    r[0] = (int)(((w << 3) & k.mask) | k.base);
    r[1] = (int)(((w >> 1) & k.mask) | k.base);
    r[2] = (int)(((w >> 5) & k.mask) | k.base);
    r[3] = (int)(((w >> 9) & k.mask) | k.base);
    return __builtin_bit_cast(v8bf, r);
}
/* the same order for 8 staged values of x */
__device__ __forceinline__ v4i w4_order(v4i x) {
    v4i r;
    r[0] = (int)__builtin_amdgcn_perm((uint32_t)x[2], (uint32_t)x[0], 0x05040100u);
    r[1] = (int)__builtin_amdgcn_perm((uint32_t)x[2], (uint32_t)x[0], 0x07060302u);
    r[2] = (int)__builtin_amdgcn_perm((uint32_t)x[3], (uint32_t)x[1], 0x05040100u);
    r[3] = (int)__builtin_amdgcn_perm((uint32_t)x[3], (uint32_t)x[1], 0x07060302u);
    return r;
}
__device__ __forceinline__ float w4_dot2(uint32_t a, uint32_t b, float acc) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, a), __builtin_bit_cast(v2bf, b), acc, false);
}
template <int CTRL>
__device__ __forceinline__ float w4_dpp_sum(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}
/* sum over aligned runs of LANES (4, 8, 16) lanes, in each of them */
template <int LANES>
__device__ __forceinline__ float w4_run_sum(float v) {
    v = w4_dpp_sum<0xB1>(v); /* quad_perm 1,0,3,2 */
    v = w4_dpp_sum<0x4E>(v); /* quad_perm 2,3,0,1 */
    if (LANES >= 8) v = w4_dpp_sum<0x141>(v); /* row_half_mirror */
    if (LANES >= 16) v = w4_dpp_sum<0x140>(v); /* row_mirror */
    return v;
}

/* CC: columns whose scales are staged together (a multiple of KS) */
template <int WT_, int WC_, int MTW_, int NBW_, int NS_, int KS_, int CC_, int G_, bool ASYM_>
struct W4Cfg {
    static constexpr int WT = WT_, WC = WC_, MTW = MTW_, NBW = NBW_, NS = NS_, KS = KS_, CC = CC_, G = G_;
    static constexpr bool ASYM = ASYM_;
    static constexpr int THREADS = WT * WC * 64, TM = WT * MTW * 16, TN = WC * NBW * 16;
    static constexpr int GS = KS / G;                      /* groups per step */
    static constexpr int XP = KS / 8, WP = KS / 32;        /* 16-byte pieces per row and step */
    static constexpr int XL = TM * XP / THREADS, WL = NS * TN * WP / THREADS; /* pieces a thread stages */
    /* a chunk's scales and zero points of one weight row: bytes, bytes per load, loads per thread, LDS pitch (16 rows
     * on different banks) */
    static constexpr int CS = CC / KS, SC = CC / G, SB = SC * 2, ZB = SC, SP = SB < 16 ? SB : 16, ZP = ZB < 16 ? ZB : 16;
    static constexpr int SN = NS * TN * (SB / SP), ZN = NS * TN * (ZB / ZP);
    static constexpr int SL = (SN + THREADS - 1) / THREADS, ZL = (ZN + THREADS - 1) / THREADS;
    static constexpr int SROW = SB <= 16 ? SB : SB + 16, ZROW = ZB <= 16 ? ZB : ZB + 16;
    static constexpr int XROW = KS * 2 + 16, WROW = KS / 2 + 16; /* LDS row pitches: rows 4 banks apart */
    static constexpr int X_BYTES = TM * XROW, W_BYTES = NS * TN * WROW, XS_BYTES = GS * TM * 4;
    static constexpr int S_BYTES = NS * TN * SROW, Z_BYTES = ASYM ? NS * TN * ZROW : 0;
    static constexpr int BUF = X_BYTES + W_BYTES + XS_BYTES, SBUF = S_BYTES + Z_BYTES;
    static constexpr int LDS = 2 * BUF + 2 * SBUF; /* two buffers of a step, two of a chunk's scales */
    static_assert(TM * XP % THREADS == 0 && NS * TN * WP % THREADS == 0 && XL >= 1 && WL >= 1, "whole pieces per thread");
    static_assert(LDS <= 160 * 1024, "two buffers fit the CU");
    static_assert(CC % KS == 0 && CC % 128 == 0 && SP >= 4 && ZP >= 4, "a chunk is whole steps");
    static_assert(THREADS % XP == 0 && XP % (G / 8) == 0, "a group's pieces lie in neighbouring lanes");
    static_assert(TN % (THREADS / WP) == 0 && XL % (G / 8 < XL ? G / 8 : XL) == 0, "a load covers rows of one stream");
};

/* what a thread has on its way for one step, and for one chunk's scales */
template <class C>
struct W4Stage {
    v4i x[C::XL], w[C::WL];
};
template <class C>
struct W4Scales {
    uint32_t s[C::SL][C::SP / 4], z[C::ASYM ? C::ZL : 1][C::ZP / 4];
};

template <class C>
__device__ __forceinline__ void w4_tile(const GroupW4& g, const W4Tiles& tl, uint8_t* lds, uint32_t e, uint32_t r0, uint32_t cnt,
                                        uint32_t rb, uint32_t n0, uint32_t slice) {
    constexpr int G = C::G, KS = C::KS, NS = C::NS;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, c = lane & 15u, q = lane >> 4;
    const uint32_t wv = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
    const uint32_t wt = wv / C::WC, wc = wv % C::WC;
    const uint32_t K = g.K, N = g.N, KG = K / (uint32_t)G;
    const uint32_t steps = (K + KS - 1u) / KS;
    const uint32_t s_lo = tl.slices ? slice * tl.steps_per : 0u;
    const uint32_t s_hi = tl.slices ? (s_lo + tl.steps_per < steps ? s_lo + tl.steps_per : steps) : steps;

    /* ---- where this thread's pieces come from ---- */
    const uint8_t* xsrc[C::XL];
    const uint32_t xp = tid % C::XP;
#pragma unroll
    for (int j = 0; j < C::XL; j++) {
        const uint32_t t = rb + (tid + (uint32_t)j * C::THREADS) / C::XP;
        uint32_t ai = PLOW_EXPERT_UNUSED;
        if (t < cnt) ai = g.a_idx ? g.a_idx[r0 + t] : r0 + t;
        xsrc[j] = (const uint8_t*)g.x + (size_t)(ai != PLOW_EXPERT_UNUSED ? ai : 0u) * g.ldx * 2u;
    }
    /* a tile's first channel of each stream, and 32-bit offsets from there (K < 2^24, so they fit) */
    auto tensor = [&](const uint64_t* tab, const void* const* direct, uint32_t st, uint32_t pitch) -> const uint8_t* {
        const uint8_t* const p = tab ? (const uint8_t*)(uintptr_t)tab[(size_t)e * 3u + g.sel[st]] : (const uint8_t*)direct[st];
        return p + (size_t)n0 * pitch;
    };
    const uint8_t *wbase[NS], *sbase[NS], *zbase[NS];
#pragma unroll
    for (int st = 0; st < NS; st++) {
        wbase[st] = tensor(g.wtab, g.w, st, K / 2u), sbase[st] = tensor(g.stab, g.s, st, KG * 2u);
        zbase[st] = C::ASYM ? tensor(g.ztab, g.z, st, KG) : nullptr;
    }
    const uint32_t wp = tid % C::WP, last = N - 1u - n0;
    constexpr int WR = C::THREADS / C::WP, XR = C::THREADS / C::XP; /* rows that the workgroup loads at once */
    uint32_t woff[C::WL];
#pragma unroll
    for (int j = 0; j < C::WL; j++) {
        const uint32_t ch = tid / C::WP + (uint32_t)(j * WR % C::TN);
        woff[j] = (ch < last ? ch : last) * (K / 2u);
    }
    /* scale piece j of this thread: weight row (stream, channel) and the first of its SP bytes in the chunk */
    auto scale_row = [&](const uint8_t* const* base, uint32_t row, uint32_t pitch) -> const uint8_t* {
        const uint32_t ch = row % C::TN;
        return (NS == 2 && row >= (uint32_t)C::TN ? base[NS - 1] : base[0]) + (ch < last ? ch : last) * pitch;
    };
    auto load_scales = [&](W4Scales<C>& b, uint32_t step) { /* of the chunk that starts with `step` */
        const uint32_t g0 = step * C::GS;
        const bool whole = g0 + C::SC <= KG;
#pragma unroll
        for (int j = 0; j < C::SL; j++) {
            const uint32_t i = tid + (uint32_t)j * C::THREADS, row = i / (C::SB / C::SP), off = (i % (C::SB / C::SP)) * C::SP;
            if (C::SN % C::THREADS == 0 || i < (uint32_t)C::SN) {
                const uint8_t* const p = scale_row(sbase, row, KG * 2u) + g0 * 2u + off;
                if (whole) {
                    __builtin_memcpy(b.s[j], p, C::SP); /* rows are aligned to an element only */
                } else {
#pragma unroll
                    for (uint32_t h = 0; h < C::SP / 4; h++) {
                        const uint32_t gi = g0 + off / 2u + 2u * h;
                        const uint32_t a = gi < KG ? *(const uint16_t*)(p + 4u * h) : 0u, c1 = gi + 1u < KG ? *(const uint16_t*)(p + 4u * h + 2u) : 0u;
                        b.s[j][h] = a | (c1 << 16);
                    }
                }
            }
        }
        if (!C::ASYM) return;
#pragma unroll
        for (int j = 0; j < C::ZL; j++) {
            const uint32_t i = tid + (uint32_t)j * C::THREADS, row = i / (C::ZB / C::ZP), off = (i % (C::ZB / C::ZP)) * C::ZP;
            if (C::ZN % C::THREADS == 0 || i < (uint32_t)C::ZN) {
                const uint8_t* const p = scale_row(zbase, row, KG) + g0 + off;
                if (whole) {
                    __builtin_memcpy(b.z[j], p, C::ZP);
                } else {
#pragma unroll
                    for (uint32_t h = 0; h < C::ZP / 4; h++) {
                        uint32_t v = 0u;
#pragma unroll
                        for (uint32_t i4 = 0; i4 < 4u; i4++) v |= (g0 + off + 4u * h + i4 < KG ? (uint32_t)p[4u * h + i4] : 0u) << (8u * i4);
                        b.z[j][h] = v;
                    }
                }
            }
        }
    };
    auto stage_scales = [&](const W4Scales<C>& b, uint8_t* buf) {
#pragma unroll
        for (int j = 0; j < C::SL; j++) {
            const uint32_t i = tid + (uint32_t)j * C::THREADS;
            if (C::SN % C::THREADS == 0 || i < (uint32_t)C::SN)
                __builtin_memcpy(__builtin_assume_aligned(buf + (i / (C::SB / C::SP)) * C::SROW + (i % (C::SB / C::SP)) * C::SP, C::SP), b.s[j], C::SP);
        }
        if (!C::ASYM) return;
#pragma unroll
        for (int j = 0; j < C::ZL; j++) {
            const uint32_t i = tid + (uint32_t)j * C::THREADS;
            if (C::ZN % C::THREADS == 0 || i < (uint32_t)C::ZN)
                __builtin_memcpy(__builtin_assume_aligned(buf + C::S_BYTES + (i / (C::ZB / C::ZP)) * C::ZROW + (i % (C::ZB / C::ZP)) * C::ZP, C::ZP), b.z[j], C::ZP);
        }
    };

    /* No load stands under a condition, so that the compiler can count what is in flight: a step past the end is the
     * last one again, a piece past the end of a row the row's last (x counts as zero there), a row that is not there
     * row 0. */
    auto load = [&](W4Stage<C>& b, uint32_t step) {
        step = step < s_hi ? step : s_hi - 1u;
        const uint32_t k = step * KS, wk = k / 2u + wp * 16u, xk = k + xp * 8u;
        const uint32_t wo = wk < K / 2u - 16u ? wk : K / 2u - 16u, xo = xk < K - 8u ? xk : K - 8u;
#pragma unroll
        for (int j = 0; j < C::WL; j++) b.w[j] = *(const v4i*)(wbase[j * WR / C::TN] + (woff[j] + wo));
#pragma unroll
        for (int j = 0; j < C::XL; j++) b.x[j] = *(const v4i*)(xsrc[j] + (size_t)xo * 2u);
    };
    /* rows that are not there hold some other row: nothing of them is stored */
    const uint32_t wst = (tid / C::WP) * C::WROW + wp * 16u, xst = (tid / C::XP) * C::XROW + xp * 16u;
    auto stage = [&](const W4Stage<C>& b, uint8_t* buf) {
        uint8_t* const xl = buf;
        uint8_t* const wl = buf + C::X_BYTES;
        float* const xs = (float*)(buf + C::X_BYTES + C::W_BYTES);
        typedef float __attribute__((ext_vector_type(C::XL))) xsum_t; /* (an array's selects become scratch memory) */
        xsum_t xsum = {};
#pragma unroll
        for (int j = 0; j < C::WL; j++)
            *(v4i*)(wl + wst + j * WR * C::WROW) = b.w[j];
#pragma unroll
        for (int j = 0; j < C::XL; j++) {
            *(v4i*)(xl + xst + j * XR * C::XROW) = w4_order(b.x[j]);
            float v = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) v = w4_dot2((uint32_t)b.x[j][i], 0x3F803F80u, v);
            xsum[j] = w4_run_sum<G / 8>(v);
        }
        /* the lanes of a group's run hold the same sum: lane j of the run stores that of row j */
        constexpr int RUN = G / 8 < C::XL ? G / 8 : C::XL;
#pragma unroll
        for (int j0 = 0; j0 < C::XL; j0 += RUN) {
            float v = xsum[j0];
            uint32_t mine = xp % (G / 8);
#pragma unroll
            for (int j = 1; j < RUN; j++) v = mine == (uint32_t)j ? xsum[j0 + j] : v;
            if (RUN == G / 8 || mine < RUN) xs[(xp / (G / 8)) * C::TM + tid / C::XP + (j0 + mine) * XR] = C::ASYM ? -v : -24.0f * v;
        }
    };
    /* columns behind K count as zero; the walk calls this for the step that has some */
    auto cut = [&](W4Stage<C>& b, uint32_t step) {
        if (step * KS + xp * 8u < K) return;
#pragma unroll
        for (int j = 0; j < C::XL; j++) b.x[j] = (v4i){0, 0, 0, 0};
    };

    const W4Bits bits = w4_bits();
    v4f acc[NS][C::NBW][C::MTW] = {};
    /* Instruction by instruction over all of the wave's tiles: 16 sums grow side by side, none waits for the one before
     * it, and x is read as it is needed. (Tile by tile, a group's instructions after one another: 2048 x 4096 x 7168 142 us
     * for 133.) */
    constexpr int TILES = NS * C::NBW;
    auto multiply = [&](const uint8_t* buf, const uint8_t* sbuf, uint32_t g0) { /* g0: the step's first group in its chunk */
        const uint8_t* const xl = buf + (wt * C::MTW * 16u + c) * C::XROW;
        const uint8_t* const wl = buf + C::X_BYTES;
        const float* const xs = (const float*)(buf + C::X_BYTES + C::W_BYTES) + wt * C::MTW * 16u + 4u * q;
        const uint8_t* const sl = sbuf + (wc * C::NBW * 16u + c) * C::SROW + g0 * 2u;
        const uint8_t* const zl = sbuf + C::S_BYTES + (wc * C::NBW * 16u + c) * C::ZROW + g0;
#pragma unroll
        for (int blk = 0; blk < KS / 128; blk++) {
            uint32_t raw[TILES][4]; /* a lane's 32 weights of each 16 channels */
#pragma unroll
            for (int i = 0; i < TILES; i++) {
                const v4i w = *(const v4i*)(wl + ((i / C::NBW) * C::TN + wc * C::NBW * 16u + (i % C::NBW) * 16u + c) * C::WROW + blk * 64u + q * 16u);
#pragma unroll
                for (int k = 0; k < 4; k++) raw[i][k] = (uint32_t)w[k];
                w4_deal<G>(raw[i]);
            }
            constexpr int RG = G / 32; /* instructions per group */
#pragma unroll
            for (int gr = 0; gr < 128 / G; gr++) {
                const int gi = blk * (128 / G) + gr;
                v4f cx[C::MTW], t[TILES][C::MTW];
#pragma unroll
                for (int mt = 0; mt < C::MTW; mt++) cx[mt] = *(const v4f*)(xs + gi * C::TM + mt * 16);
#pragma unroll
                for (int r = 0; r < RG; r++) {
                    const int at = gr * RG + r;
                    v8bf a[C::MTW];
#pragma unroll
                    for (int mt = 0; mt < C::MTW; mt++) a[mt] = *(const v8bf*)(xl + mt * 16 * C::XROW + (blk * 128u + w4_koff<G>(q, at)) * 2u);
#pragma unroll
                    for (int i = 0; i < TILES; i++) {
                        const v8bf b = w4_unpack(raw[i][at], bits);
                        float zc = 0.0f;
                        if (C::ASYM && r == 0) zc = 16.0f + (float)zl[((i / C::NBW) * C::TN + (i % C::NBW) * 16) * C::ZROW + gi];
#pragma unroll
                        for (int mt = 0; mt < C::MTW; mt++) {
                            v4f from = r ? t[i][mt] : cx[mt];
                            if (C::ASYM && r == 0) {
#pragma unroll
                                for (int k = 0; k < 4; k++) from[k] *= zc;
                            }
                            t[i][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[mt], b, from, 0, 0, 0);
                        }
                    }
                    /* Whether reads may move up over an instruction's products, in the four-wave forms (the eight-wave forms
                     * let them; their groups of 32 take 239 us for 218 without). us let / held back, for 64 rows of 7168 x
                     * 7168, a GLU of 64 rows of 4096 x 7168, and 512 and 2048 tokens over 64 experts of 2048 x 1408, top 6:
                     *   G 32     37.9 38.3   31.4 32.7   285 305   818 878     zero points  37.3 37.3   41.5 42.1   366 373   1085 1126
                     *   G 64     32.3 32.4   28.3 28.3   256 259   716 728     zero points  33.9 32.9   32.1 31.1   304 298    845  825
                     *   G 128    31.2 27.8   28.7 27.4   189 184   482 454     zero points  30.8 29.1   29.0 28.4   270 261    756  733
                     * G 128 without zero points is best with the GLU's let and the plain product's held back (175 and 458). */
                    if (C::WT == 1 && (C::ASYM ? G != 32 : G == 128 && NS == 1)) __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int i = 0; i < TILES; i++) {
                    const float sc = w4_f32(*(const uint16_t*)(sl + ((i / C::NBW) * C::TN + (i % C::NBW) * 16) * C::SROW + gi * 2), g.s_f16);
#pragma unroll
                    for (int mt = 0; mt < C::MTW; mt++)
#pragma unroll
                        for (int k = 0; k < 4; k++) acc[i / C::NBW][i % C::NBW][mt][k] = fmaf(t[i][mt][k], sc, acc[i / C::NBW][i % C::NBW][mt][k]);
                }
            }
        }
    };

    /* ---- the walk over K: the next step is on its way in registers, two LDS buffers ---- */
    W4Stage<C> ring;
    W4Scales<C> sring;
    load_scales(sring, s_lo);
    load(ring, s_lo);
    for (uint32_t s = s_lo; s < s_hi; s++) { /* (slices are not empty) */
        const uint32_t n = s - s_lo;
        uint8_t* const buf = lds + (n & 1u) * C::BUF;
        uint8_t* const sbuf = lds + 2 * C::BUF + ((n / C::CS) & 1u) * C::SBUF;
        if ((s + 1u) * KS > K) cut(ring, s);
        stage(ring, buf);
        if (n % C::CS == 0u) {
            stage_scales(sring, sbuf);
            if (s + C::CS < s_hi) load_scales(sring, s + C::CS);
        }
        load(ring, s + 1u);
        /* a buffer is written again two steps (chunks) later: its readers passed the barrier in between */
        lds_barrier();
        multiply(buf, sbuf, (n % C::CS) * C::GS);
    }

    /* ---- results: lane holds channel c of each 16, rows 4 q + i ---- */
#pragma unroll
    for (int mt = 0; mt < C::MTW; mt++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t t = rb + (wt * C::MTW + mt) * 16u + 4u * q + i;
            if (t >= cnt) continue;
            if (tl.slices) {
#pragma unroll
                for (int st = 0; st < NS; st++)
#pragma unroll
                    for (int nb = 0; nb < C::NBW; nb++) {
                        const uint32_t n = n0 + (wc * C::NBW + nb) * 16u + c;
                        if (n < N) tl.part[(((size_t)slice * NS + st) * g.M + t) * N + n] = acc[st][nb][mt][i];
                    }
                continue;
            }
            const uint32_t r = r0 + t, oi = g.o_idx ? g.o_idx[r] : r;
            if (oi == PLOW_EXPERT_UNUSED || (g.a_idx && g.a_idx[r] == PLOW_EXPERT_UNUSED)) continue;
            const float gate = g.gate ? g.gate[r] : 1.0f;
#pragma unroll
            for (int nb = 0; nb < C::NBW; nb++) {
                const uint32_t n = n0 + (wc * C::NBW + nb) * 16u + c;
                if (n >= N) continue;
                const float v = NS == 2 ? moe_glu(acc[0][nb][mt][i], acc[NS - 1][nb][mt][i], g.act, g.f0, g.f1) : gate * acc[0][nb][mt][i];
                if (NS == 1 && g.out_f32) ((float*)g.out)[(size_t)oi * g.ldo + n] = v;
                else ((bf16_t*)g.out)[(size_t)oi * g.ldo + n] = f2bf(v);
            }
        }
}

/* grid: x = channel tiles, y = row tiles (routed experts: over all of them, from gridDim.y on the workgroups take
 * another), z = K slice. CHOICE: routed experts behind a choice made on the device */
template <class C, bool CHOICE>
__global__ __launch_bounds__(C::THREADS, 2) void k_w4_tile(GroupW4 g, W4Tiles tl) {
    extern __shared__ __attribute__((aligned(16))) uint8_t w4_lds[];
    constexpr bool EXPERTS = C::TM == (int)PLOW_MPF_BM; /* meta counts tiles of that many rows */
    const bool routed = EXPERTS && g.meta;
    if (CHOICE && !w4_chosen(g, 1u)) return;
    const int32_t* const tilep = g.meta + 2u * g.E;
    const uint32_t n0 = blockIdx.x * C::TN, lane = threadIdx.x & 63u, total = routed ? (uint32_t)tilep[g.E] : gridDim.y;
    uint32_t e = 0u, r0 = 0u, cnt = g.M;
    for (uint32_t want = blockIdx.y; want < total; want += gridDim.y) {
        uint32_t rb = want * C::TM;
        if (routed) { /* the expert whose tiles reach past `want` first */
            e = g.E;
            for (uint32_t e0 = 0; e0 < g.E && e == g.E; e0 += WAVE) {
                const uint32_t next = e0 + lane + 1u;
                const unsigned long long m = __ballot((uint32_t)tilep[next < g.E ? next : g.E] > want);
                if (m) e = e0 + (uint32_t)__ffsll(m) - 1u; /* (tilep[E] is total) */
            }
            if (e >= g.E) return;
            rb = (want - (uint32_t)tilep[e]) * C::TM, cnt = (uint32_t)g.meta[g.E + e], r0 = (uint32_t)g.meta[e];
            bool here = rb < cnt;
            for (int st = 0; st < C::NS; st++) {
                const size_t at = (size_t)e * 3u + g.sel[st];
                here = here && g.wtab[at] && g.stab[at] && (!C::ASYM || g.ztab[at]);
            }
            if (!here) continue; /* not resident */
        }
        w4_tile<C>(g, tl, w4_lds, e, r0, cnt, rb, n0, blockIdx.z);
        lds_barrier(); /* the next tile's first step may write the buffer that a slower wave still reads */
    }
}

/* workgroups of the kernel that a CU holds, asked once */
template <class C>
static int w4_per_cu = 1;

template <class C>
static bool w4_setup() {
    const void* const k = (const void*)k_w4_tile<C, false>;
    if constexpr (C::TM == (int)PLOW_MPF_BM) {
        if (hipFuncSetAttribute((const void*)k_w4_tile<C, true>, hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS) != hipSuccess) return false;
    }
    return hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS) == hipSuccess &&
           hipOccupancyMaxActiveBlocksPerMultiprocessor(&w4_per_cu<C>, k, C::THREADS, C::LDS) == hipSuccess && w4_per_cu<C> > 0;
}
#endif
