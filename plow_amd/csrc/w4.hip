/* w4.hip — products with 4-bit integer weights and group scales: dense (GEMM_W4, GEMM_GLU_W4) and routed experts
 * (ops 48 / 49 and 85 / 86 at enc 16). Dispatch between the kernel forms, and the matrix-vector form.
 *
 *   out[m][n] = sum over groups g of s[n][g] * sum_{k in g} x[m][k] * (q[n][k] - z[n][g])
 *
 * GLU: bf16(act(gate) * up) of two such sums; DOWN of routed experts: gate_r * sum as f32. */
#include "common.h"
#include "kernels.h"
#include "tuning.h"
#include "w4_forms.h"
#include "w4_tile.h"

/* whether expert e can be served for stream column `sel` */
__device__ __forceinline__ bool w4_resident(const GroupW4& g, uint32_t e, uint32_t sel) {
    const size_t at = (size_t)e * 3u + sel;
    return g.wtab[at] && g.stab[at] && (!g.ztab || g.ztab[at]);
}

/* slot-major DOWN: the f32 rows of slots that no expert serves (sentinel id, expert not resident) are zero */
__global__ __launch_bounds__(256) void k_w4_zero_unserved(GroupW4 g) {
    const uint32_t e = ((const PlowMoeRoute*)g.tab)[blockIdx.x].eid;
    if (e < g.E && w4_resident(g, e, g.sel[0])) return;
    for (uint32_t n = threadIdx.x; n < g.N; n += 256u) ((float*)g.out)[blockIdx.x * g.ldo + n] = 0.0f;
}

/* ---- matrix-vector form: one row of x (the dense ops at one token, a routing slot) --------------------------
 *
 * A wave keeps its row of x in registers, 32 columns per lane and piece, already in the order in which the nibbles of a
 * dword come out (w4_unpack), and walks a run of weight rows four at a time (GLU: gate and up of two channels): every
 * lane loads 16 bytes of each row per 1 KB, the next four rows' loads are issued before these are multiplied, two bit
 * operations and one v_dot2_f32_bf16 per two weights. A lane's 32 columns lie in one group: the dot product starts
 * from -(16 + z) * (their sum of x), which takes the 16 + z off again, and is scaled once. The four rows' sums meet in
 * a reduction of ten instructions: two cross-lane swaps leave one row per 16 lanes.
 *
 * The weight stream bounds it: 120001 x 4096, G = 64, takes 45 us = 5.8 TB/s; eight of 384 experts of 7168 x 2048,
 * G = 32, 49 us for gate, up, down and the combine = 4.1 TB/s, a walk of few rows per wave; 2048 x 2816 takes 4.3 us,
 * little more than a launch. Four rows at a time: two leave too few loads in flight, eight do not fit the
 * registers at K = 7168. */
#define V_WAVES 4u

template <int ITER, bool GLU, bool ASYM>
struct VecRows { /* four weight rows' share of a lane */
    v4i w[4][ITER];
    uint16_t s[4][ITER];
    uint8_t z[4][ASYM ? ITER : 1];
};

template <int ITER, bool GLU, bool ASYM>
__global__ __launch_bounds__(V_WAVES* WAVE) void k_w4_vec(GroupW4 g, uint32_t chunks) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t unit = (uint32_t)__builtin_amdgcn_readfirstlane((int)(blockIdx.x * V_WAVES + (threadIdx.x >> 6)));
    const uint32_t row = unit / chunks, chunk = unit % chunks;
    const uint32_t N = g.N, K = g.K;
    constexpr uint32_t NC = GLU ? 2u : 4u; /* channels per four rows */
    if (row >= (g.tab ? g.nslot : g.M)) return;
    const uint32_t q_all = (N + NC - 1u) / NC; /* (at most as many chunks as that) */
    const uint32_t q_lo = (uint32_t)((uint64_t)q_all * chunk / chunks), q_hi = (uint32_t)((uint64_t)q_all * (chunk + 1u) / chunks);

    const void *w[2] = {g.w[0], g.w[1]}, *s[2] = {g.s[0], g.s[1]}, *z[2] = {g.z[0], g.z[1]};
    float gate = 1.0f;
    uint32_t xrow = row;
    if (g.tab) {
        const PlowMoeRoute rt = ((const PlowMoeRoute*)g.tab)[row];
        bool ok = rt.eid < g.E;
        for (uint32_t j = 0; ok && j < (GLU ? 2u : 1u); j++) {
            const size_t at = (size_t)rt.eid * 3u + g.sel[j];
            w[j] = (const void*)(uintptr_t)g.wtab[at], s[j] = (const void*)(uintptr_t)g.stab[at];
            z[j] = ASYM ? (const void*)(uintptr_t)g.ztab[at] : nullptr;
            ok = w[j] && s[j] && (!ASYM || z[j]);
        }
        if (!ok) { /* no expert serves the slot: DOWN's rows are zero, GLU's stay */
            if (!GLU)
                for (uint32_t n = q_lo * NC + lane; n < q_hi * NC && n < N; n += WAVE) ((float*)g.out)[(size_t)row * g.ldo + n] = 0.0f;
            return;
        }
        if (GLU) xrow = row / g.kx;
        else gate = rt.gate;
    }

    const uint32_t pieces = K / 32u, KG = K / g.G, gshift = g.G == 32u ? 0u : g.G == 64u ? 1u : 2u;
    typedef const __attribute__((address_space(1))) uint8_t* gptr; /* global memory: a pointer out of a table is generic to the compiler */
    auto load = [&](VecRows<ITER, GLU, ASYM>& b, uint32_t quad) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int st = GLU ? r & 1 : 0;
            uint32_t ch = quad * NC + (uint32_t)(GLU ? r >> 1 : r);
            ch = ch < N ? ch : N - 1u;
            const gptr wr = (gptr)w[st] + (size_t)ch * (K / 2u), sr = (gptr)s[st] + (size_t)ch * KG * 2u, zr = (gptr)z[st] + (ASYM ? (size_t)ch * KG : 0u);
#pragma unroll
            for (int it = 0; it < ITER; it++) {
                const uint32_t p = (uint32_t)it * 64u + lane;
                const bool in = p < pieces;
                b.w[r][it] = in ? __builtin_nontemporal_load((const __attribute__((address_space(1))) v4i*)(wr + (size_t)p * 16u)) : (v4i){0, 0, 0, 0};
                b.s[r][it] = in ? *(const __attribute__((address_space(1))) uint16_t*)(sr + (p >> gshift) * 2u) : (uint16_t)0;
                if (ASYM) b.z[r][it] = in ? zr[p >> gshift] : (uint8_t)0;
            }
        }
    };
    VecRows<ITER, GLU, ASYM> ring[2];
    load(ring[0], q_lo);

    v4i x[ITER][4];
    float xs[ITER]; /* -24 (or, with zero points, -1) times the piece's sum of x */
    const uint8_t* const xsrc = (const uint8_t*)g.x + (size_t)xrow * g.ldx * 2u;
#pragma unroll
    for (int it = 0; it < ITER; it++) {
        const uint32_t p = (uint32_t)it * 64u + lane;
        float v = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const v4i t = p < pieces ? *(const v4i*)(xsrc + (size_t)p * 64u + j * 16u) : (v4i){0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 4; i++) v = w4_dot2((uint32_t)t[i], 0x3F803F80u, v);
            x[it][j] = w4_order(t);
        }
        xs[it] = ASYM ? -v : -24.0f * v;
    }

    const W4Bits bits = w4_bits();
    auto finish = [&](const VecRows<ITER, GLU, ASYM>& b, uint32_t quad) {
        float sum[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            float acc = 0.0f;
#pragma unroll
            for (int it = 0; it < ITER; it++) {
                float t = ASYM ? (16.0f + (float)b.z[r][it]) * xs[it] : xs[it];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const v4i u = __builtin_bit_cast(v4i, w4_unpack((uint32_t)b.w[r][it][j], bits));
#pragma unroll
                    for (int i = 0; i < 4; i++) t = w4_dot2((uint32_t)u[i], (uint32_t)x[it][j][i], t);
                }
                acc = fmaf(t, w4_f32(b.s[r][it], g.s_f16), acc);
            }
            sum[r] = acc;
        }
        /* lanes 0-31 hold row 0 (1), lanes 32-63 row 2 (3); then 16 lanes per row */
        float h[2];
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum[r]), __float_as_uint(sum[r + 2]), false, false);
            h[r] = __uint_as_float(p[0]) + __uint_as_float(p[1]);
        }
        const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(h[0]), __float_as_uint(h[1]), false, false);
        const float v = w4_run_sum<16>(__uint_as_float(p[0]) + __uint_as_float(p[1]));
        const uint32_t r = lane >> 4;
        const float other = GLU ? __shfl_xor(v, 16, 64) : 0.0f;
        const uint32_t ch = quad * NC + (GLU ? r >> 1 : r);
        if ((lane & 15u) == 0u && (!GLU || !(r & 1u)) && ch < N) {
            const float res = GLU ? moe_glu(v, other, g.act, g.f0, g.f1) : gate * v;
            if (!GLU && g.out_f32) ((float*)g.out)[(size_t)row * g.ldo + ch] = res;
            else ((bf16_t*)g.out)[(size_t)row * g.ldo + ch] = f2bf(res);
        }
    };
    for (uint32_t quad = q_lo;;) {
        if (quad + 1u < q_hi) load(ring[1], quad + 1u);
        finish(ring[0], quad);
        if (++quad >= q_hi) break;
        if (quad + 1u < q_hi) load(ring[0], quad + 1u);
        finish(ring[1], quad);
        if (++quad >= q_hi) break;
    }
}

/* a lane holds its share of the row: 64 registers at 8192 columns. Longer rows run as a tile of 16 with K split: 4096 x
 * 8192, G = 128, takes 7.3 us here, 4096 x 11008 13.4 us and 4096 x 14336 15.1 us there (2 TB/s; two launches), 7168 x
 * 18432, G = 32, 22.8 us, 8192 x 28672 30.8 us (3.9 TB/s) */
#define W4_VEC_MAX_K 8192u
/* Which calls take the matrix-vector form: one dense row, or a few routing slots, each of which streams its expert's
 * weights by itself (and needs no sort). Measured against the tiles of 16 rows: dense 120001 x 4096 45 us for 58, 2048 x
 * 2816 6.4 for 8.8, 7168 x 7168 10.2 for 12.3 (two rows, one after the other: 86 for 60, 6.4 for 8.8, 17.8 for 12.7).
 * Slots: GLU and DOWN of random routing in us, matrix-vector / tiles (rows of experts, top 2 to 8):
 *                     4096 x 1536, G 128                        7168 x 2048, G 32                       2048 x 1408, G 64
 *   E       16 slots 24      32       48      64   |  16       24       32       48       64   |  16     24     32     48     64
 *     1,2    32/93  46/93   56/93   82/99 101/99   | 71/200 117/200  127/203  206/208  238/208 | 20/76  30/76  32/76  51/81  54/80
 *     4      33/51  47/51   56/52   84/53 102/57   | 70/102 117/102  127/103  207/104  245/109 | 20/41  30/41  32/41  51/42  55/45
 *     8      35/45  49/46   56/47   85/48 104/48   | 74/85  116/86   131/88   215/89   251/89  | 21/37  30/38  32/38  50/38  55/39
 *    16      37/53  49/55   58/56   87/58 105/58   | 78/102 116/106  137/117  214/120  256/121 | 22/41  31/42  33/43  50/43  55/44
 *    32      38/60  47/63   61/65   83/67 112/79   | 79/127 116/139  140/143  215/156  263/195 | 22/48  30/50  34/51  50/53  58/54
 *    64      37/60  51/62   63/74   86/95 113/109  | 81/131 117/142  144/194  214/222  271/240 | 22/49  30/50  34/52  49/63  59/66
 *   128      37/60  49/63   61/87   90/107 116/121 | 83/132 117/151  147/200  219/261  278/302 | 21/50  29/51  33/52  47/72  60/75
 * The more slots share an expert, the sooner the tiles win, which read it once: from 20 slots and one more per two
 * experts on (never past 64: 128 slots over 128 experts of 4096 x 1536 227 us for 194; of two experts the tiles have too
 * few workgroups to win below that). Off the best by up to a third around 24 slots of 8 experts, to either side. */
#define W4_VEC_MAX_SLOTS 64u

bool w4_vec_serves(const GroupW4& g) {
    if (g.K > W4_VEC_MAX_K || g.meta) return false;
    if (!g.tab) return g.M == 1u;
    return g.nslot <= W4_VEC_MAX_SLOTS && (g.E <= 2u || g.nslot <= 20u + g.E / 2u);
}

template <int ITER, bool GLU>
static int launch_vec(const GroupW4& g, uint32_t n_cu, hipStream_t st) {
    const uint32_t rows = g.tab ? g.nslot : g.M, NC = GLU ? 2u : 4u;
    const uint64_t quads = ((uint64_t)g.N + NC - 1u) / NC;
    /* One set of waves walks it all, as many a CU as have enough in flight (4, 8 and 16 KB each, by the row's length):
     * more of them fetch x more often and walk too short a run. 8 of the longest rows' waves instead of 4: eight of 384
     * experts of 7168 x 2048 53 us for 50, 7168 x 7168 12.2 for 10.2; 8 and 16 of the middle ones instead of 12: 120001 x
     * 4096 47 and 48.5 us for 45; 8 of the shortest instead of 16: 32000 x 2048 9.7 us for 8.7. */
    const uint64_t waves = (uint64_t)n_cu * (ITER == 1 ? 16u : ITER == 2 ? 12u : 4u);
    /* never more than that set (ten slots of 385 experts of 7168 x 2048: 62 us, 76 with a few waves too many), in shares
     * that differ by one; where a share is one or two, in equal ones (14336 x 4096: 9.1 us, 11.1 unequal) */
    uint64_t chunks = waves / rows;
    if (chunks == 0) chunks = 1;
    if (chunks > quads) chunks = quads;
    const uint64_t most = (quads + chunks - 1u) / chunks;
    if (most <= 2u) chunks = (quads + most - 1u) / most;
    const uint32_t grid = (uint32_t)((chunks * rows + V_WAVES - 1u) / V_WAVES);
    if (g.z[0] || g.ztab) k_w4_vec<ITER, GLU, true><<<grid, V_WAVES * WAVE, 0, st>>>(g, (uint32_t)chunks);
    else k_w4_vec<ITER, GLU, false><<<grid, V_WAVES * WAVE, 0, st>>>(g, (uint32_t)chunks);
    return 0;
}

/* ---- tensors of fewer than 64 groups (W4_TINY_GROUPS), which the tiles' runs of scales do not fit: a thread per
 * output. At most 64 groups of weights: a launch's time whatever the form ---- */
__global__ __launch_bounds__(64) void k_w4_tiny(GroupW4 g, uint32_t glu) {
    const uint32_t n = blockIdx.x * 64u + threadIdx.x, e = blockIdx.y;
    if (n >= g.N || (g.meta && !(w4_resident(g, e, g.sel[0]) && (!glu || w4_resident(g, e, g.sel[1]))))) return;
    const uint32_t r0 = g.meta ? (uint32_t)g.meta[e] : 0u, cnt = g.meta ? (uint32_t)g.meta[g.E + e] : g.M;
    for (uint32_t r = r0 + blockIdx.z; r < r0 + cnt; r += gridDim.z) {
        const uint32_t ai = g.a_idx ? g.a_idx[r] : r, oi = g.o_idx ? g.o_idx[r] : r;
        if (ai == PLOW_EXPERT_UNUSED || oi == PLOW_EXPERT_UNUSED) continue;
        const bf16_t* const x = (const bf16_t*)g.x + (size_t)ai * g.ldx;
        float v[2];
        for (uint32_t st = 0; st < 1u + glu; st++) {
            const size_t at = (size_t)e * 3u + g.sel[st];
            const uint8_t* const w = (g.wtab ? (const uint8_t*)(uintptr_t)g.wtab[at] : (const uint8_t*)g.w[st]) + (size_t)n * (g.K / 2u);
            const uint16_t* const s = (g.wtab ? (const uint16_t*)(uintptr_t)g.stab[at] : (const uint16_t*)g.s[st]) + (size_t)n * (g.K / g.G);
            const uint8_t* z = g.wtab ? (g.ztab ? (const uint8_t*)(uintptr_t)g.ztab[at] : nullptr) : (const uint8_t*)g.z[st];
            float acc = 0.0f;
            for (uint32_t k0 = 0, gi = 0; k0 < g.K; k0 += g.G, gi++) {
                const float zf = z ? (float)z[(size_t)n * (g.K / g.G) + gi] : 8.0f;
                float t = 0.0f;
                for (uint32_t k = k0; k < k0 + g.G; k++) t = fmaf((float)((w[k / 2u] >> (4u * (k & 1u))) & 15u) - zf, bf2f(x[k]), t);
                acc = fmaf(t, w4_f32(s[gi], g.s_f16), acc);
            }
            v[st] = acc;
        }
        const float res = glu ? moe_glu(v[0], v[1], g.act, g.f0, g.f1) : (g.gate ? g.gate[r] : 1.0f) * v[0];
        if (g.out_f32) ((float*)g.out)[(size_t)oi * g.ldo + n] = res;
        else ((bf16_t*)g.out)[(size_t)oi * g.ldo + n] = f2bf(res);
    }
}

/* ---- K split: sum of the slices' partial results in slice order, through the activation for the GLU. Bound by the
 * partial sums' way from memory: 4 slices of 16 x 7168 take 3 us, 8 slices of 128 x 7168 (29 MB) 8.3 us ---- */
__global__ __launch_bounds__(256) void k_w4_join(GroupW4 g, const float* __restrict__ part, uint32_t slices, uint32_t glu) {
    const size_t plane = (size_t)g.M * g.N;
    for (size_t i = (size_t)blockIdx.x * 256u + threadIdx.x; i < plane; i += (size_t)gridDim.x * 256u) {
        float a = 0.0f, b = 0.0f;
        for (uint32_t s = 0; s < slices; s++) {
            a += part[(size_t)s * (1u + glu) * plane + i];
            if (glu) b += part[((size_t)s * 2u + 1u) * plane + i];
        }
        if (glu) a = moe_glu(a, b, g.act, g.f0, g.f1);
        const size_t m = i / g.N, at = m * g.ldo + (i - m * g.N);
        if (g.out_f32) ((float*)g.out)[at] = a;
        else ((bf16_t*)g.out)[at] = f2bf(a);
    }
}

/* How a matrix-unit call is cut: rows and channels of a tile, slices of K */
struct W4Plan {
    uint32_t tm, tn, nt, steps, slices, steps_per;
    bool few, wide;
    uint64_t ns;
};
static W4Plan w4_shape(const GroupW4& g, bool glu, uint32_t tm, uint32_t row_tiles, uint32_t n_cu) {
    W4Plan p = {};
    p.tm = tm, p.few = tm <= 32u;
    /* 32 channels per wave while that leaves every CU two workgroups: x is staged for twice the channels. 16 x 120001
     * x 4096 G = 64 takes 67 us so and 71 us with 16; 16 x 7168 x 7168, with too few tiles for it, 17 and 15. */
    const uint32_t tw = w4_rows_channels(glu, true);
    p.wide = (uint64_t)((g.N + tw - 1u) / tw) * row_tiles >= 2u * n_cu;
    p.tn = p.few ? w4_rows_channels(glu, p.wide) : w4_tiled_channels(glu);
    const uint32_t ks = p.few ? w4_rows_kstep() : w4_tiled_kstep();
    p.nt = (g.N + p.tn - 1u) / p.tn, p.steps = p.steps_per = (g.K + ks - 1u) / ks, p.slices = 1u;
    return p;
}
/* The time a dense call takes, counted: workgroups run in rounds of what the chip holds; one takes its steps and about
 * two more to start and end; slices of K cost their sums' way to memory and back and a second launch. A step of a
 * full chip was measured at 1.35 us (16 rows), 1.75 (32), 2.5 and 3.3 (the same with 32 weight rows a wave; a sixth
 * less up to two thirds full), 2.8 (64 rows; 2.2 where a CU holds one workgroup) and 2.5 (128 rows); the join at
 * 4 us and 1 us per 2.5 MB. Picks the slices that take the least; against none they have to win by a fifteenth, since
 * a call that streams weights at the memory's rate gains nothing from fuller rounds (16 x 120001 x 4096: 67 us, 73 in
 * two slices). 7168 x 7168 G = 128 without slices / with: 16 rows 28 / 16 us, 64 rows 108 / 28, 128 rows 137 / 34, 512
 * rows 138 / 75; with slices up to two workgroups a CU whatever fits / by this count: 33 rows 30 / 25, 96 rows 46 / 33 (16 rows lose:
 * 14.7 / 15.9). */
static W4Plan w4_dense_plan(const GroupW4& g, bool glu, uint32_t tm, uint32_t n_cu) {
    const uint32_t gy = (g.M + tm - 1u) / tm;
    W4Plan p = w4_shape(g, glu, tm, gy, n_cu);
    p.ns = ~0ull;
    if (gy > 65535u) return p; /* (the grid's limit; 128 rows always fit) */
    const uint32_t per_cu = (uint32_t)(p.few ? w4_rows_per_cu(g, glu, p.wide, tm) : w4_tiled_per_cu(g, glu, tm));
    const bool two = glu || p.wide;
    const uint64_t step = tm == 16u ? (two ? 2500u : 1350u) : tm == 32u ? (two ? 3300u : 1750u) : tm == 64u && per_cu > 1u ? 2800u : tm == 64u ? 2200u : 2500u;
    const uint64_t plane = (uint64_t)g.M * g.N * (glu ? 2u : 1u) * 4u, tiles = (uint64_t)p.nt * gy, cap = (uint64_t)n_cu * per_cu;
    const uint32_t steps = p.steps;
    for (uint32_t s = 1u; s == 1u || (s <= steps / 2u && s <= 128u && tiles * (s - 1u) < 2u * cap && g.ws && plane * s <= g.ws_bytes); s++) {
        const uint32_t per = (steps + s - 1u) / s, n = (steps + per - 1u) / per;
        const uint64_t one = p.few && tiles * n * 3u <= cap * 2u ? step * 5u / 6u : step;
        uint64_t ns = (tiles * n + cap - 1u) / cap * (per + 2u) * one;
        if (n > 1u) ns = (ns + 4000u + plane * n / 2500u) * 15u / 14u;
        if (ns < p.ns) p.ns = ns, p.slices = n, p.steps_per = per;
    }
    return p;
}

int launch_w4(const GroupW4& g, bool glu, hipStream_t st) {
    if (!g.N || !g.K || !g.E || !g.G || g.K % g.G) return PLOW_MOE_EINVAL;
    const uint32_t n_cu = plow_moe_n_cu();
    if (!n_cu) return PLOW_MOE_EDEVICE;
    if (w4_vec_serves(g)) {
        const uint32_t it = (g.K / 32u + 63u) / 64u;
        if (it <= 1u) return glu ? launch_vec<1, true>(g, n_cu, st) : launch_vec<1, false>(g, n_cu, st);
        if (it <= 2u) return glu ? launch_vec<2, true>(g, n_cu, st) : launch_vec<2, false>(g, n_cu, st);
        return glu ? launch_vec<4, true>(g, n_cu, st) : launch_vec<4, false>(g, n_cu, st);
    }
    if (g.wtab && !g.meta) return PLOW_MOE_EINVAL;
    if (g.zero_unserved) k_w4_zero_unserved<<<g.nslot, 256, 0, st>>>(g);

    if ((uint64_t)g.N * (g.K / g.G) < W4_TINY_GROUPS) {
        const uint32_t z = g.meta ? 16u : g.M < 65535u ? g.M : 65535u;
        k_w4_tiny<<<dim3((g.N + 63u) / 64u, g.E, z), 64, 0, st>>>(g, glu ? 1u : 0u);
        return 0;
    }
    if (g.meta && g.ws) {
        /* the rows are known to the device only: both sides of the rule below go out behind its count (tiles of 16 rows
         * up to 24 rows per expert on average, else of 64), and the one that it does not name returns at once. Ops one at
         * a time over 64 experts of 2048 x 1408, top 6, always tiles of 16 / so / with the count stated: 2048 tokens GLU
         * 496 / 266 / 281 us, DOWN 360 / 164 / 160; 512 tokens 158 / 102 / 103 and 105 / 76 / 73; one token, where the
         * count and the launch that returns are for nothing, 16 / 21 / 17 and 9 / 14 / 9. */
        int rc = launch_pick_form((uint32_t*)g.ws, g.meta, g.E, 24u * g.E + 1u, st);
        if (rc) return rc;
        W4Plan p = w4_shape(g, glu, 16u, 0u, n_cu);
        rc = w4_rows_launch(g, W4Tiles{}, glu, p.wide, p.tm, dim3(p.nt, g.E), st);
        if (rc) return rc;
        p = w4_shape(g, glu, 64u, 0u, n_cu);
        const uint32_t gy = (8u * n_cu + p.nt - 1u) / p.nt; /* (whatever it is, the workgroups walk all row tiles) */
        return w4_tiled_launch(g, W4Tiles{}, glu, p.tm, dim3(p.nt, gy), st);
    }
    W4Tiles tl = {};
    W4Plan p;
    uint64_t gy;
    if (!g.meta) {
        /* dense: the rows of a tile that take the least time by the count above (128 rows of 2048 x 2816, whose weights
         * stay in the cache: 16 rows a tile 13.6 us, 128 rows 16.2; of 7168 x 7168 58.7 and 34.7) */
        p = w4_dense_plan(g, glu, 16u, n_cu);
        for (uint32_t tm = 32u; tm <= 128u && tm / 2u < g.M; tm *= 2u) {
            const W4Plan o = w4_dense_plan(g, glu, tm, n_cu);
            if (o.ns < p.ns) p = o;
        }
        gy = ((uint64_t)g.M + p.tm - 1u) / p.tm;
        if (p.slices > 1u) tl.slices = p.slices, tl.steps_per = p.steps_per, tl.part = (float*)g.ws;
    } else {
        /* routed experts: by the rows of a hit expert on average. Some get more, and a second tile reads the weights
         * again, so that 64 rows pay from 24 on: 4096 x 1536 over 128 experts take 475 us (32 rows a tile) and 490
         * (64) at 24 rows on average, 626 and 508 at 32, 416 and 475 at 16. Tiles of 128 rows lose by what the last
         * one leaves empty: 2048 x 1408 over 64 experts 568 us for 554 at 240 rows, 1550 for 1493 at 768. */
        const uint32_t hit = g.slots < g.E ? g.slots : g.E;
        const uint32_t rows = g.slots ? (g.slots + hit - 1u) / hit : 1u;
        p = w4_shape(g, glu, rows <= 16u ? 16u : rows <= 24u ? 32u : 64u, hit, n_cu);
        gy = p.few ? g.E : (uint64_t)g.slots / p.tm + hit; /* (more row tiles than those there cannot be) */
        if (!p.few && gy > 65535u) gy = 65535u;
    }
    if (gy > 65535u) return PLOW_MOE_EINVAL;
    const dim3 grid(p.nt, (uint32_t)gy, tl.slices ? tl.slices : 1u);
    const int rc = p.few ? w4_rows_launch(g, tl, glu, p.wide, p.tm, grid, st) : w4_tiled_launch(g, tl, glu, p.tm, grid, st);
    if (rc || !tl.slices) return rc;
    const uint64_t blocks = ((uint64_t)g.M * g.N + 255u) / 256u;
    k_w4_join<<<(uint32_t)(blocks < 4096u ? blocks : 4096u), 256, 0, st>>>(g, tl.part, tl.slices, glu ? 1u : 0u);
    return 0;
}

int plow_moe_w4_setup() { return w4_rows_setup() && w4_tiled_setup() ? 0 : PLOW_MOE_EDEVICE; }
