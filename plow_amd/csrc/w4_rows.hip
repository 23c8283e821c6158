/* w4_rows.hip — int4 group-scale products of a few rows: tiles of 16 or 32 rows x 64 or 128 channels (GLU: gate and up
 * of 64), a wave per 32 weight rows. Operands, groups and scales as described in w4_tile.h; what differs is that the
 * weight stream sets the pace here:
 *   weights  a wave loads its own rows, 256 columns (a whole 128-byte line per row) a step, a step ahead in registers,
 *            from a base that is the same in all lanes plus 32-bit offsets; each 128-column half passes through a
 *            piece of LDS that only this wave uses, which turns "8 lanes a row" into the operand layout
 *   scales   the same way, 64 groups (a line per row) at a time
 *   x        shared by the waves, 512 columns at a time: two barriers per chunk, none per step, so that the waves of
 *            a CU drift apart and one's arithmetic hides another's loads; rows that are not there are not staged
 * Twelve waves a CU (three workgroups) in 168 registers: with eight of them, two steps ahead, 64 tokens over 128
 * experts (4096 x 1536, G = 128, zero points) took 325 us for 288, four steps ahead 555.
 *
 * What it reaches: those experts' gate and up 163 us for 843 MB (5.2 TB/s), their down, whose rows are short (6 steps),
 * 117 us for 421 MB (3.6 TB/s, the launch that zeroes the rows of padding included); 16 rows of 120001 x 4096, G = 64, 67
 * us for 261 MB (3.9 TB/s); 16 rows of 7168 x 2048, G = 32, where four slices of K and their join are all latency, 8.5 + 3
 * us. */
#include "w4_forms.h"
#include "w4_tile.h"

/* GLU: NS = 2, gate and up rows of 16 channels per wave; else NS sets of 16 channels per wave */
template <int MTW_, int NS_, bool GLU_, int G_, bool ASYM_>
struct RowsCfg {
    static constexpr bool GLU = GLU_;
    static constexpr int WC = 4, MTW = MTW_, NS = NS_, G = G_, D = 1, KS = 256, XC = 512;
    static constexpr bool ASYM = ASYM_;
    static constexpr int THREADS = WC * 64, TM = MTW * 16, TN = WC * 16 * (GLU ? 1 : NS), CS = XC / KS;
    static constexpr int XP = XC / 8, XL = TM * XP / THREADS, XROW = XC * 2 + 16;
    static constexpr int WROW = 80; /* 64 bytes of a row: 16 rows on different banks */
    /* scales of a run of RUN groups (a 128-byte line per weight row), kept in LDS as they come: pitches off the banks */
    static constexpr int RUN = 64, SROW = RUN * 2 + 4, ZROW = RUN + 4, CR = RUN * G / XC; /* chunks per run */
    static constexpr int X_BYTES = TM * XROW, XS_BYTES = (XC / G) * TM * 4, W_BYTES = NS * 16 * WROW, S_BYTES = NS * 16 * SROW, Z_BYTES = ASYM ? NS * 16 * ZROW : 0;
    static constexpr int WAVE_BYTES = W_BYTES + S_BYTES + Z_BYTES;
    static constexpr int LDS = X_BYTES + XS_BYTES + WC * WAVE_BYTES;
    static_assert(LDS <= 160 * 1024 && CS % D == 0 && TM * XP % THREADS == 0 && THREADS % XP == 0 && XP % (G / 8) == 0, "geometry");
    static_assert(W_BYTES % 16 == 0 && S_BYTES % 16 == 0 && Z_BYTES % 16 == 0 && XS_BYTES % 16 == 0, "aligned pieces");
};

typedef const __attribute__((address_space(1))) uint8_t* w4_gptr; /* global memory: a pointer out of a table is generic to the compiler */
typedef const __attribute__((address_space(1))) v4i* w4_gvec;

/* lanes of the wave exchange data through LDS here: nothing is emitted, but the compiler must not carry a value read
 * before over it, nor move a read into the lanes that wrote */
__device__ __forceinline__ void w4_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

template <class C>
__device__ __forceinline__ void w4_rows_tile(const GroupW4& g, const W4Tiles& tl, uint8_t* lds, uint32_t e, uint32_t r0, uint32_t cnt,
                                             uint32_t rb, uint32_t n0, uint32_t slice) {
    constexpr int G = C::G, NS = C::NS;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, c = lane & 15u, q = lane >> 4;
    const uint32_t wv = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
    const uint32_t K = g.K, N = g.N, KG = K / (uint32_t)G;
    const uint32_t steps = (K + C::KS - 1u) / C::KS;
    const uint32_t s_lo = tl.slices ? slice * tl.steps_per : 0u;
    const uint32_t s_hi = tl.slices ? (s_lo + tl.steps_per < steps ? s_lo + tl.steps_per : steps) : steps;
    const uint32_t k_end = s_hi * C::KS < K ? s_hi * C::KS : K;
    /* Workgroups start their walk at different chunks: all of them at column 0 would ask for lines a row pitch (a power
     * of two, often) apart at the same time, which lie on a few memory channels. */
    const uint32_t chunks = (s_hi - s_lo + C::CS - 1u) / C::CS, rot = (blockIdx.x + blockIdx.y) % chunks;
    auto chunk_step = [&](uint32_t j) -> uint32_t { /* first step of the j-th chunk of the walk */
        const uint32_t a = j + rot < chunks ? j + rot : j + rot - chunks;
        return s_lo + a * C::CS;
    };
    uint8_t* const xl = lds;
    float* const xs = (float*)(lds + C::X_BYTES);
    uint8_t* const wl = lds + C::X_BYTES + C::XS_BYTES + wv * C::WAVE_BYTES;
    uint8_t* const sl = wl + C::W_BYTES;
    uint8_t* const zl = sl + C::S_BYTES;

    /* ---- this wave's 16 channels: one base per stream, lane offsets inside the 16 rows ---- */
    uint32_t ch0[NS], last[NS]; /* rows past the last one read it again */
    w4_gptr wb[NS], sb[NS], zb[NS];
#pragma unroll
    for (int st = 0; st < NS; st++) {
        const int ts = C::GLU ? st : 0;
        const uint32_t ch = n0 + (C::GLU ? wv * 16u : (wv * NS + st) * 16u);
        ch0[st] = ch < N ? ch : N - 1u, last[st] = N - 1u - ch0[st];
        const size_t at = (size_t)e * 3u + g.sel[ts];
        wb[st] = (w4_gptr)(g.wtab ? (const uint8_t*)(uintptr_t)g.wtab[at] : (const uint8_t*)g.w[ts]) + (size_t)ch0[st] * (K / 2u);
        sb[st] = (w4_gptr)(g.wtab ? (const uint8_t*)(uintptr_t)g.stab[at] : (const uint8_t*)g.s[ts]) ; /* (runs are counted from the tensor's start) */
        zb[st] = C::ASYM ? (w4_gptr)(g.wtab ? (const uint8_t*)(uintptr_t)g.ztab[at] : (const uint8_t*)g.z[ts]) : nullptr;
    }
    const uint32_t wr = lane >> 3, wp = lane & 7u;
    uint32_t wrow[NS][2];
#pragma unroll
    for (int st = 0; st < NS; st++)
#pragma unroll
        for (uint32_t h = 0; h < 2u; h++) {
            const uint32_t r = h * 8u + wr;
            wrow[st][h] = (r < last[st] ? r : last[st]) * (K / 2u);
        }
    struct Step {
        v4i w[NS][2];
    } ring[C::D];
    /* No load of the walk stands under a condition, so that the compiler can count what is in flight and waits for a
     * step's own loads only: a step past the end is the last one again, a piece past the end of a row the row's last. */
    auto load_w = [&](Step& b, uint32_t s) {
        s = s < s_hi ? s : s_hi - 1u;
        uint32_t at = s * (C::KS / 2) + wp * 16u;
        at = at < K / 2u - 16u ? at : K / 2u - 16u;
#pragma unroll
        for (int st = 0; st < NS; st++)
#pragma unroll
            for (int h = 0; h < 2; h++) b.w[st][h] = *(w4_gvec)(wb[st] + (wrow[st][h] + at));
    };
    auto stage_w = [&](const Step& b, uint32_t blk) { /* the 128-column half blk */
        w4_wave_sync();
        if ((wp >> 2) == blk) {
#pragma unroll
            for (int st = 0; st < NS; st++)
#pragma unroll
                for (int h = 0; h < 2; h++) *(v4i*)(wl + (st * 16 + h * 8 + wr) * C::WROW + (wp & 3u) * 16u) = b.w[st][h];
        }
        w4_wave_sync();
    };

    /* ---- scales and zero points, a run of RUN groups at a time: whole lines. (Read chunk by chunk, 8 or 16 bytes of a
     * row each, they made a third of all requests: 16 rows of 120001 x 4096, G = 64, 77 us.) A run that would leave the
     * tensor starts earlier; the tensor holds one run at least (W4_TINY_GROUPS). */
    const size_t all_groups = (size_t)N * KG;
    const uint32_t g_lo = s_lo * (C::KS / G); /* runs are counted from the slice's first group */
    auto channel = [&](uint32_t row) -> uint32_t { /* of weight row `row` of the wave's NS * 16 */
        const int st = NS == 2 && row >= 16u ? NS - 1 : 0;
        const uint32_t r = row % 16u, l = st ? last[NS - 1] : last[0];
        return (st ? ch0[NS - 1] : ch0[0]) + (r < l ? r : l);
    };
    auto run_start = [&](uint32_t ch, uint32_t run) -> size_t {
        const size_t at = (size_t)ch * KG + g_lo + run * C::RUN, end = all_groups - C::RUN;
        return at < end ? at : end;
    };
    uint32_t soff[NS]; /* where the run's first group stands in this lane's channel's row */
    /* (bytes: they are read back as 16-bit scales and 8-bit zero points) */
    auto put4 = [](uint8_t* p, int v) { __builtin_memcpy(__builtin_assume_aligned(p, 4), &v, 4); };
    auto stage_run = [&](uint32_t run) {
        v4i sv[2 * NS], zv[C::ASYM ? NS : 1];
        const uint32_t left = KG - g_lo - run * C::RUN, run_groups = left < (uint32_t)C::RUN ? left : (uint32_t)C::RUN;
        /* (a run that starts earlier than its row asks for groups further on in it) */
#pragma unroll
        for (int it = 0; it < 2 * NS; it++) {
            const uint32_t ch = channel(it * 8u + (lane >> 3));
            const size_t at = run_start(ch, run);
            const uint32_t need = run_groups + (uint32_t)((size_t)ch * KG + g_lo + run * C::RUN - at);
            sv[it] = (v4i){0, 0, 0, 0};
            if ((lane & 7u) * 8u < need) __builtin_memcpy(&sv[it], (const uint8_t*)((it >= 2 ? sb[NS - 1] : sb[0]) + at * 2u + (lane & 7u) * 16u), 16);
        }
        if (C::ASYM) {
#pragma unroll
            for (int it = 0; it < NS; it++)
                __builtin_memcpy(&zv[it], (const uint8_t*)((it ? zb[NS - 1] : zb[0]) + run_start(channel(it * 16u + (lane >> 2)), run) + (lane & 3u) * 16u), 16);
        }
        w4_wave_sync();
#pragma unroll
        for (int it = 0; it < 2 * NS; it++)
#pragma unroll
            for (int i = 0; i < 4; i++) put4(sl + (it * 8 + (lane >> 3)) * C::SROW + (lane & 7u) * 16u + i * 4, sv[it][i]);
        if (C::ASYM) {
#pragma unroll
            for (int it = 0; it < NS; it++)
#pragma unroll
                for (int i = 0; i < 4; i++) put4(zl + (it * 16 + (lane >> 2)) * C::ZROW + (lane & 3u) * 16u + i * 4, zv[it][i]);
        }
        w4_wave_sync();
#pragma unroll
        for (int st = 0; st < NS; st++) {
            const uint32_t ch = channel(st * 16u + c);
            soff[st] = (uint32_t)((size_t)ch * KG + g_lo + run * C::RUN - run_start(ch, run));
        }
    };

    /* ---- a chunk of x ---- */
    const uint8_t* xsrc[C::XL];
    bool xok[C::XL];
    const uint32_t xp = tid % C::XP;
#pragma unroll
    for (int j = 0; j < C::XL; j++) {
        const uint32_t t = rb + (tid + (uint32_t)j * C::THREADS) / C::XP;
        uint32_t ai = PLOW_EXPERT_UNUSED;
        if (t < cnt) ai = g.a_idx ? g.a_idx[r0 + t] : r0 + t;
        xok[j] = ai != PLOW_EXPERT_UNUSED;
        xsrc[j] = (const uint8_t*)g.x + (size_t)(xok[j] ? ai : 0u) * g.ldx * 2u; /* (row 0 is there: dense rows, or a token) */
    }
    v4i xr[C::XL];
    uint32_t xk; /* the loaded piece's column; from K on it counts as zero */
    auto load_x = [&](uint32_t s) {
        const uint32_t k = s * C::KS + xp * 8u, at = k < K - 8u ? k : K - 8u;
        xk = k;
#pragma unroll
        for (int j = 0; j < C::XL; j++) xr[j] = *(const v4i*)(xsrc[j] + (size_t)at * 2u);
    };
    auto stage_x = [&]() {
#pragma unroll
        for (int j = 0; j < C::XL; j++) {
            const uint32_t t = (tid + j * C::THREADS) / C::XP;
            if (C::XP % 64 == 0 && rb + (uint32_t)__builtin_amdgcn_readfirstlane((int)t) >= cnt) continue; /* a wave's pieces are of one row: none, and its results are dropped */
            const v4i xv = xok[j] && xk < K ? xr[j] : (v4i){0, 0, 0, 0};
            *(v4i*)(xl + t * C::XROW + xp * 16u) = w4_order(xv);
            float v = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) v = w4_dot2((uint32_t)xv[i], 0x3F803F80u, v);
            v = w4_run_sum<G / 8>(v);
            if (xp % (G / 8) == 0u) xs[(xp / (G / 8)) * C::TM + t] = C::ASYM ? -v : -24.0f * v;
        }
    };

    const W4Bits bits = w4_bits();
    v4f acc[NS][C::MTW] = {};
    auto multiply = [&](uint32_t kc, uint32_t k0) { /* kc: the 128-column block in the chunk, from column k0 on */
        constexpr int RG = G / 32;
        uint32_t raw[NS][4];
#pragma unroll
        for (int st = 0; st < NS; st++) {
            const v4i w = *(const v4i*)(wl + (st * 16 + c) * C::WROW + q * 16u);
#pragma unroll
            for (int i = 0; i < 4; i++) raw[st][i] = (uint32_t)w[i];
            w4_deal<G>(raw[st]);
        }
#pragma unroll
        for (int gr = 0; gr < 128 / G; gr++) {
            const uint32_t gi = kc * (128 / G) + gr, gs = (k0 / G - g_lo + gr) % C::RUN; /* the group in the chunk, in the run */
            if (k0 + gr * G < k_end) { /* the same in every lane */
            v8bf b[NS][RG];
            float s[NS], zc[NS];
#pragma unroll
            for (int st = 0; st < NS; st++) {
                s[st] = w4_f32(*(const uint16_t*)(sl + (st * 16 + c) * C::SROW + (gs + soff[st]) * 2u), g.s_f16);
                zc[st] = C::ASYM ? 16.0f + (float)zl[(st * 16 + c) * C::ZROW + gs + soff[st]] : 0.0f;
#pragma unroll
                for (int r = 0; r < RG; r++) b[st][r] = w4_unpack(raw[st][gr * RG + r], bits);
            }
#pragma unroll
            for (int mt = 0; mt < C::MTW; mt++) {
                const v4f cx = *(const v4f*)(xs + gi * C::TM + mt * 16 + 4u * q);
                v4f t[NS];
#pragma unroll
                for (int st = 0; st < NS; st++) {
                    t[st] = cx;
                    if (C::ASYM) {
#pragma unroll
                        for (int i = 0; i < 4; i++) t[st][i] *= zc[st];
                    }
                }
#pragma unroll
                for (int r = 0; r < RG; r++) {
                    const v8bf a = *(const v8bf*)(xl + (mt * 16 + c) * C::XROW + (kc * 128u + w4_koff<G>(q, gr * RG + r)) * 2u);
#pragma unroll
                    for (int st = 0; st < NS; st++) t[st] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[st][r], t[st], 0, 0, 0);
                }
#pragma unroll
                for (int st = 0; st < NS; st++)
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[st][mt][i] = fmaf(t[st][i], s[st], acc[st][mt][i]);
            }
            }
        }
    };

    load_x(chunk_step(0u));
#pragma unroll
    for (int d = 0; d < C::D; d++) load_w(ring[d], chunk_step(0u) + d);
    uint32_t run = 0xFFFFFFFFu;
    for (uint32_t j = 0; j < chunks; j++) {
        const uint32_t s0 = chunk_step(j), next = chunk_step(j + 1u < chunks ? j + 1u : j);
        if ((s0 - s_lo) / (C::CS * C::CR) != run) { /* the same in every lane; only this wave's LDS */
            run = (s0 - s_lo) / (C::CS * C::CR);
            stage_run(run);
        }
        lds_barrier(); /* every wave has left the chunk before */
        stage_x();
        lds_barrier();
        load_x(next);
#pragma unroll
        for (int i = 0; i < C::CS; i++) {
            const uint32_t s = s0 + i;
            Step& b = ring[i % C::D];
            stage_w(b, 0u);
            multiply(2u * i, s * C::KS);
            stage_w(b, 1u);
            load_w(b, i + C::D < C::CS ? s + C::D : next + (i + C::D - C::CS));
            multiply(2u * i + 1u, s * C::KS + 128u);
        }
    }

    /* ---- results: lane holds channel c, rows 4 q + i ---- */
    constexpr int OUT = C::GLU ? 1 : NS;
#pragma unroll
    for (int mt = 0; mt < C::MTW; mt++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t t = rb + mt * 16u + 4u * q + i;
            if (t >= cnt) continue;
            const uint32_t r = r0 + t, oi = g.o_idx ? g.o_idx[r] : r;
            if (oi == PLOW_EXPERT_UNUSED || (g.a_idx && g.a_idx[r] == PLOW_EXPERT_UNUSED)) continue;
#pragma unroll
            for (int o = 0; o < OUT; o++) {
                const uint32_t n = n0 + (wv * OUT + o) * 16u + c;
                if (n >= N) continue;
                if (tl.slices) {
                    tl.part[((size_t)slice * (C::GLU ? 2u : 1u) * g.M + t) * N + n] = acc[o][mt][i];
                    if (C::GLU) tl.part[(((size_t)slice * 2u + 1u) * g.M + t) * N + n] = acc[NS - 1][mt][i];
                    continue;
                }
                const float v = C::GLU ? moe_glu(acc[0][mt][i], acc[NS - 1][mt][i], g.act, g.f0, g.f1) : (g.gate ? g.gate[r] : 1.0f) * acc[o][mt][i];
                if (!C::GLU && g.out_f32) ((float*)g.out)[(size_t)oi * g.ldo + n] = v;
                else ((bf16_t*)g.out)[(size_t)oi * g.ldo + n] = f2bf(v);
            }
        }
}

/* grid: x = channel tiles, y = dense row tile or expert (its row tiles one after the other), z = K slice. CHOICE: behind
 * a choice made on the device (instances of their own: with the test in all of them the GLU of groups of 128 with zero
 * points needs four registers more than it has, and 64 tokens over 128 experts take 316 us for 298) */
template <class C, bool CHOICE>
__global__ __launch_bounds__(C::THREADS, C::MTW == 1 ? 3 : 1) void k_w4_rows(GroupW4 g, W4Tiles tl) {
    extern __shared__ __attribute__((aligned(16))) uint8_t w4_lds[];
    const uint32_t n0 = blockIdx.x * C::TN;
    if (!g.meta) {
        w4_rows_tile<C>(g, tl, w4_lds, 0u, 0u, g.M, blockIdx.y * C::TM, n0, blockIdx.z);
        return;
    }
    if (CHOICE && !w4_chosen(g, 0u)) return;
    const uint32_t e = blockIdx.y, cnt = (uint32_t)g.meta[g.E + e], r0 = (uint32_t)g.meta[e];
    if (cnt == 0u) return;
    for (int st = 0; st < (C::GLU ? 2 : 1); st++) {
        const size_t at = (size_t)e * 3u + g.sel[st];
        if (!g.wtab[at] || !g.stab[at] || (C::ASYM && !g.ztab[at])) return; /* not resident */
    }
    for (uint32_t rb = 0; rb < cnt; rb += C::TM) {
        w4_rows_tile<C>(g, tl, w4_lds, e, r0, cnt, rb, n0, 0u);
    }
}

uint32_t w4_rows_channels(bool glu, bool wide) { return 64u * (!glu && wide ? 2u : 1u); }
uint32_t w4_rows_kstep() { return 256u; }

/* f(configuration that serves g) */
template <int MTW, int NS, bool GLU, class F>
static int by_group(const GroupW4& g, F&& f) {
    const bool z = g.ztab || g.z[0];
    if (g.G == 32u) return z ? f(RowsCfg<MTW, NS, GLU, 32, true>()) : f(RowsCfg<MTW, NS, GLU, 32, false>());
    if (g.G == 64u) return z ? f(RowsCfg<MTW, NS, GLU, 64, true>()) : f(RowsCfg<MTW, NS, GLU, 64, false>());
    return z ? f(RowsCfg<MTW, NS, GLU, 128, true>()) : f(RowsCfg<MTW, NS, GLU, 128, false>());
}
template <class F>
static int by_form(const GroupW4& g, bool glu, bool wide, uint32_t rows, F&& f) {
    if (rows == 16u) return glu ? by_group<1, 2, true>(g, f) : wide ? by_group<1, 2, false>(g, f) : by_group<1, 1, false>(g, f);
    return glu ? by_group<2, 2, true>(g, f) : wide ? by_group<2, 2, false>(g, f) : by_group<2, 1, false>(g, f);
}
/* workgroups of the kernel that a CU holds, asked once */
template <class C>
static int rows_per_cu = 1;
/* the forms that a choice on the device is made for: tiles of 16 rows x 64 channels */
template <class C>
static constexpr bool behind_choice = C::MTW == 1 && (C::GLU || C::NS == 1);

int w4_rows_launch(const GroupW4& g, const W4Tiles& tl, bool glu, bool wide, uint32_t rows, dim3 grid, hipStream_t st) {
    return by_form(g, glu, wide, rows, [&](auto c) {
        using C = decltype(c);
        if (!g.meta || !g.ws) {
            k_w4_rows<C, false><<<grid, C::THREADS, C::LDS, st>>>(g, tl);
            return 0;
        }
        if constexpr (behind_choice<C>) {
            k_w4_rows<C, true><<<grid, C::THREADS, C::LDS, st>>>(g, tl);
            return 0;
        }
        return (int)PLOW_MOE_EINVAL;
    });
}
int w4_rows_per_cu(const GroupW4& g, bool glu, bool wide, uint32_t rows) {
    return by_form(g, glu, wide, rows, [](auto c) { return rows_per_cu<decltype(c)>; });
}

template <class C>
static bool setup1() {
    const void* const k = (const void*)k_w4_rows<C, false>;
    if constexpr (behind_choice<C>) {
        if (hipFuncSetAttribute((const void*)k_w4_rows<C, true>, hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS) != hipSuccess) return false;
    }
    return hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS) == hipSuccess &&
           hipOccupancyMaxActiveBlocksPerMultiprocessor(&rows_per_cu<C>, k, C::THREADS, C::LDS) == hipSuccess && rows_per_cu<C> > 0;
}
template <int MTW, int NS, bool GLU>
static bool setup2() {
    return setup1<RowsCfg<MTW, NS, GLU, 32, true>>() && setup1<RowsCfg<MTW, NS, GLU, 32, false>>() && setup1<RowsCfg<MTW, NS, GLU, 64, true>>() &&
           setup1<RowsCfg<MTW, NS, GLU, 64, false>>() && setup1<RowsCfg<MTW, NS, GLU, 128, true>>() && setup1<RowsCfg<MTW, NS, GLU, 128, false>>();
}
bool w4_rows_setup() {
    return setup2<1, 1, false>() && setup2<1, 2, false>() && setup2<1, 2, true>() && setup2<2, 1, false>() && setup2<2, 2, false>() && setup2<2, 2, true>();
}
