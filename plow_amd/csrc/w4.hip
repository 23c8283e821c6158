/* w4.hip — products with 4-bit integer weights and group scales: dense (GEMM_W4, GEMM_GLU_W4) and routed experts
 * (ops 48 / 49 and 85 / 86 at enc 16).
 *
 *   out[m][n] = sum over groups g of s[n][g] * sum_{k in g} x[m][k] * (q[n][k] - z[n][g])
 *
 * GLU: bf16(act(gate) * up) of two such sums; DOWN of routed experts: gate_r * sum as f32. */
#include "common.h"
#include "kernels.h"
#include "tuning.h"

#define W4_WAVES 4u

__device__ __forceinline__ float w4_scale(const void* s, size_t i, uint32_t f16) {
    const uint16_t h = ((const uint16_t*)s)[i];
    return f16 ? (float)__builtin_bit_cast(_Float16, h) : bf2f(h);
}

/* one weight row times one row of x, the wave's lanes taking 8 k each in turn; the sum in every lane */
__device__ __forceinline__ float w4_dot(const uint8_t* w, const void* s, const uint8_t* z, size_t row, const bf16_t* x,
                                        uint32_t K, uint32_t G, uint32_t f16, uint32_t lane) {
    float acc = 0.0f;
    const uint32_t* wr = (const uint32_t*)(w + row * (K / 2u));
    for (uint32_t p = lane; p < K / 8u; p += WAVE) {
        const size_t gi = row * (K / G) + p * 8u / G;
        const float zf = z ? (float)z[gi] : 8.0f;
        const uint32_t q = wr[p];
        float t = 0.0f;
#pragma unroll
        for (uint32_t j = 0; j < 8u; j++) t = fmaf((float)((q >> (4u * j)) & 15u) - zf, bf2f(x[p * 8u + j]), t);
        acc = fmaf(t, w4_scale(s, gi, f16), acc);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) acc += __shfl_xor(acc, o, 64);
    return acc;
}

/* a wave per output channel and, in turn, the rows of one expert (or the dense rows) */
__global__ __launch_bounds__(W4_WAVES* WAVE) void k_w4_plain(GroupW4 g, uint32_t glu) {
    const uint32_t lane = threadIdx.x & 63u, e = blockIdx.y;
    const uint32_t n = blockIdx.x * W4_WAVES + (threadIdx.x >> 6);
    if (n >= g.N) return;
    const void *w[2], *s[2], *z[2];
    for (uint32_t j = 0; j < 1u + glu; j++) {
        w[j] = g.wtab ? (const void*)(uintptr_t)g.wtab[(size_t)e * 3u + g.sel[j]] : g.w[j];
        s[j] = g.stab ? (const void*)(uintptr_t)g.stab[(size_t)e * 3u + g.sel[j]] : g.s[j];
        z[j] = g.ztab ? (const void*)(uintptr_t)g.ztab[(size_t)e * 3u + g.sel[j]] : g.z[j];
        if (!w[j] || !s[j] || (g.ztab && !z[j])) return; /* expert not resident */
    }
    const uint32_t r0 = g.meta ? (uint32_t)g.meta[e] : 0u, cnt = g.meta ? (uint32_t)g.meta[g.E + e] : g.M;
    for (uint32_t r = r0 + blockIdx.z; r < r0 + cnt; r += gridDim.z) {
        const uint32_t ai = g.a_idx ? g.a_idx[r] : r, oi = g.o_idx ? g.o_idx[r] : r;
        if (ai == PLOW_EXPERT_UNUSED || oi == PLOW_EXPERT_UNUSED) continue;
        const bf16_t* x = (const bf16_t*)g.x + (size_t)ai * g.ldx;
        float v = w4_dot((const uint8_t*)w[0], s[0], (const uint8_t*)z[0], n, x, g.K, g.G, g.s_f16, lane);
        if (glu) v = moe_glu(v, w4_dot((const uint8_t*)w[1], s[1], (const uint8_t*)z[1], n, x, g.K, g.G, g.s_f16, lane), g.act, g.f0, g.f1);
        if (g.gate) v *= g.gate[r];
        if (lane) continue;
        if (g.out_f32) ((float*)g.out)[(size_t)oi * g.ldo + n] = v;
        else ((bf16_t*)g.out)[(size_t)oi * g.ldo + n] = f2bf(v);
    }
}

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

int launch_w4(const GroupW4& g, bool glu, hipStream_t st) {
    if (!g.N || !g.K || !g.E) return PLOW_MOE_EINVAL;
    if (g.zero_unserved) {
        k_w4_zero_unserved<<<g.nslot, 256, 0, st>>>(g);
    }
    const uint32_t rows = g.meta ? 4u : (g.M < 1024u ? g.M : 1024u);
    k_w4_plain<<<dim3((g.N + W4_WAVES - 1u) / W4_WAVES, g.E, rows), W4_WAVES * WAVE, 0, st>>>(g, glu ? 1u : 0u);
    return 0;
}
