/* w4_tiled.hip — int4 group-scale products of many rows (w4_tile.h): tiles of 64 or 128 rows x 256 channels (GLU: 128
 * channels of gate and up), a wave per 64 rows x 64 weight rows, so that a weight unpacked feeds four matrix
 * instructions and a row read from LDS four.
 *
 * 2048 x 4096 x 7168, G = 128: 133 us = 903 TFLOP/s (a library product of bf16 by bf16 reaches 1314 at 8192 cubed), the
 * GLU of 2048 x 2048 x 7168 135 us; the products with groups of 32 and zero points 218 us both. 512 tokens over 64 experts
 * of 2048 x 1408, top 6: 102 us for gate and up, 55 for down (347 and 322 TFLOP/s: 48 of a tile's 64 rows count, and the
 * tiles come to 1.4 and just over 1 rounds of what the chip holds). Bound by a SIMD's two waves waiting on LDS and on their
 * barrier: the matrix units are busy 39 % of the time, the vector units (unpacking, scaling, x staged anew by every channel
 * tile) 58 %, LDS 41 % (under the profiler, where the first call takes 156 us). Groups of 32 have a matrix instruction
 * beside four scaling ones and, with zero points, four more that multiply its C operand. Tried and slower, each beside
 * what the first call took at the time: staging the next step between this one's products 183 us for 145, waves of 128 x
 * 64 at one per SIMD 195 for 145, two steps on their way 382 for 145, none of which fits the registers; row tiles of one
 * XCD side by side 155 for 156. */
#include "w4_forms.h"
#include "w4_tile.h"

template <int WT, int NS, int G, bool ASYM>
using Cfg = W4Cfg<WT, 4, 4, NS == 2 ? 2 : 4, NS, 128, 512, G, ASYM>;

uint32_t w4_tiled_channels(bool glu) { return glu ? 128u : 256u; }
uint32_t w4_tiled_kstep() { return 128u; }

/* f(Config) of the configuration that serves g */
template <int WT, int NS, class F>
static int by_group(const GroupW4& g, F&& f) {
    const bool z = g.ztab || g.z[0];
    if (g.G == 32u) return z ? f(Cfg<WT, NS, 32, true>()) : f(Cfg<WT, NS, 32, false>());
    if (g.G == 64u) return z ? f(Cfg<WT, NS, 64, true>()) : f(Cfg<WT, NS, 64, false>());
    return z ? f(Cfg<WT, NS, 128, true>()) : f(Cfg<WT, NS, 128, false>());
}
template <class F>
static int by_form(const GroupW4& g, bool glu, uint32_t rows, F&& f) {
    if (rows == 64u) return glu ? by_group<1, 2>(g, f) : by_group<1, 1>(g, f);
    return glu ? by_group<2, 2>(g, f) : by_group<2, 1>(g, f);
}
int w4_tiled_launch(const GroupW4& g, const W4Tiles& tl, bool glu, uint32_t rows, dim3 grid, hipStream_t st) {
    return by_form(g, glu, rows, [&](auto c) {
        using C = decltype(c);
        if (!g.meta || !g.ws) {
            k_w4_tile<C, false><<<grid, C::THREADS, C::LDS, st>>>(g, tl);
            return 0;
        }
        if constexpr (C::TM == (int)PLOW_MPF_BM) {
            k_w4_tile<C, true><<<grid, C::THREADS, C::LDS, st>>>(g, tl);
            return 0;
        }
        return (int)PLOW_MOE_EINVAL;
    });
}
int w4_tiled_per_cu(const GroupW4& g, bool glu, uint32_t rows) {
    return by_form(g, glu, rows, [](auto c) { return w4_per_cu<decltype(c)>; });
}

template <int WT, int NS>
static bool setup2() {
    return w4_setup<Cfg<WT, NS, 32, true>>() && w4_setup<Cfg<WT, NS, 32, false>>() && w4_setup<Cfg<WT, NS, 64, true>>() &&
           w4_setup<Cfg<WT, NS, 64, false>>() && w4_setup<Cfg<WT, NS, 128, true>>() && w4_setup<Cfg<WT, NS, 128, false>>();
}
bool w4_tiled_setup() { return setup2<1, 1>() && setup2<1, 2>() && setup2<2, 1>() && setup2<2, 2>(); }
