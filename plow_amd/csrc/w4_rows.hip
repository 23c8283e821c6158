/* w4_rows.hip — int4 group-scale products of a few rows (w4_tile.h): tiles of 16 or 32 rows x 128 channels, a wave per
 * 16 channels, steps of 256 columns (a whole 128-byte line per weight row). */
#include "w4_forms.h"
#include "w4_tile.h"

template <int MTW, int NS, int G, bool ASYM>
using Cfg = W4Cfg<1, 8, MTW, 1, NS, 256, 3, G, ASYM>;

uint32_t w4_rows_channels(bool, uint32_t) { return 128u; }
uint32_t w4_rows_kstep() { return 256u; }

template <int MTW, int NS, int G>
static int by_zero(const GroupW4& g, const W4Tiles& tl, dim3 grid, hipStream_t st) {
    return (g.ztab || g.z[0]) ? w4_launch<Cfg<MTW, NS, G, true>>(g, tl, grid, st) : w4_launch<Cfg<MTW, NS, G, false>>(g, tl, grid, st);
}
template <int MTW, int NS>
static int by_group(const GroupW4& g, const W4Tiles& tl, dim3 grid, hipStream_t st) {
    return g.G == 32u ? by_zero<MTW, NS, 32>(g, tl, grid, st) : g.G == 64u ? by_zero<MTW, NS, 64>(g, tl, grid, st) : by_zero<MTW, NS, 128>(g, tl, grid, st);
}
int w4_rows_launch(const GroupW4& g, const W4Tiles& tl, bool glu, uint32_t rows, dim3 grid, hipStream_t st) {
    if (rows == 16u) return glu ? by_group<1, 2>(g, tl, grid, st) : by_group<1, 1>(g, tl, grid, st);
    return glu ? by_group<2, 2>(g, tl, grid, st) : by_group<2, 1>(g, tl, grid, st);
}

template <int MTW, int NS>
static bool setup2() {
    return w4_setup<Cfg<MTW, NS, 32, true>>() && w4_setup<Cfg<MTW, NS, 32, false>>() && w4_setup<Cfg<MTW, NS, 64, true>>() &&
           w4_setup<Cfg<MTW, NS, 64, false>>() && w4_setup<Cfg<MTW, NS, 128, true>>() && w4_setup<Cfg<MTW, NS, 128, false>>();
}
bool w4_rows_setup() { return setup2<1, 1>() && setup2<1, 2>() && setup2<2, 1>() && setup2<2, 2>(); }
