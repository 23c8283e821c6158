/* w4_forms.h — the instances of the int4 matrix-unit kernel (w4_tile.h) by name, for the dispatch in w4.hip. */
#ifndef PLOW_MOE_W4_FORMS_H
#define PLOW_MOE_W4_FORMS_H

#include "kernels.h"

/* the kernels for a few rows read scales in runs of 64: a tensor holds one at least */
#define W4_TINY_GROUPS 64u
struct W4Tiles;
/* rows of one workgroup's tile */
enum W4Form { W4_ROWS16 = 16, W4_ROWS32 = 32, W4_ROWS64 = 64, W4_ROWS128 = 128 };

uint32_t w4_rows_channels(bool glu, bool wide); /* channels of a tile; wide: 32 per wave */
uint32_t w4_rows_kstep();
uint32_t w4_tiled_channels(bool glu, uint32_t rows);
uint32_t w4_tiled_kstep();
int w4_rows_launch(const GroupW4& g, const W4Tiles& tl, bool glu, bool wide, uint32_t rows, dim3 grid, hipStream_t st);
int w4_tiled_launch(const GroupW4& g, const W4Tiles& tl, bool glu, uint32_t rows, dim3 grid, hipStream_t st);
bool w4_rows_setup();
bool w4_tiled_setup();
#endif
