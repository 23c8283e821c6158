/* w4_forms.h — the int4 matrix-unit kernels (w4_rows.hip, w4_tiled.hip) as the dispatch in w4.hip sees them. */
#ifndef PLOW_MOE_W4_FORMS_H
#define PLOW_MOE_W4_FORMS_H

#include "kernels.h"

/* the kernels for a few rows read scales in runs of 64: a tensor holds one at least */
#define W4_TINY_GROUPS 64u
struct W4Tiles;

uint32_t w4_rows_channels(bool glu, bool wide); /* channels of a tile; wide: 32 per wave */
uint32_t w4_rows_kstep();
uint32_t w4_tiled_channels(bool glu);
uint32_t w4_tiled_kstep();
int w4_rows_launch(const GroupW4& g, const W4Tiles& tl, bool glu, bool wide, uint32_t rows, dim3 grid, hipStream_t st);
int w4_tiled_launch(const GroupW4& g, const W4Tiles& tl, bool glu, uint32_t rows, dim3 grid, hipStream_t st);
/* workgroups of that kernel that a CU holds at once */
int w4_rows_per_cu(const GroupW4& g, bool glu, bool wide, uint32_t rows);
int w4_tiled_per_cu(const GroupW4& g, bool glu, uint32_t rows);
bool w4_rows_setup();
bool w4_tiled_setup();
#endif
