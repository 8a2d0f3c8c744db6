// The table of one type's attention variants: included by the translation unit that instantiates them.
#pragma once
#include "hstu_paged_fp8_tile_kernel.hip.h"
#include "hstu_paged_fp8_variants.h"

#define FP8_ONE(tag, tagname, NC, NB, WK, WR, W, wname)                                                                         \
    {"hstu_paged_fp8_" tagname "_d" #NC "x32_rows" #NB "x32_waves" #WK "x" #WR wname,                                            \
     hstu::hstu_paged_fp8_attend_kernel<hstu::tag, NC, NB, WK, WR, W>, 64 * (WK) * (WR), 32 * (NB), 32 * (NB) * (WR)}
#define FP8_TILE_ONE(tag, tagname, NC, RG, KG, W, wname)                                                                        \
    {"hstu_paged_fp8_" tagname "_d" #NC "x32_rows" #RG "x32_shares" #KG wname, hstu::hstu_paged_fp8_tile_kernel<hstu::tag, NC, RG, KG, W>, 64 * (RG) * (KG), 32, \
     32 * (RG)}
#define FP8_TILE(tag, tagname, NC, RG, KG) {FP8_TILE_ONE(tag, tagname, NC, RG, KG, false, ""), FP8_TILE_ONE(tag, tagname, NC, RG, KG, true, "_weights")}
#define FP8_BOTH(tag, tagname, NC, NB, WK, WR) \
    {FP8_ONE(tag, tagname, NC, NB, WK, WR, false, ""), FP8_ONE(tag, tagname, NC, NB, WK, WR, true, "_weights")}
// up to 128 dims eight wavefronts of one column have 256 registers each, four of two columns 512; above, one column with 512
#define FP8_NARROW(tag, tagname, NC) \
    {FP8_BOTH(tag, tagname, NC, 1, 8, 1), FP8_TILE(tag, tagname, NC, 2, 2), FP8_TILE(tag, tagname, NC, 4, 1)}
#define FP8_WIDE(tag, tagname, NC) \
    {FP8_BOTH(tag, tagname, NC, 1, 4, 1), FP8_BOTH(tag, tagname, NC, 1, 4, 1), FP8_BOTH(tag, tagname, NC, 1, 1, 4)}
#define FP8_TABLE(tag, tagname)                                                                                                \
    {FP8_NARROW(tag, tagname, 1), FP8_NARROW(tag, tagname, 2), FP8_NARROW(tag, tagname, 3), FP8_NARROW(tag, tagname, 4),       \
     FP8_WIDE(tag, tagname, 6), FP8_WIDE(tag, tagname, 8)}
