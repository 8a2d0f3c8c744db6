// The table of one type's attention variants: included by the translation unit that instantiates them.
#pragma once
#include "hstu_paged_fp8_tile_kernel.hip.h"
#include "hstu_paged_fp8_variants.h"

#define FP8_ONE(tag, tagname, NC, WK, WR, W, wname)                                      \
    {"hstu_paged_fp8_" tagname "_d" #NC "x32_keys" #WK "_rows" #WR "x32" wname,           \
     hstu::hstu_paged_fp8_attend_kernel<hstu::tag, NC, WK, WR, W>, 64 * (WK) * (WR), 32 * (WR)}
#define FP8_TILE_ONE(tag, tagname, NC, W, wname) \
    {"hstu_paged_fp8_" tagname "_d" #NC "x32_tile" wname, hstu::hstu_paged_fp8_tile_kernel<hstu::tag, NC, W>, hstu::kFp8TileThreads, hstu::kFp8TileRows}
#define FP8_TILE(tag, tagname, NC) {FP8_TILE_ONE(tag, tagname, NC, false, ""), FP8_TILE_ONE(tag, tagname, NC, true, "_weights")}
#define FP8_BOTH(tag, tagname, NC, WK, WR) {FP8_ONE(tag, tagname, NC, WK, WR, false, ""), FP8_ONE(tag, tagname, NC, WK, WR, true, "_weights")}
// up to 128 dims a wavefront needs less than 256 registers and eight fit a CU's files; above, 512 and four; the tile kernel's
// buffers of converted codes fit LDS three times up to 128 dims
#define FP8_NARROW(tag, tagname, NC) {FP8_BOTH(tag, tagname, NC, 8, 1), FP8_TILE(tag, tagname, NC)}
#define FP8_WIDE(tag, tagname, NC) {FP8_BOTH(tag, tagname, NC, 4, 1), FP8_BOTH(tag, tagname, NC, 1, 4)}
#define FP8_TABLE(tag, tagname)                                                                                                \
    {FP8_NARROW(tag, tagname, 1), FP8_NARROW(tag, tagname, 2), FP8_NARROW(tag, tagname, 3), FP8_NARROW(tag, tagname, 4),       \
     FP8_WIDE(tag, tagname, 6), FP8_WIDE(tag, tagname, 8)}
