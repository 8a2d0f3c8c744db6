// The table of one type's attention variants: included by the translation unit that instantiates them.
#pragma once
#include "hstu_paged_fp8_tile_kernel.hip.h"

#define FP8_ONE(tag, tagname, NC, WK, W, wname) \
    {"hstu_paged_fp8_" tagname "_d" #NC "x32_keys" #WK wname, hstu::hstu_paged_fp8_attend_kernel<hstu::tag, NC, WK, W>, 64 * (WK), hstu::kFp8KeysRows}
#define FP8_BOTH(tag, tagname, NC, WK) {FP8_ONE(tag, tagname, NC, WK, false, ""), FP8_ONE(tag, tagname, NC, WK, true, "_weights")}
// up to 128 dims a wavefront needs less than 256 registers and eight fit a CU's files; above, 512 and four
#define FP8_NARROW(tag, tagname, NC) {FP8_BOTH(tag, tagname, NC, 8), FP8_BOTH(tag, tagname, NC, 4)}
#define FP8_WIDE(tag, tagname, NC) {FP8_BOTH(tag, tagname, NC, 4), FP8_BOTH(tag, tagname, NC, 2)}
#define FP8_TABLE(tag, tagname)                                                                                          \
    {{FP8_NARROW(tag, tagname, 1), FP8_NARROW(tag, tagname, 2), FP8_NARROW(tag, tagname, 3), FP8_NARROW(tag, tagname, 4), \
      FP8_WIDE(tag, tagname, 6), FP8_WIDE(tag, tagname, 8)},                                                              \
     {"hstu_paged_fp8_" tagname "_d4x32_tile", hstu::hstu_paged_fp8_tile_kernel<hstu::tag, 4>, hstu::kFp8TileThreads, hstu::kFp8TileRows}}
