// The variants of the attention kernel over the 8-bit paged cache, by type of q (hstu_paged_fp8_kernels_*.hip).
#pragma once
#include "hstu_paged_fp8.h"

namespace hstu {

// (row, head) pairs of a workgroup whose wavefronts share the keys, and of one of the tile kernel
constexpr int kFp8KeysRows = 32, kFp8TileRows = 128, kFp8TileThreads = 256;

struct Fp8AttendVariant {
    const char* name;
    void (*kernel)(const Fp8AttendArgs);
    int threads;
    int tile_rows;
};

// dims in groups of 32 that a variant is built for: the smallest of these that holds the head dim
constexpr int kFp8Groups[] = {1, 2, 3, 4, 6, 8};
constexpr int kFp8GroupCounts = 6;

struct Fp8AttendTable {
    Fp8AttendVariant keys[kFp8GroupCounts][2][2];  // [wavefronts: as many as fit a CU, half of them][without, with weights]
    Fp8AttendVariant tile;                         // of four groups, without weights
};
extern const Fp8AttendTable kFp8AttendBf16, kFp8AttendF16;

}  // namespace hstu
