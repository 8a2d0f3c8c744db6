// The variants of the attention kernel over the 8-bit paged cache, by type of q (hstu_paged_fp8_kernels_*.hip).
#pragma once
#include "hstu_paged_fp8.h"

namespace hstu {

// how a workgroup's wavefronts are dealt: over the keys of one tile of 32 rows, or over four tiles
enum Fp8Shape { kFp8Keys = 0, kFp8Rows = 1, kFp8Shapes = 2 };

struct Fp8AttendVariant {
    const char* name;
    void (*kernel)(const Fp8AttendArgs);
    int threads;
    int tile_rows;  // (row, head) pairs of a workgroup; a wavefront has 32
};

// dims in groups of 32 that a variant is built for: the smallest of these that holds the head dim
constexpr int kFp8Groups[] = {1, 2, 3, 4, 6, 8};
constexpr int kFp8GroupCounts = 6;

using Fp8AttendTable = Fp8AttendVariant[kFp8GroupCounts][kFp8Shapes][2];  // [2]: without and with weights
extern const Fp8AttendTable kFp8AttendBf16, kFp8AttendF16;

}  // namespace hstu
