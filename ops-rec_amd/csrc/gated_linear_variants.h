// The gated projections' kernels by type.
#pragma once
#include "gated_linear_args.h"

namespace hstu {

struct GatedTile {
    void (*kernel)(const GatedGemmArgs);
    int cols;  // of the output, per workgroup (in the forward: of hidden)
    int rows;
};

enum { kGatedTileWide, kGatedTileSquare, kGatedTileLow, kGatedTiles };

struct GatedKernels {
    GatedTile forward[kGatedTiles];
    GatedTile x_grad[kGatedTiles];
    GatedTile weight_grad[2];  // wide, square
    void (*few_rows[3][2])(const GatedFewRowsArgs);  // up to 16, 32, 64 rows; 8 or 16 columns of hidden per workgroup
    void (*stage)(const GatedStageArgs);
    void (*sum)(const GatedSumArgs);
};

const GatedKernels& gated_kernels_bf16();
const GatedKernels& gated_kernels_f16();

}  // namespace hstu
