// The gated projections' kernels by type.
#pragma once
#include "gated_linear_args.h"

namespace hstu {

struct GatedTile {
    void (*kernel)(const GatedGemmArgs);
    int cols;  // of the output, per workgroup (in the forward: of hidden)
    int rows;
    int per_cu;  // workgroups that a compute unit holds
};

constexpr int kGatedForwardTiles = 4, kGatedXGradTiles = 5, kGatedWeightTiles = 3;  // by falling size

struct GatedKernels {
    GatedTile forward[kGatedForwardTiles];
    GatedTile x_grad[kGatedXGradTiles];
    GatedTile weight_grad[kGatedWeightTiles];
    void (*few_rows[3][2])(const GatedFewRowsArgs);  // up to 16, 32, 64 rows; 8 or 16 columns of hidden per workgroup
    void (*stage)(const GatedStageArgs);
    void (*sum)(const GatedSumArgs);
};

const GatedKernels& gated_kernels_bf16();
const GatedKernels& gated_kernels_f16();

}  // namespace hstu
