// The gated projections' kernels by type.
#pragma once
#include "gated_linear_args.h"

namespace hstu {

struct GatedTile {
    void (*kernel)(const GatedGemmArgs);
    const char* name;
    int cols;  // of the output, per workgroup (in the forward: of hidden)
    int rows;
    // what a workgroup takes, in us (measured at 512 .. 4096 deep products): a step of the depth with a compute unit to itself, its share of a step where
    // the units are full, and everything before the first and behind the last step.  Among tiles their ratios decide; against the bytes of the kernel for few
    // rows, and the traffic and the launch of partial outputs, their size
    float alone, step, fixed;
};

constexpr int kGatedForwardTiles = 4, kGatedMixedTiles = 3, kGatedXGradTiles = 5, kGatedWeightTiles = 3;  // by falling size

struct GatedKernels {
    GatedTile forward[kGatedForwardTiles];
    GatedTile mixed_grad[kGatedMixedTiles];
    GatedTile x_grad[kGatedXGradTiles];
    GatedTile weight_grad[kGatedWeightTiles];
    void (*few_rows[6][4])(const GatedFewRowsArgs);  // up to 16, 32, .. 96 rows; 8, 16, 24, 32 columns of hidden per workgroup
    void (*stage)(const GatedStageArgs);
    void (*sum)(const GatedSumArgs);
};

const GatedKernels& gated_kernels_bf16();
const GatedKernels& gated_kernels_f16();

}  // namespace hstu
