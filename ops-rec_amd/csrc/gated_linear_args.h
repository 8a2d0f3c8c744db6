// Arguments of the gated projections' kernels.
#pragma once
#include <stdint.h>

namespace hstu {

// What d_mixed is multiplied by in fp16 where its values allow it: from 2^-11 to 255 for the largest (gated_range_kernel).
constexpr float kGatedScale = 256.0f;

constexpr int kActSilu = 0, kActGelu = 1, kActSigmoid = 2;

// gated_gemm_kernel (gated_linear_gemm.hip.h): out[rows, cols] = a . b over `depth`
struct GatedGemmArgs {
    const void* n_side;  // forward, d_mixed: the weight [2 inner, depth]; x gradient: the weight [depth, cols]; weight gradient: x [depth, cols]
    const void* m_side;  // forward, d_mixed: x [rows, depth]; x gradient: d_mixed [rows, depth]; weight gradient: d_mixed [depth, rows]
    const void* bias;    // forward, d_mixed: [2 cols], 16-bit, or nullptr
    void* out;           // forward: hidden [rows, cols], or nullptr; d_mixed: [rows, 2 cols]; gradients: [rows, cols]
    void* mixed;         // forward: [rows, 3 cols] (kept_high), or nullptr
    const void* grad;    // d_mixed: the gradient of hidden [rows, cols]
    float* range;        // d_mixed, fp16: the largest of each wavefront's values [tiles][4], or nullptr
    const float* scale;  // fp16: [0] what d_mixed is multiplied by, [1] the inverse.  d_mixed: of a second pass, nullptr in the first; gradients: always
    float* partial;      // gradients in several chunks of the depth: [chunks][rows][cols]; d_mixed: column sums [2 row tiles][2 cols], or nullptr
    int64_t rows;
    int64_t depth;
    int64_t chunk;  // of the depth, per workgroup: a multiple of 32, or the whole of it
    int cols;       // of the output
    int chunks;
    int activation;
    int tiles_m, tiles_n;
    uint32_t first, count;  // of the tiles of all chunks: what this launch has
};

// gated_few_rows_kernel (gated_linear_few_rows.hip.h)
struct GatedFewRowsArgs {
    const void* x;       // [rows, depth]
    const void* weight;  // [2 inner, depth]
    const void* bias;    // [2 inner], 16-bit, or nullptr
    void* hidden;        // [rows, inner], or nullptr
    void* mixed;         // [rows, 3 inner], or nullptr
    int64_t rows;
    int depth;
    int inner;
    int activation;
};

// gated_stage_kernel and gated_sum_kernel (gated_linear_bwd_kernel.hip.h)
struct GatedStageArgs {
    const void* grad;   // [rows, inner]
    const void* mixed;  // [rows, 3 inner]
    void* d_mixed;      // [rows, 2 inner]
    float* partial;     // [slices][2 inner] column sums, or nullptr
    float* range;       // as in GatedGemmArgs, [workgroups][4]
    const float* scale;
    int64_t rows;
    int inner;
    int slices;
    int activation;
};
struct GatedSumArgs {
    const float* partial;  // [chunks][n]
    const float* scale;    // fp16: as in GatedGemmArgs
    void* out;             // [n], 16-bit
    int64_t n;             // a multiple of 8
    int chunks;
};

}  // namespace hstu
