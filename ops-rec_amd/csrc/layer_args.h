// Arguments of the kernels around attention in a layer: norms with residual and gate, rotary positions, gated projections.
#pragma once
#include <stdint.h>

namespace hstu {

// norm_fwd_kernel (layer_norm_kernel.hip.h).  A row of `groups` * `len` columns; rows of the outputs are contiguous.
struct NormArgs {
    const void* x;
    const void* residual;  // in front of a block: the stream the sum starts from; behind one: what the result is added to, or nullptr
    const void* gate;      // behind a block: or nullptr
    const void* gamma;
    const void* beta;   // or nullptr
    const void* scale;  // in front of a block: per column, or nullptr
    void* out;          // the norm's result (in front), the block's (behind)
    void* sum;          // in front of a block: residual + scale * x
    int64_t x_stride;   // elements from row to row
    int64_t residual_stride;
    int64_t gate_stride;
    uint32_t units;  // rows * groups
    int groups;
    int len;  // columns that share a mean
    float epsilon;
    float residual_scale;
    int affine_f32;  // gamma, beta and scale are fp32, not of the type of x
    int rms;
    int silu;
};

// norm_bwd_kernel
struct NormBwdArgs {
    NormArgs f;            // x, residual, gate, gamma, beta (behind a block), scale, strides and options as above; out and sum unused
    const void* sum;       // in front of a block, a stream in fp32: the sum, contiguous (16-bit streams: from residual and x)
    const void* grad;      // of `out`, contiguous, or nullptr
    const void* sum_grad;  // of the sum, contiguous, or nullptr
    void* x_grad;          // or nullptr (in front of a block: the same as residual_grad)
    void* residual_grad;   // in front of a block
    void* gate_grad;       // behind a block, with a gate
    float* partial;        // [kinds][slices][groups * len]: sums over the slice's rows for gamma, then beta, then scale
    int slices;
    int want_beta;
    int want_scale;
};

// norm_sums_kernel
struct NormSumsArgs {
    const float* partial;
    void* out[3];  // gradients of gamma, beta, scale, in the order of the partial sums
    int kinds;
    int slices;
    int cols;
    int out_dtype;  // HSTU_DT_*
};

// launches it (layer_norm_mi355.hip): HSTU_OK, or the code of set_error
int launch_column_sums(const NormSumsArgs& a, void* stream);

// rotary_kernel (rotary_kernel.hip.h)
struct RotaryArgs {
    const void* q;  // from the launch's first row on, as are k, the outputs and positions
    const void* k;
    void* q_out;
    void* k_out;
    const double* frequencies;
    const void* positions;  // or nullptr
    const void* seq_offset;
    const void* start;  // or nullptr
    int64_t row0;       // the launch's first row
    int64_t q_stride_row, q_stride_head, k_stride_row, k_stride_head;
    uint32_t rows;  // of this launch
    int heads_q, heads;  // of q; of q and k
    int dim, pairs;
    int n_offsets;
    int heads_each;   // heads a thread turns
    int head_blocks;  // threads that share a row and its pairs
    int turned, items;  // threads of a head: with pairs to turn, and with those that copy
    int positions64, offsets64, start64;
    float magnitude;
    float sign;  // of sin
};

}  // namespace hstu
