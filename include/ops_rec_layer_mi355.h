/*
 * C ABI of the MI355X (gfx950) build of further operators around HSTU attention in a layer: the norms in front of and behind a block, with
 * residual, scale and gate, and their backward; rotary positions; the projections of a gated feed-forward block.  Same library, status codes,
 * dtype codes and error text (hstu_last_error) as hstu_mi355.h.  The reference has no operator of the kind.
 *
 * Every call takes a hipStream_t (NULL = the default stream), launches on it and returns without waiting: HSTU_OK, or HSTU_ERR_NULLPTR /
 * HSTU_ERR_INVALID / HSTU_ERR_WORKSPACE (nothing launched) / HSTU_ERR_RUNTIME.  Strides are in elements; the values of a row lie side by side.
 */
#ifndef OPS_REC_LAYER_MI355_H
#define OPS_REC_LAYER_MI355_H

#include "hstu_mi355.h"

#ifdef __cplusplus
extern "C" {
#endif

/* columns that share a mean, at most */
#define OPS_REC_NORM_MAX_LEN 16384

/*
 * residual_norm, in front of a block:  s = residual + scale * x;  sum = s in the type of the stream;  y = norm(s) * gamma + beta
 *   norm(s) = (s - mean) * rstd over a row, or s * rstd with rms != 0;  rstd = 1 / sqrt(mean of the squares + epsilon); arithmetic in fp32
 */
typedef struct residual_norm_params {
    uint32_t struct_size; /* sizeof(residual_norm_params), checked */
    int32_t rms;
    const void* x;        /* [rows, cols], fp32, bf16 or fp16 */
    const void* residual; /* [rows, cols], the type of x or fp32 (stream_dtype) */
    const void* gamma;    /* [cols]; gamma, beta and scale are all fp32 or all of the type of x (affine_dtype) */
    const void* beta;     /* [cols], or NULL for none */
    const void* scale;    /* [cols], or NULL for 1 */
    void* y;              /* [rows, cols], contiguous, the type of x */
    void* sum;            /* [rows, cols], contiguous, stream_dtype */
    int64_t rows;
    int64_t cols;
    int64_t x_stride;
    int64_t residual_stride;
    int32_t dtype;
    int32_t stream_dtype;
    int32_t affine_dtype;
    float epsilon;
} residual_norm_params;

HSTU_API int residual_norm_fwd(const residual_norm_params* params, void* stream);

/* The gradients of residual_norm.  `fwd` describes the call as it was (y and sum are not read through it). */
typedef struct residual_norm_bwd_params {
    uint32_t struct_size; /* sizeof(residual_norm_bwd_params), checked */
    uint32_t reserved0;
    residual_norm_params fwd; /* x may be NULL where sum is given and scale is not, residual where sum is given */
    const void* sum;          /* what the forward wrote, where stream_dtype is fp32; NULL otherwise */
    const void* y_grad;       /* [rows, cols], contiguous, the type of x, or NULL for zeros */
    const void* sum_grad;     /* [rows, cols], contiguous, stream_dtype, or NULL for zeros */
    void* x_grad;             /* [rows, cols], the type of x, or NULL (without scale and in one type it is residual_grad) */
    void* residual_grad;      /* [rows, cols], stream_dtype */
    void* gamma_grad;         /* [cols], affine_dtype */
    void* beta_grad;          /* [cols], affine_dtype, or NULL */
    void* scale_grad;         /* [cols], affine_dtype, or NULL */
} residual_norm_bwd_params;

HSTU_API int residual_norm_bwd_workspace_size(const residual_norm_bwd_params* params, uint64_t* workspace_bytes);
HSTU_API int residual_norm_bwd(const residual_norm_bwd_params* params, void* workspace, uint64_t workspace_bytes, void* stream);

/*
 * norm_gate, behind a block:  m = norm(x) * gamma + beta, the norm over each of `groups` equal parts of a row;
 *   out = m * act(gate), or residual + residual_scale * m * act(gate);  act is the identity, or silu with silu != 0
 */
typedef struct norm_gate_params {
    uint32_t struct_size; /* sizeof(norm_gate_params), checked */
    int32_t rms;
    const void* x;        /* [rows, cols], fp32, bf16 or fp16 */
    const void* gate;     /* [rows, cols], the type of x, or NULL for 1 */
    const void* gamma;    /* [cols]; gamma and beta are both fp32 or both of the type of x (affine_dtype) */
    const void* beta;     /* [cols], or NULL for none */
    const void* residual; /* [rows, cols], stream_dtype, or NULL for none */
    void* out;            /* [rows, cols], contiguous; stream_dtype (without a residual: the type of x) */
    int64_t rows;
    int64_t cols;
    int64_t x_stride;
    int64_t gate_stride;
    int64_t residual_stride;
    int32_t groups;
    int32_t silu;
    int32_t dtype;
    int32_t stream_dtype; /* the type of x or fp32; without a residual the type of x */
    int32_t affine_dtype;
    float epsilon;
    float residual_scale;
    uint32_t reserved0;
} norm_gate_params;

HSTU_API int norm_gate_fwd(const norm_gate_params* params, void* stream);

/* The gradients of norm_gate; that of the residual is the gradient of `out` itself. */
typedef struct norm_gate_bwd_params {
    uint32_t struct_size; /* sizeof(norm_gate_bwd_params), checked */
    uint32_t reserved0;
    norm_gate_params fwd; /* residual says only whether there is one: it is not read; out is not read */
    const void* out_grad; /* [rows, cols], contiguous, the type of out */
    void* x_grad;         /* [rows, cols], the type of x */
    void* gate_grad;      /* [rows, cols], the type of x; NULL without a gate */
    void* gamma_grad;     /* [cols], affine_dtype */
    void* beta_grad;      /* [cols], affine_dtype, or NULL */
} norm_gate_bwd_params;

HSTU_API int norm_gate_bwd_workspace_size(const norm_gate_bwd_params* params, uint64_t* workspace_bytes);
HSTU_API int norm_gate_bwd(const norm_gate_bwd_params* params, void* workspace, uint64_t workspace_bytes, void* stream);

/*
 * rotary: pairs (a, b) of the first 2 * pairs values of every head of q and k are turned by the row's position times their frequency,
 *   (a, b) -> magnitude * (a cos - b sin, b cos + a sin);  inverse != 0: sin negated (the transpose: what gradients go through)
 * pairs are (j, j + pairs), or (2 j, 2 j + 1) with interleaved != 0; the other values of a head are copied.  The position of a row is
 * positions[row], or its place in its sequence plus start[sequence]; rows of no sequence come out as zeros.  Angles are formed in 64 bits.
 */
typedef struct rotary_params {
    uint32_t struct_size; /* sizeof(rotary_params), checked */
    int32_t dtype;        /* of q and k: fp32, bf16 or fp16 */
    const void* q;        /* [rows, heads_q, dim] */
    const void* k;        /* [rows, heads_k, dim] */
    void* q_out;          /* contiguous */
    void* k_out;
    const double* frequencies; /* [pairs], radians per position */
    const void* positions;     /* [rows], or NULL: by seq_offset */
    const void* seq_offset;    /* [n_offsets], not decreasing */
    const void* start;         /* [n_offsets - 1], or NULL for zeros */
    int64_t rows;
    int64_t heads_q;
    int64_t heads_k;
    int64_t dim;
    int64_t pairs;
    int64_t n_offsets;
    int64_t q_stride_row;
    int64_t q_stride_head;
    int64_t k_stride_row;
    int64_t k_stride_head;
    double magnitude;
    int32_t positions_dtype; /* HSTU_IDX_I32 or HSTU_IDX_I64, each */
    int32_t seq_offset_dtype;
    int32_t start_dtype;
    int32_t interleaved;
    int32_t inverse;
    uint32_t reserved0;
} rotary_params;

HSTU_API int rotary_fwd(const rotary_params* params, void* stream);

/* activations of gated_linear: z sigmoid(z); gelu by its tanh form, z sigmoid(2 sqrt(2 / pi) (z + 0.044715 z^3)); sigmoid(z) */
#define OPS_REC_ACT_SILU 0
#define OPS_REC_ACT_GELU 1
#define OPS_REC_ACT_SIGMOID 2

/*
 * gated_linear, both projections of a gated feed-forward block with activation and product:
 *   mixed = x weight^T + bias = (g, u);  hidden = act(g) * u
 * sums in fp32, of which hidden is taken.  A backward reads mixed: 24 bits of every sum, in 3 * inner words of 16 bits per row, in an order of this
 * library's own.
 */
typedef struct gated_linear_params {
    uint32_t struct_size; /* sizeof(gated_linear_params), checked */
    int32_t activation;
    const void* x;      /* [rows, cols], bf16 or fp16, contiguous, 16-byte aligned, as are all tensors here */
    const void* weight; /* [2 * inner, cols], same type: the rows of g, then those of u */
    const void* bias;   /* [2 * inner], same type, or NULL for none */
    void* hidden;       /* [rows, inner], same type, or NULL */
    void* mixed;        /* [rows, 3 * inner] words of 16 bits, or NULL; the forward writes one of the two at least */
    int64_t rows;
    int64_t cols;  /* a multiple of 8, at most 2^21 */
    int64_t inner; /* a multiple of 8, at most 2^21; inner * cols below 2^29 */
    int32_t dtype; /* HSTU_DT_BF16 or HSTU_DT_FP16 */
    uint32_t reserved0;
} gated_linear_params;

HSTU_API int gated_linear_fwd(const gated_linear_params* params, void* stream);

/* name of the kernel variant gated_linear_fwd would launch, or NULL after an error */
HSTU_API const char* gated_linear_fwd_kernel_name(const gated_linear_params* params);

/* The gradients of gated_linear.  `fwd` describes the call as it was, with mixed as it was written (hidden is not read), or
 * NULL: g and u are then multiplied again.  The gradients of g and u are rounded to the type of x for the products behind them, half a step of it; in fp16 all
 * of a call's are multiplied by a power of two first, chosen on the device by the largest, so that none is past 65504 and the steps of the smallest are 2^-22 of
 * the largest at most. */
typedef struct gated_linear_bwd_params {
    uint32_t struct_size; /* sizeof(gated_linear_bwd_params), checked */
    uint32_t reserved0;
    gated_linear_params fwd;
    const void* grad;  /* [rows, inner], gradient of hidden */
    void* x_grad;      /* [rows, cols], or NULL */
    void* weight_grad; /* [2 * inner, cols], or NULL */
    void* bias_grad;   /* [2 * inner], or NULL */
} gated_linear_bwd_params;

/* the parts of a backward: the gradients of g and u, out of mixed or multiplied again, and the products behind them */
#define OPS_REC_GATED_MIXED_GRAD 0
#define OPS_REC_GATED_X_GRAD 1
#define OPS_REC_GATED_WEIGHT_GRAD 2

/* name of the kernel variant gated_linear_bwd would launch for a part, and the chunks its depth is cut into (chunks may be NULL); NULL for a part the call does
 * not have, or after an error */
HSTU_API const char* gated_linear_bwd_kernel_name(const gated_linear_bwd_params* params, int part, int64_t* chunks);

HSTU_API int gated_linear_bwd_workspace_size(const gated_linear_bwd_params* params, uint64_t* workspace_bytes);
HSTU_API int gated_linear_bwd(const gated_linear_bwd_params* params, void* workspace, uint64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
