// The norm kernels by type: a table of variants per translation unit, by growing capacity.
#pragma once
#include "layer_args.h"

namespace hstu {

constexpr int kNormVariants = 10;
constexpr int kNormMaxLen = 16384;  // columns that share a mean, at most: the last variant's capacity

struct NormVariant {
    int capacity;                    // columns that share a mean, at most
    int lanes;                       // that share a row
    int fwd_threads, bwd_threads;    // of a workgroup
    void (*fwd[2])(const NormArgs);  // in front of a block, behind one
    void (*bwd[2])(const NormBwdArgs);
};

const NormVariant* norm_variants_bf16(bool stream_f32);
const NormVariant* norm_variants_f16(bool stream_f32);
const NormVariant* norm_variants_f32();

}  // namespace hstu
