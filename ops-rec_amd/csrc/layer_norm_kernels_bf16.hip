// The norm kernels for x of bf16.
#include "layer_norm_table.h"

namespace hstu {

const NormVariant* norm_variants_bf16(bool stream_f32)
{
    return stream_f32 ? norm_table<ln_bf16_tag, ln_f32_tag>() : norm_table<ln_bf16_tag, ln_bf16_tag>();
}

}  // namespace hstu
