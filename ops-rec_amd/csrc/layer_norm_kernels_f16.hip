// The norm kernels for x of fp16.
#include "layer_norm_table.h"

namespace hstu {

const NormVariant* norm_variants_f16(bool stream_f32)
{
    return stream_f32 ? norm_table<ln_f16_tag, ln_f32_tag>() : norm_table<ln_f16_tag, ln_f16_tag>();
}

}  // namespace hstu
