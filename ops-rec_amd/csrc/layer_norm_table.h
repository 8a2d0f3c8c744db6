// Instantiates the norm kernels of one type of x for one type of stream (for the translation units of layer_norm_kernels_*.hip).
#pragma once
#include "layer_norm_kernel.hip.h"
#include "layer_norm_variants.h"

namespace hstu {

// The forward and the backward kernel of a capacity: the backward holds three sums per column beside the row and takes more lanes
// with fewer pieces each (4 pieces a lane would put 60 to 400 registers into scratch memory).
template <typename T, typename R, int G, int NV, int BG, int BNV>
constexpr NormVariant norm_variant()
{
    static_assert(G * NV == BG * BNV, "both hold the same rows");
    return {8 * G * NV,
            G,
            norm_fwd_threads(G),
            BG,
            norm_bwd_threads(BG),
            {norm_fwd_kernel<T, R, kNormFront, G, NV>, norm_fwd_kernel<T, R, kNormBehind, G, NV>},
            {norm_bwd_kernel<T, R, kNormFront, BG, BNV>, norm_bwd_kernel<T, R, kNormBehind, BG, BNV>}};
}

template <typename T, typename R>
const NormVariant* norm_table()
{
    static const NormVariant table[kNormVariants] = {
        norm_variant<T, R, 8, 1, 8, 1>(),    norm_variant<T, R, 16, 1, 16, 1>(),   norm_variant<T, R, 32, 1, 32, 1>(),
        norm_variant<T, R, 64, 1, 64, 1>(),  norm_variant<T, R, 64, 2, 64, 2>(),   norm_variant<T, R, 64, 4, 256, 1>(),
        norm_variant<T, R, 256, 2, 256, 2>(), norm_variant<T, R, 256, 4, 512, 2>(), norm_variant<T, R, 1024, 2, 1024, 2>()};
    return table;
}

}  // namespace hstu
