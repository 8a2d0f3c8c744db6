// Instantiates the norm kernels of one type of x for one type of stream (for the translation units of layer_norm_kernels_*.hip).
#pragma once
#include "layer_norm_kernel.hip.h"
#include "layer_norm_variants.h"

namespace hstu {

// parts of rows whose loads are in flight together: two where a lane has one piece of each
constexpr int norm_units(int g, int nv) { return g <= 64 && nv == 1 ? 2 : 1; }

// G lanes with NV pieces of 8 columns each; SHORT: rows of up to 7 columns.  (One piece a lane where there are lanes enough: 2048 columns on 64 lanes with four took 34 us for 8192 rows, on 256
// 27; with two the backward holds 200 registers, with four 60 to 400 of them would be in scratch memory.)
template <typename T, typename R, int G, int NV, bool SHORT = false>
constexpr NormVariant norm_variant()
{
    return {SHORT ? 7 : 8 * G * NV,
            G,
            norm_fwd_threads(G),
            norm_bwd_threads(G),
            {norm_fwd_kernel<T, R, kNormFront, G, NV, norm_units(G, NV), SHORT>, norm_fwd_kernel<T, R, kNormBehind, G, NV, norm_units(G, NV), SHORT>},
            {norm_bwd_kernel<T, R, kNormFront, G, NV, SHORT>, norm_bwd_kernel<T, R, kNormBehind, G, NV, SHORT>}};
}

template <typename T, typename R>
const NormVariant* norm_table()
{
    static const NormVariant table[kNormVariants] = {norm_variant<T, R, 8, 1, true>(), norm_variant<T, R, 8, 1>(),   norm_variant<T, R, 16, 1>(),
                                                     norm_variant<T, R, 32, 1>(),      norm_variant<T, R, 64, 1>(),  norm_variant<T, R, 64, 2>(),
                                                     norm_variant<T, R, 256, 1>(),     norm_variant<T, R, 512, 1>(), norm_variant<T, R, 1024, 1>(),
                                                     norm_variant<T, R, 1024, 2>()};
    return table;
}

}  // namespace hstu
