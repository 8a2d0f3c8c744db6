// Instantiates the gated projections' kernels of one type (for the translation units gated_linear_kernels_*.hip).
#pragma once
#include "gated_linear_bwd_kernel.hip.h"
#include "gated_linear_few_rows.hip.h"
#include "gated_linear_gemm.hip.h"
#include "gated_linear_variants.h"

namespace hstu {

template <typename Tag, int MODE, int BN, int BM, int STAGES>
constexpr GatedTile gated_tile()
{
    return {gated_gemm_kernel<Tag, MODE, BN, BM, STAGES>, MODE == kGemmForward ? BN / 2 : BN, BM};
}

template <typename Tag>
const GatedKernels& gated_table()
{
    static const GatedKernels table = {
        {gated_tile<Tag, kGemmForward, 256, 128, 3>(), gated_tile<Tag, kGemmForward, 128, 128, 3>(), gated_tile<Tag, kGemmForward, 128, 64, 3>()},
        {gated_tile<Tag, kGemmXGrad, 256, 128, 3>(), gated_tile<Tag, kGemmXGrad, 128, 128, 3>(), gated_tile<Tag, kGemmXGrad, 128, 64, 3>()},
        {gated_tile<Tag, kGemmWeightGrad, 256, 128, 3>(), gated_tile<Tag, kGemmWeightGrad, 128, 128, 3>()},
        {{gated_few_rows_kernel<Tag, 1, 8>, gated_few_rows_kernel<Tag, 1, 16>},
         {gated_few_rows_kernel<Tag, 2, 8>, gated_few_rows_kernel<Tag, 2, 16>},
         {gated_few_rows_kernel<Tag, 4, 8>, gated_few_rows_kernel<Tag, 4, 16>}},
        gated_stage_kernel<Tag>,
        gated_sum_kernel<Tag>};
    return table;
}

}  // namespace hstu
