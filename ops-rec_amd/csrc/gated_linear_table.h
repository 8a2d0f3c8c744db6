// Instantiates the gated projections' kernels of one type (for the translation units gated_linear_kernels_*.hip).
#pragma once
#include "gated_linear_bwd_kernel.hip.h"
#include "gated_linear_few_rows.hip.h"
#include "gated_linear_gemm.hip.h"
#include "gated_linear_variants.h"

namespace hstu {

template <typename Tag, int MODE, int WM, int WN, int MB, int NB, int STAGES, int PER_CU>
constexpr GatedTile gated_tile()
{
    return {gated_gemm_kernel<Tag, MODE, WM, WN, MB, NB, STAGES, PER_CU>, 32 * WN * NB / (MODE == kGemmForward ? 2 : 1), 32 * WM * MB, PER_CU};
}

template <typename Tag>
const GatedKernels& gated_table()
{
    static const GatedKernels table = {
        {gated_tile<Tag, kGemmForward, 2, 2, 4, 4, 4, 1>(), gated_tile<Tag, kGemmForward, 2, 2, 2, 4, 3, 2>(), gated_tile<Tag, kGemmForward, 2, 2, 2, 2, 3, 3>(),
         gated_tile<Tag, kGemmForward, 2, 2, 1, 2, 3, 4>()},
        {gated_tile<Tag, kGemmXGrad, 2, 2, 4, 4, 4, 1>(), gated_tile<Tag, kGemmXGrad, 2, 2, 3, 4, 4, 1>(), gated_tile<Tag, kGemmXGrad, 2, 2, 2, 4, 3, 2>(),
         gated_tile<Tag, kGemmXGrad, 2, 2, 2, 2, 3, 3>(), gated_tile<Tag, kGemmXGrad, 2, 2, 1, 2, 3, 4>()},
        {gated_tile<Tag, kGemmWeightGrad, 2, 2, 4, 4, 4, 1>(), gated_tile<Tag, kGemmWeightGrad, 2, 2, 2, 4, 3, 2>(),
         gated_tile<Tag, kGemmWeightGrad, 2, 2, 2, 2, 3, 3>()},
        {{gated_few_rows_kernel<Tag, 1, 8>, gated_few_rows_kernel<Tag, 1, 16>},
         {gated_few_rows_kernel<Tag, 2, 8>, gated_few_rows_kernel<Tag, 2, 16>},
         {gated_few_rows_kernel<Tag, 4, 8>, gated_few_rows_kernel<Tag, 4, 16>}},
        gated_stage_kernel<Tag>,
        gated_sum_kernel<Tag>};
    return table;
}

}  // namespace hstu
