// Instantiates the gated projections' kernels of one type (for the translation units gated_linear_kernels_*.hip).
#pragma once
#include "gated_linear_bwd_kernel.hip.h"
#include "gated_linear_few_rows.hip.h"
#include "gated_linear_gemm.hip.h"
#include "gated_linear_variants.h"

namespace hstu {

template <typename Tag, int MODE, int MB, int NB, int STAGES, int PER_CU, int STEP = kGemmStep>
constexpr GatedTile gated_tile(const char* name, float alone, float step, float fixed)
{
    return {gated_gemm_kernel<Tag, MODE, 2, 2, MB, NB, STAGES, PER_CU, STEP>, name, 64 * NB / (MODE == kGemmForward || MODE == kGemmMixedGrad ? 2 : 1), 64 * MB, alone, step, fixed};
}

// (names: rows x columns of the products' tiles)
template <typename Tag>
const GatedKernels& gated_table()
{
    static const GatedKernels table = {
        {gated_tile<Tag, kGemmForward, 4, 4, 2, 1, 64>("gated_gemm_256x256", 0.64f, 0.73f, 10.0f), gated_tile<Tag, kGemmForward, 2, 4, 3, 2>("gated_gemm_128x256", 0.45f, 0.45f, 3.5f),
         gated_tile<Tag, kGemmForward, 2, 2, 3, 3>("gated_gemm_128x128", 0.33f, 0.26f, 3.0f), gated_tile<Tag, kGemmForward, 1, 2, 3, 4>("gated_gemm_64x128", 0.25f, 0.17f, 2.0f)},
        {gated_tile<Tag, kGemmMixedGrad, 2, 4, 3, 2>("gated_gemm_128x256", 0.45f, 0.45f, 3.5f), gated_tile<Tag, kGemmMixedGrad, 2, 2, 3, 3>("gated_gemm_128x128", 0.33f, 0.26f, 3.0f),
         gated_tile<Tag, kGemmMixedGrad, 1, 2, 3, 4>("gated_gemm_64x128", 0.25f, 0.17f, 2.0f)},
        {gated_tile<Tag, kGemmXGrad, 4, 4, 4, 1>("gated_gemm_256x256", 0.76f, 0.76f, 5.0f), gated_tile<Tag, kGemmXGrad, 3, 4, 4, 1>("gated_gemm_192x256", 0.62f, 0.62f, 4.0f),
         gated_tile<Tag, kGemmXGrad, 2, 4, 3, 2>("gated_gemm_128x256", 0.42f, 0.40f, 3.0f), gated_tile<Tag, kGemmXGrad, 2, 2, 3, 3>("gated_gemm_128x128", 0.30f, 0.25f, 2.0f),
         gated_tile<Tag, kGemmXGrad, 1, 2, 3, 4>("gated_gemm_64x128", 0.25f, 0.17f, 1.5f)},
        {gated_tile<Tag, kGemmWeightGrad, 4, 4, 4, 1>("gated_gemm_256x256", 0.85f, 0.85f, 5.0f), gated_tile<Tag, kGemmWeightGrad, 2, 4, 3, 2>("gated_gemm_128x256", 0.45f, 0.41f, 3.0f),
         gated_tile<Tag, kGemmWeightGrad, 2, 2, 3, 3>("gated_gemm_128x128", 0.30f, 0.23f, 2.0f)},
        {{gated_few_rows_kernel<Tag, 1, 1>, gated_few_rows_kernel<Tag, 1, 2>, gated_few_rows_kernel<Tag, 1, 3>, gated_few_rows_kernel<Tag, 1, 4>},
         {gated_few_rows_kernel<Tag, 2, 1>, gated_few_rows_kernel<Tag, 2, 2>, gated_few_rows_kernel<Tag, 2, 3>, gated_few_rows_kernel<Tag, 2, 4>},
         {gated_few_rows_kernel<Tag, 3, 1>, gated_few_rows_kernel<Tag, 3, 2>, gated_few_rows_kernel<Tag, 3, 3>, gated_few_rows_kernel<Tag, 3, 4>},
         {gated_few_rows_kernel<Tag, 4, 1>, gated_few_rows_kernel<Tag, 4, 2>, gated_few_rows_kernel<Tag, 4, 3>, gated_few_rows_kernel<Tag, 4, 4>},
         {gated_few_rows_kernel<Tag, 5, 1>, gated_few_rows_kernel<Tag, 5, 2>, gated_few_rows_kernel<Tag, 5, 3>, gated_few_rows_kernel<Tag, 5, 4>},
         {gated_few_rows_kernel<Tag, 6, 1>, gated_few_rows_kernel<Tag, 6, 2>, gated_few_rows_kernel<Tag, 6, 3>, gated_few_rows_kernel<Tag, 6, 4>}},
        gated_stage_kernel<Tag>,
        gated_sum_kernel<Tag>};
    return table;
}

}  // namespace hstu
