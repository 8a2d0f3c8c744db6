// The gated projections' kernels for bf16.
#include "gated_linear_table.h"

namespace hstu {

const GatedKernels& gated_kernels_bf16() { return gated_table<bf16_tag>(); }

}  // namespace hstu
