// The gated projections' kernels for fp16.
#include "gated_linear_table.h"

namespace hstu {

const GatedKernels& gated_kernels_f16() { return gated_table<f16_tag>(); }

}  // namespace hstu
