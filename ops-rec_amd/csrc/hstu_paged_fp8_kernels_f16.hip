// Attention over the 8-bit paged cache, fp16 queries.
#include <hip/hip_runtime.h>

#include "hstu_paged_fp8_table.h"

namespace hstu {

extern const Fp8AttendTable kFp8AttendF16 = FP8_TABLE(f16_tag, "f16");

}  // namespace hstu
