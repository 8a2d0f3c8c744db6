// Attention over the 8-bit paged cache, bf16 queries.
#include <hip/hip_runtime.h>

#include "hstu_paged_fp8_table.h"

namespace hstu {

extern const Fp8AttendTable kFp8AttendBf16 = FP8_TABLE(bf16_tag, "bf16");

}  // namespace hstu
