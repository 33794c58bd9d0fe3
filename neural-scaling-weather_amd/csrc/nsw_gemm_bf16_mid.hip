// GEMM instances: bf16, mid tiles.
#undef NSW_GEMM_STAMPS
#include "nsw_gemm_kernel.h"

#define NSW_GEMM_T bf16
#define NSW_GEMM_SIZE Mid

namespace nsw {
NSW_GEMM_FORMS(NSW_GEMM_INSTANCE)
NSW_GEMM_KTAIL_FORMS(NSW_GEMM_INSTANCE)
}  // namespace nsw
