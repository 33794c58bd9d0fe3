// GEMM instances: fp32, the gated products and the batch, all tile sizes.
#include "nsw_gemm_kernel.h"

#define NSW_GEMM_T float

namespace nsw {
#define NSW_GEMM_SIZE Big
NSW_GEMM_GATED_FORMS(NSW_GEMM_INSTANCE)
NSW_GEMM_BATCH_FORMS(NSW_GEMM_INSTANCE)
#undef NSW_GEMM_SIZE
#define NSW_GEMM_SIZE Mid
NSW_GEMM_GATED_FORMS(NSW_GEMM_INSTANCE)
NSW_GEMM_BATCH_FORMS(NSW_GEMM_INSTANCE)
#undef NSW_GEMM_SIZE
#define NSW_GEMM_SIZE Small
NSW_GEMM_GATED_FORMS(NSW_GEMM_INSTANCE)
NSW_GEMM_BATCH_FORMS(NSW_GEMM_INSTANCE)
}  // namespace nsw
