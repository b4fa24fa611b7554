// ffn_gemm_dx.cu -- ffn_gemm_kernel, form kFfnDx.
#include "ffn_gemm.cuh"

namespace tcab {
FfnKernel ffn_kernel_dx(int shape) { return ffn_kernel_of<kFfnDx, TCAB_ACT_NONE>(shape); }
}  // namespace tcab
