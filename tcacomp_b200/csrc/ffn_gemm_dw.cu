// ffn_gemm_dw.cu -- ffn_gemm_kernel, form kFfnDw.
#include "ffn_gemm.cuh"

namespace tcab {
FfnKernel ffn_kernel_dw(int shape) { return ffn_kernel_of<kFfnDw, TCAB_ACT_NONE>(shape); }
}  // namespace tcab
