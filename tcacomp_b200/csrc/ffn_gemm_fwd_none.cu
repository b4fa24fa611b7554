// ffn_gemm_fwd_none.cu -- ffn_gemm_kernel, form kFfnFwd, activation none (one translation unit per instance: they
// compile side by side).
#include "ffn_gemm.cuh"

namespace tcab {
FfnKernel ffn_kernel_fwd_none(int shape) { return ffn_kernel_of<kFfnFwd, TCAB_ACT_NONE>(shape); }
}  // namespace tcab
