// ffn_gemm_fwd_gelu.cu -- ffn_gemm_kernel, form kFfnFwd, activation gelu (one translation unit per instance: they
// compile side by side).
#include "ffn_gemm.cuh"

namespace tcab {
FfnKernel ffn_kernel_fwd_gelu(int shape) { return ffn_kernel_of<kFfnFwd, TCAB_ACT_GELU>(shape); }
}  // namespace tcab
