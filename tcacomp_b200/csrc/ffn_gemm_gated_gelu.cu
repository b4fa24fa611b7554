// ffn_gemm_gated_gelu.cu -- ffn_gemm_kernel, form kFfnGated, activation gelu (one translation unit per instance: they
// compile side by side).
#include "ffn_gemm.cuh"

namespace tcab {
FfnKernel ffn_kernel_gated_gelu(int shape) { return ffn_kernel_of<kFfnGated, TCAB_ACT_GELU>(shape); }
}  // namespace tcab
