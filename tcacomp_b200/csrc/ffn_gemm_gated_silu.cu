// ffn_gemm_gated_silu.cu -- ffn_gemm_kernel, form kFfnGated, activation silu (one translation unit per instance: they
// compile side by side).
#include "ffn_gemm.cuh"

namespace tcab {
FfnKernel ffn_kernel_gated_silu(int shape) { return ffn_kernel_of<kFfnGated, TCAB_ACT_SILU>(shape); }
}  // namespace tcab
