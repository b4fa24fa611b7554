// ffn_gemm_fwd_silu.cu -- ffn_gemm_kernel, form kFfnFwd, activation silu (one translation unit per instance: they
// compile side by side).
#include "ffn_gemm.cuh"

namespace tcab {
FfnKernel ffn_kernel_fwd_silu(int shape) { return ffn_kernel_of<kFfnFwd, TCAB_ACT_SILU>(shape); }
}  // namespace tcab
