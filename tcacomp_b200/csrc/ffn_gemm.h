// ffn_gemm.h -- the contractions of a feed-forward layer and of its backward pass (ffn_gemm.cuh), as their callers see them.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace tcab {

enum FfnForm {
  kFfnFwd = 0,    // c = act(a @ b + bias) + residual            a [M, K], b [K, N]
  kFfnGated = 1,  // c = act(a @ b0 + bias0) * (a @ b1 + bias1)  a [M, K], b0, b1 [K, N]
  kFfnDx = 2,     // c = a0 @ b0^T (+ a1 @ b1^T)                 a0, a1 [M, K], b0, b1 [N, K]
  kFfnDw = 3      // c0 = a^T @ b0 (, c1 = a^T @ b1)             a [K, M], b0, b1 [K, N]
};

// One contraction. M, N: the extents of an output, K: the contracted one. Pointers are 16-byte aligned, the innermost
// extents of every operand multiples of eight; any extent may be zero.
struct FfnProblem {
  const __nv_bfloat16* a[2] = {nullptr, nullptr};
  const __nv_bfloat16* b[2] = {nullptr, nullptr};
  __nv_bfloat16* c[2] = {nullptr, nullptr};
  __nv_bfloat16* z[2] = {nullptr, nullptr};  // kFfnFwd: a @ b + bias, kFfnGated: both projections with their biases; or null
  const float* bias[2] = {nullptr, nullptr};
  const __nv_bfloat16* residual = nullptr;
  uint32_t M = 0, N = 0, K = 0;
  int act = TCAB_ACT_NONE;
  // The launch before this one on the stream belongs to the same call and writes none of the operands. The kernel then runs
  // beside it (515 x 1032 x 2056 backward: the second product on the SMs that the first leaves) and waits for it at its own
  // end, so that whoever waits for this kernel has waited for both. What the operands need was complete before: a kernel
  // lets its successor start only when it runs itself, and the first of a call runs on only after everything before it.
  bool beside = false;
  // SMs that the launch beside it holds and for how long by its estimate: the kernel may be cut for the others.
  uint32_t taken = 0;
  double taken_us = 0;
};

// What a launch took, for the one that may run beside it.
struct FfnTaken {
  uint32_t sms = 0;
  double us = 0;
};

int launch_ffn_gemm(const char* op, int form, const FfnProblem& p, cudaStream_t s, FfnTaken* taken = nullptr);
int ffn_device_status(int* out);

// ffn_small.cuh: few rows or few output tiles
struct FfnSmallPlan {
  int tm = 128;                 // output rows per tile
  uint64_t tiles = 0;
  uint32_t ks = 1, blocks_per_range = 0;  // CTAs per tile (1, 2, 4, 8), K blocks of each
  int per_sm = 1;                         // CTAs that share an SM
  double us = 0;                          // the estimate that chose them
};
FfnSmallPlan ffn_small_plan(int form, uint32_t m, uint32_t n, uint32_t k, uint32_t pairs, int sms, int forced_ks);
int launch_ffn_small(const char* op, int form, const FfnProblem& p, int sms, cudaStream_t s);
int ffn_small_status(int* out);
void ffn_plan(int form, uint32_t m, uint32_t n, uint32_t k, uint32_t pairs, int sms, uint32_t* rows, uint32_t* cols, uint32_t* ranges,
              uint32_t* blocks);

// dz = dc * act'(z) (gated: dgate = dh * up * act'(gate), dup = dh * act(gate)), with the column sums of each where
// wanted (act_backward.cu). dz may be null (column sums alone; act none). Partials of the sums go to `ws`.
// Whether column sums take a second launch, behind the one that writes dz.
bool act_backward_finishes(uint32_t rows, uint32_t cols, int gated);
uint64_t act_backward_workspace(uint32_t rows, uint32_t cols, int gated);
int launch_act_backward(const char* op, int act, const __nv_bfloat16* dc, const __nv_bfloat16* z, __nv_bfloat16* dz,
                        float* dbias, uint32_t rows, uint32_t cols, void* ws, cudaStream_t s);
int launch_gated_backward(const char* op, int act, const __nv_bfloat16* dh, const __nv_bfloat16* gate, const __nv_bfloat16* up,
                          __nv_bfloat16* dgate, __nv_bfloat16* dup, float* dbias_gate, float* dbias_up, uint32_t rows,
                          uint32_t cols, void* ws, cudaStream_t s);

// A 2-D bf16 row-major tensor as a TMA tensor map (gemm_bias_act.cu): boxes of 64 columns (128-byte swizzle) or 32
// columns (64-byte swizzle).
int make_tensor_map(const char* op, CUtensorMap* m, const void* base, uint64_t rows, uint64_t cols, uint32_t box_rows,
                    uint32_t box_cols);

}  // namespace tcab
