// act_backward.cu -- the elementwise part of the backward passes of gemm_bias_act_residual and gated_gemm, with the
// column sums that the gradients of the biases are:
//
//   plain   dz = dc * act'(z)                                          dbias = sum over rows of dz
//   gated   dgate = dh * up * act'(gate),  dup = dh * act(gate)        one such sum each
//
// fp32 arithmetic; the sums are taken over the unrounded values, the stored dz / dgate / dup are rounded to bf16 because
// they are operands of the tensor-core contractions that follow.
//
// Bound: HBM (plain 6, gated 10 bytes per element). A thread owns a vector of eight columns and walks every
// (8 gridDim.y)-th row of them, so the column sums are register accumulators; the eight warps of a CTA meet in shared
// memory, the CTAs that share a strip leave partial rows that a second launch adds in ascending order (no atomics).
#include "activation.cuh"
#include "ffn_gemm.h"
#include "rowvec.cuh"
#include "sm100_ptx.cuh"

namespace tcab {
namespace {

using IO = VecIO<__nv_bfloat16, 8>;

constexpr uint32_t kStripCols = 256, kCtaRows = 8;

// GATED: in0 = dh, in1 = gate, in2 = up, out0 = dgate, out1 = dup. Otherwise in0 = dc, in1 = z, out0 = dz (null: column
// sums of in0 alone). `sum` [gridDim.y][GATED ? 2 : 1][cols] where SUMS.
template <int ACT, bool GATED, bool SUMS>
__global__ void __launch_bounds__(256, GATED ? 1 : 3)
act_backward_kernel(const __nv_bfloat16* __restrict__ in0, const __nv_bfloat16* __restrict__ in1,
                    const __nv_bfloat16* __restrict__ in2, __nv_bfloat16* __restrict__ out0, __nv_bfloat16* __restrict__ out1,
                    float* __restrict__ sum, uint32_t rows, uint32_t cols) {
  constexpr int NS = GATED ? 2 : 1;
  ptx::pdl_wait();
  ptx::pdl_launch();
  __shared__ float part[SUMS ? kCtaRows : 1][SUMS ? kStripCols + 8 : 1];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t col = blockIdx.x * kStripCols + lane * 8;
  const bool live = col < cols;
  float acc[NS][8];
#pragma unroll
  for (int n = 0; n < NS; ++n)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[n][j] = 0.0f;
  const uint32_t nvec = cols / 8, v = col / 8;
  // Two rows are computed while the next two are on their way (AHEAD): a slope is some fifteen instructions per element, as
  // long as the load takes (gelu with column sums 4096 x 11008: 50 -> 43 us, gelu_tanh 61 -> 47). The gated form has six
  // loads in flight for two rows; with one row and one ahead it was slower (81 -> 101 us).
  constexpr int U = 2;
  constexpr bool AHEAD = !GATED;
  const uint64_t step = static_cast<uint64_t>(gridDim.y) * kCtaRows;
  uint4 q0[U], q1[U], q2[U], p0[U], p1[U], p2[U];
  auto load = [&](uint64_t row0, uint4 (&a)[U], uint4 (&b)[U], uint4 (&c)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t row = row0 + u * step;
      if (row < rows) {
        const uint64_t at = row * nvec + v;
        a[u] = ld_stream(reinterpret_cast<const uint4*>(in0) + at);
        if (ACT != TCAB_ACT_NONE) b[u] = ld_stream(reinterpret_cast<const uint4*>(in1) + at);
        if (GATED) c[u] = ld_stream(reinterpret_cast<const uint4*>(in2) + at);
      }
    }
  };
  uint64_t row0 = static_cast<uint64_t>(blockIdx.y) * kCtaRows + warp;
  if (AHEAD && live) load(row0, q0, q1, q2);
  for (; live && row0 < rows; row0 += U * step) {
    if (AHEAD) load(row0 + U * step, p0, p1, p2);
    else load(row0, q0, q1, q2);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t row = row0 + u * step;
      if (row >= rows) continue;
      const uint64_t at = row * nvec + v;
      float d[8], up[8], o1[8];
      IO::unpack(q0[u], d);
      if constexpr (ACT != TCAB_ACT_NONE) {
        float z[8], value[8], slope[8];
        IO::unpack(q1[u], z);
        if (GATED) IO::unpack(q2[u], up);
        act_values_slopes<ACT>(z, value, slope);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (GATED) o1[j] = d[j] * value[j];
          d[j] = (GATED ? d[j] * up[j] : d[j]) * slope[j];
        }
      }
      if constexpr (SUMS) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          acc[0][j] += d[j];
          if (GATED) acc[NS - 1][j] += o1[j];
        }
      }
      if (out0 != nullptr) reinterpret_cast<uint4*>(out0)[at] = IO::pack(d);  // the contractions read it next: keep it in L2
      if (GATED) reinterpret_cast<uint4*>(out1)[at] = IO::pack(o1);
    }
    if (AHEAD) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        q0[u] = p0[u];
        q1[u] = p1[u];
      }
    }
  }
  if constexpr (SUMS) {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      if (n > 0) __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) part[warp][lane * 8 + j] = acc[n][j];
      __syncthreads();
      const uint32_t c = blockIdx.x * kStripCols + threadIdx.x;
      if (c < cols) {
        float t = 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < kCtaRows; ++k) t += part[k][threadIdx.x];
        sum[(static_cast<uint64_t>(blockIdx.y) * NS + n) * cols + c] = t;
      }
    }
  }
}

// out_n[c] = sum over p of sum[p][n][c]: eight interleaved ascending chains that meet in order.
__global__ void __launch_bounds__(256)
act_backward_finish(const float* __restrict__ sum, uint32_t parts, uint32_t ns, uint32_t cols, float* __restrict__ out0,
                    float* __restrict__ out1) {
  __shared__ float meet[8][33];
  ptx::pdl_wait();
  ptx::pdl_launch();
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t c = static_cast<uint64_t>(blockIdx.x) * 32 + lane, width = static_cast<uint64_t>(ns) * cols;
  float t = 0.0f;
  if (c < width) {
#pragma unroll 8
    for (uint32_t p = warp; p < parts; p += 8) t += sum[p * width + c];
  }
  meet[warp][lane] = t;
  __syncthreads();
  if (warp == 0 && c < width) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += meet[k][lane];
    if (c < cols) {
      if (out0 != nullptr) out0[c] = s;
    } else if (out1 != nullptr) {
      out1[c - cols] = s;
    }
  }
}

// CTAs that share a strip of columns: about eight per SM in all, each with at least four rows per warp.
uint32_t row_parts(uint32_t rows, uint32_t cols) {
  const uint64_t strips = (static_cast<uint64_t>(cols) + kStripCols - 1) / kStripCols;
  uint64_t parts = (static_cast<uint64_t>(sm_count()) * 8 + strips - 1) / (strips ? strips : 1);
  const uint64_t most = (static_cast<uint64_t>(rows) + 4 * kCtaRows - 1) / (4 * kCtaRows);
  if (parts > most) parts = most;
  if (parts > 65535) parts = 65535;
  return static_cast<uint32_t>(parts < 1 ? 1 : parts);
}

template <int ACT, bool GATED>
int launch(const char* op, const __nv_bfloat16* in0, const __nv_bfloat16* in1, const __nv_bfloat16* in2, __nv_bfloat16* out0,
           __nv_bfloat16* out1, float* dbias0, float* dbias1, uint32_t rows, uint32_t cols, void* ws, cudaStream_t s) {
  if (cols == 0) return TCAB_OK;
  const bool sums = dbias0 != nullptr || dbias1 != nullptr;
  if (rows == 0 && !sums) return TCAB_OK;
  const uint32_t parts = row_parts(rows, cols);
  const dim3 grid((cols + kStripCols - 1) / kStripCols, parts);
  float* sum = static_cast<float*>(ws);
  const bool direct = sums && !act_backward_finishes(rows, cols, GATED);  // one partial row: it is the result
  if (direct) sum = dbias0;
  if (sums) launch_pdl(act_backward_kernel<ACT, GATED, true>, grid, dim3(256), 0, s, in0, in1, in2, out0, out1, sum, rows, cols);
  else launch_pdl(act_backward_kernel<ACT, GATED, false>, grid, dim3(256), 0, s, in0, in1, in2, out0, out1, static_cast<float*>(nullptr), rows, cols);
  count_launch();
  const int rc = check_launch(op);
  if (rc != TCAB_OK || !sums || direct) return rc;
  const uint32_t ns = GATED ? 2 : 1;
  launch_pdl(act_backward_finish, dim3(static_cast<unsigned>((static_cast<uint64_t>(ns) * cols + 31) / 32)), dim3(256), 0, s,
             static_cast<const float*>(sum), parts, ns, cols, dbias0, dbias1);
  count_launch();
  return check_launch(op);
}

}  // namespace

bool act_backward_finishes(uint32_t rows, uint32_t cols, int gated) { return gated || row_parts(rows, cols) > 1; }

uint64_t act_backward_workspace(uint32_t rows, uint32_t cols, int gated) {
  return static_cast<uint64_t>(row_parts(rows, cols)) * (gated ? 2 : 1) * cols * sizeof(float);
}

int launch_act_backward(const char* op, int act, const __nv_bfloat16* dc, const __nv_bfloat16* z, __nv_bfloat16* dz,
                        float* dbias, uint32_t rows, uint32_t cols, void* ws, cudaStream_t s) {
  switch (act) {
#define TCAB_CASE(A) case A: return launch<A, false>(op, dc, z, nullptr, dz, nullptr, dbias, nullptr, rows, cols, ws, s);
    TCAB_CASE(TCAB_ACT_NONE) TCAB_CASE(TCAB_ACT_RELU) TCAB_CASE(TCAB_ACT_SILU) TCAB_CASE(TCAB_ACT_GELU) TCAB_CASE(TCAB_ACT_GELU_TANH)
#undef TCAB_CASE
    default: return fail(TCAB_ERR_UNSUPPORTED, "%s: no kernel for activation %d", op, act);
  }
}

int launch_gated_backward(const char* op, int act, const __nv_bfloat16* dh, const __nv_bfloat16* gate, const __nv_bfloat16* up,
                          __nv_bfloat16* dgate, __nv_bfloat16* dup, float* dbias_gate, float* dbias_up, uint32_t rows,
                          uint32_t cols, void* ws, cudaStream_t s) {
  switch (act) {
#define TCAB_CASE(A) case A: return launch<A, true>(op, dh, gate, up, dgate, dup, dbias_gate, dbias_up, rows, cols, ws, s);
    TCAB_CASE(TCAB_ACT_RELU) TCAB_CASE(TCAB_ACT_SILU) TCAB_CASE(TCAB_ACT_GELU) TCAB_CASE(TCAB_ACT_GELU_TANH) TCAB_CASE(TCAB_ACT_SIGMOID)
#undef TCAB_CASE
    default: return fail(TCAB_ERR_UNSUPPORTED, "%s: no kernel for activation %d", op, act);
  }
}

}  // namespace tcab
