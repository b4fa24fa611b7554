// layernorm_backward.cu -- the backward pass of layernorm_rows.cu, with the reductions over rows that gamma's and
// beta's gradients are. With u = (x - mean) * rstd and w = dy * gamma, per row of n columns:
//
//   dx     = rstd * (w - sum(w) / n - u * sum(w * u) / n)
//   dgamma = sum over rows of dy * u        dbeta = sum over rows of dy
//
// mean and rstd come from the forward pass (tcab_layernorm_rows_stats). All arithmetic and every sum is fp32; dx is
// rounded once, to the type of x.
//
// Bound: HBM. x and dy are read once, dx written once (6 bytes per bf16 element, 12 per fp32 element). A thread keeps
// the columns it owns for all the rows its CTA walks, so the column sums are plain register accumulators; a CTA leaves
// one partial row of each and a second launch adds the partials in ascending order (no atomics: the same bits on every
// run). The partials are 8 bytes per column and CTA, about 1 % of the traffic at 65536 rows.
//
//   ln_bwd_warp   rows of up to 128 vectors: 8, 16 or 32 lanes hold a row, sums by shuffles, no barrier in the loop
//   ln_bwd_cta    a CTA per row, up to 512 threads x 4 vectors (16 single elements where rows are not whole vectors);
//                 the next row's loads are issued before the current row's sums are formed
//   ln_bwd_sums + ln_bwd_tile   longer rows: the two row sums first, then dx and the column sums over strips of columns
#include "rowvec.cuh"

namespace tcab {
namespace {

constexpr int kMaxWarps = 16;  // ln_bwd_cta: at most 512 threads

// (a, b) summed over the CTA; every thread gets both. The caller alternates between two slot arrays (one barrier).
__device__ __forceinline__ void cta_allreduce2(float& a, float& b, float2* slots, int nwarps) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    a += __shfl_xor_sync(kFullMask, a, off);
    b += __shfl_xor_sync(kFullMask, b, off);
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) slots[warp] = make_float2(a, b);
  __syncthreads();
  const float2 p = lane < nwarps ? slots[lane] : make_float2(0.0f, 0.0f);
  a = p.x;
  b = p.y;
#pragma unroll
  for (int off = kMaxWarps / 2; off > 0; off >>= 1) {  // nwarps <= 16: the partials sit in lanes 0..15
    a += __shfl_xor_sync(kFullMask, a, off);
    b += __shfl_xor_sync(kFullMask, b, off);
  }
  a = __shfl_sync(kFullMask, a, 0);
  b = __shfl_sync(kFullMask, b, 0);
}

// Where a CTA leaves its column sums: row `blockIdx.x` of pg / pb, `stride` floats apart (one CTA: the outputs).
struct Partials {
  float* pg;
  float* pb;
  size_t stride;
};

template <typename T, int V, int VPT>
__global__ void __launch_bounds__(512, 1)
ln_bwd_cta(const T* __restrict__ dy, const T* __restrict__ x, const T* __restrict__ gamma, const float* __restrict__ mean,
           const float* __restrict__ rstd, T* __restrict__ dx, Partials part, uint64_t rows, uint32_t cols) {
  using IO = VecIO<T, V>;
  using Raw = typename IO::Raw;
  __shared__ float2 slots[2][kMaxWarps];
  const uint32_t nvec = cols / V, threads = blockDim.x;
  const int nwarps = static_cast<int>(threads >> 5);
  const float inv_n = 1.0f / static_cast<float>(cols);

  Raw gq[VPT];
  float ag[VPT][V], ab[VPT][V];
  bool own[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const uint32_t idx = threadIdx.x + i * threads;
    own[i] = idx < nvec;
    if (own[i]) gq[i] = IO::load_keep(gamma, idx);
#pragma unroll
    for (int j = 0; j < V; ++j) ag[i][j] = ab[i][j] = 0.0f;
  }

  Raw xq[VPT], dq[VPT], xn[VPT], dn[VPT];
  float mu = 0.0f, rs = 0.0f, mu_n = 0.0f, rs_n = 0.0f;
  uint64_t row = blockIdx.x;
  if (row < rows) {
    mu = mean[row];
    rs = rstd[row];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const uint32_t idx = threadIdx.x + i * threads;
      if (own[i]) {
        xq[i] = IO::load(x + row * cols, idx);
        dq[i] = IO::load(dy + row * cols, idx);
      }
    }
  }
  int parity = 0;
  for (; row < rows; row += gridDim.x, parity ^= 1) {
    const uint64_t next = row + gridDim.x;
    if (next < rows) {
      mu_n = mean[next];
      rs_n = rstd[next];
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const uint32_t idx = threadIdx.x + i * threads;
        if (own[i]) {
          xn[i] = IO::load(x + next * cols, idx);
          dn[i] = IO::load(dy + next * cols, idx);
        }
      }
    }
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (!own[i]) continue;
      float xf[V], df[V], gf[V];
      IO::unpack(xq[i], xf);
      IO::unpack(dq[i], df);
      IO::unpack(gq[i], gf);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float u = (xf[j] - mu) * rs, w = df[j] * gf[j];
        s1 += w;
        s2 += w * u;
        ag[i][j] += df[j] * u;
        ab[i][j] += df[j];
      }
    }
    cta_allreduce2(s1, s2, slots[parity], nwarps);
    const float c1 = s1 * inv_n, c2 = s2 * inv_n;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (!own[i]) continue;
      float xf[V], df[V], gf[V];
      IO::unpack(xq[i], xf);
      IO::unpack(dq[i], df);
      IO::unpack(gq[i], gf);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float u = (xf[j] - mu) * rs;
        xf[j] = rs * (df[j] * gf[j] - c1 - u * c2);
      }
      IO::store(dx + row * cols, threadIdx.x + i * threads, IO::pack(xf));
      xq[i] = xn[i];
      dq[i] = dn[i];
    }
    mu = mu_n;
    rs = rs_n;
  }
  float* pg = part.pg + blockIdx.x * part.stride;
  float* pb = part.pb + blockIdx.x * part.stride;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (!own[i]) continue;
    const uint32_t c0 = (threadIdx.x + i * threads) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      pg[c0 + j] = ag[i][j];
      pb[c0 + j] = ab[i][j];
    }
  }
}

// Short rows: TPR lanes of a warp hold a row, 32 / TPR rows per warp and step. The column sums of the rows a warp sees
// side by side meet by shuffles at the end, those of the CTA's warps in shared memory.
template <typename T, int V, int TPR, int VPT>
__global__ void __launch_bounds__(256)
ln_bwd_warp(const T* __restrict__ dy, const T* __restrict__ x, const T* __restrict__ gamma, const float* __restrict__ mean,
            const float* __restrict__ rstd, T* __restrict__ dx, Partials part, uint64_t rows, uint32_t cols) {
  using IO = VecIO<T, V>;
  using Raw = typename IO::Raw;
  constexpr int RPW = 32 / TPR, WARPS = 8;
  __shared__ float sums[WARPS][TPR * VPT * V];
  const uint32_t nvec = cols / V;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = lane % TPR, g = lane / TPR;
  const float inv_n = 1.0f / static_cast<float>(cols);
  float gf[VPT][V], ag[VPT][V], ab[VPT][V];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const uint32_t idx = t + i * TPR;
    if (idx < nvec) {
      IO::unpack(IO::load_keep(gamma, idx), gf[i]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) gf[i][j] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) ag[i][j] = ab[i][j] = 0.0f;
  }
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * WARPS * RPW;
  for (uint64_t row0 = (static_cast<uint64_t>(blockIdx.x) * WARPS + warp) * RPW; row0 < rows; row0 += step) {
    const uint64_t row = row0 + g;
    const bool live = row < rows;
    Raw xq[VPT], dq[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const uint32_t idx = t + i * TPR;
      if (live && idx < nvec) {
        xq[i] = IO::load(x + row * cols, idx);
        dq[i] = IO::load(dy + row * cols, idx);
      }
    }
    const float mu = live ? mean[row] : 0.0f, rs = live ? rstd[row] : 0.0f;
    float s1 = 0.0f, s2 = 0.0f;
    float u[VPT][V], w[VPT][V];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const uint32_t idx = t + i * TPR;
      if (live && idx < nvec) {
        float df[V];
        IO::unpack(xq[i], u[i]);
        IO::unpack(dq[i], df);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          u[i][j] = (u[i][j] - mu) * rs;
          w[i][j] = df[j] * gf[i][j];
          s1 += w[i][j];
          s2 += w[i][j] * u[i][j];
          ag[i][j] += df[j] * u[i][j];
          ab[i][j] += df[j];
        }
      }
    }
    s1 = warp_allreduce<OpSum, TPR>(s1);
    s2 = warp_allreduce<OpSum, TPR>(s2);
    const float c1 = s1 * inv_n, c2 = s2 * inv_n;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const uint32_t idx = t + i * TPR;
      if (live && idx < nvec) {
#pragma unroll
        for (int j = 0; j < V; ++j) u[i][j] = rs * (w[i][j] - c1 - u[i][j] * c2);
        IO::store(dx + row * cols, idx, IO::pack(u[i]));
      }
    }
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float* out = (which == 0 ? part.pg : part.pb) + blockIdx.x * part.stride;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float v = which == 0 ? ag[i][j] : ab[i][j];
#pragma unroll
        for (int off = TPR; off < 32; off <<= 1) v += __shfl_xor_sync(kFullMask, v, off);
        if (g == 0) sums[warp][(t + i * TPR) * V + j] = v;
      }
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < cols; c += 256) {
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) v += sums[k][c];
      out[c] = v;
    }
    __syncthreads();
  }
}

// Long rows, first pass: a CTA per row leaves sum(w) / n and sum(w * u) / n.
template <typename T, int V>
__global__ void __launch_bounds__(512)
ln_bwd_sums(const T* __restrict__ dy, const T* __restrict__ x, const T* __restrict__ gamma, const float* __restrict__ mean,
            const float* __restrict__ rstd, float2* __restrict__ row_sums, uint64_t rows, uint32_t cols) {
  using IO = VecIO<T, V>;
  __shared__ float2 slots[2][kMaxWarps];
  const uint32_t nvec = cols / V;
  int parity = 0;
  for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x, parity ^= 1) {
    const float mu = mean[row], rs = rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll 4
    for (uint32_t idx = threadIdx.x; idx < nvec; idx += 512) {
      float xf[V], df[V], gf[V];
      IO::unpack(IO::load_keep(x + row * cols, idx), xf);
      IO::unpack(IO::load_keep(dy + row * cols, idx), df);
      IO::unpack(IO::load_keep(gamma, idx), gf);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float w = df[j] * gf[j];
        s1 += w;
        s2 += w * ((xf[j] - mu) * rs);
      }
    }
    cta_allreduce2(s1, s2, slots[parity], 16);
    if (threadIdx.x == 0) row_sums[row] = make_float2(s1 / static_cast<float>(cols), s2 / static_cast<float>(cols));
  }
}

// Long rows, second pass: a CTA takes a strip of 256 vectors of columns and every gridDim.y-th row.
template <typename T, int V>
__global__ void __launch_bounds__(256)
ln_bwd_tile(const T* __restrict__ dy, const T* __restrict__ x, const T* __restrict__ gamma, const float* __restrict__ mean,
            const float* __restrict__ rstd, const float2* __restrict__ row_sums, T* __restrict__ dx, Partials part,
            uint64_t rows, uint32_t cols) {
  using IO = VecIO<T, V>;
  using Raw = typename IO::Raw;
  const uint32_t idx = blockIdx.x * 256 + threadIdx.x;
  if (idx >= cols / V) return;
  float gf[V], ag[V], ab[V];
  IO::unpack(IO::load_keep(gamma, idx), gf);
#pragma unroll
  for (int j = 0; j < V; ++j) ag[j] = ab[j] = 0.0f;
  constexpr int U = 4;
  const uint64_t step = gridDim.y;
  for (uint64_t row0 = blockIdx.y; row0 < rows; row0 += U * step) {
    Raw xq[U], dq[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const uint64_t row = row0 + k * step;
      if (row < rows) {
        xq[k] = IO::load(x + row * cols, idx);
        dq[k] = IO::load(dy + row * cols, idx);
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const uint64_t row = row0 + k * step;
      if (row < rows) {
        const float mu = mean[row], rs = rstd[row];
        const float2 c = row_sums[row];
        float xf[V], df[V];
        IO::unpack(xq[k], xf);
        IO::unpack(dq[k], df);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float u = (xf[j] - mu) * rs;
          ag[j] += df[j] * u;
          ab[j] += df[j];
          xf[j] = rs * (df[j] * gf[j] - c.x - u * c.y);
        }
        IO::store(dx + row * cols, idx, IO::pack(xf));
      }
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    part.pg[blockIdx.y * part.stride + static_cast<size_t>(idx) * V + j] = ag[j];
    part.pb[blockIdx.y * part.stride + static_cast<size_t>(idx) * V + j] = ab[j];
  }
}

// out[c] = sum over p of partial[p][c], ascending in p within each of eight interleaved chains that then meet in order.
// Columns 0..cols-1 are dgamma's, cols..2 cols-1 dbeta's.
__global__ void __launch_bounds__(256)
ln_bwd_finish(const float* __restrict__ partial, uint32_t parts, uint32_t cols, float* __restrict__ dgamma,
              float* __restrict__ dbeta) {
  __shared__ float sums[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t c = static_cast<uint64_t>(blockIdx.x) * 32 + lane, width = 2ull * cols;
  float v = 0.0f;
  if (c < width) {
#pragma unroll 4
    for (uint32_t p = warp; p < parts; p += 8) v += partial[p * width + c];
  }
  sums[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && c < width) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += sums[k][lane];
    if (c < cols) dgamma[c] = s;
    else dbeta[c - cols] = s;
  }
}

// How a size is cut up: decided without looking at pointers beyond their alignment, so that the workspace can be asked
// for beforehand.
struct Plan {
  int kind;          // 0 ln_bwd_warp, 1 ln_bwd_cta, 2 the two-pass form
  int tpr, vpt;      // ln_bwd_warp: lanes per row; vectors per thread
  uint32_t threads;  // ln_bwd_cta
  uint32_t parts;    // CTAs that leave partial column sums
  uint64_t row_sums_bytes, partial_bytes;
};

Plan make_plan(uint64_t rows, uint32_t cols, int es, bool vec) {
  Plan p = {};
  const int V = vec ? 16 / es : 1;
  const uint32_t nvec = cols / V;
  const uint64_t sms = static_cast<uint64_t>(sm_count());
  if (nvec <= 128) {
    p.kind = 0;
    p.tpr = nvec <= 8 ? 8 : nvec <= 16 ? 16 : 32;
    p.vpt = nvec <= 32 ? 1 : nvec <= 64 ? 2 : 4;
    const uint64_t need = (rows + 8 * (32 / p.tpr) - 1) / (8 * (32 / p.tpr)), most = sms * (p.vpt * V > 16 ? 2 : 4);
    p.parts = static_cast<uint32_t>(need < most ? need : most);
  } else if (nvec <= (vec ? 2048u : 8192u)) {
    p.kind = 1;
    const uint32_t most_vpt = vec ? 4 : 16;
    p.vpt = vec ? 1 : 4;  // single elements: at least four per thread, two bytes per load are few
    while (p.vpt < static_cast<int>(most_vpt) && nvec > 512u * p.vpt) p.vpt *= 2;
    p.threads = (((nvec + p.vpt - 1) / p.vpt) + 31) / 32 * 32;
    const uint64_t most = sms * (512 / p.threads < 1 ? 1 : 512 / p.threads);
    p.parts = static_cast<uint32_t>(rows < most ? rows : most);
  } else {
    p.kind = 2;
    const uint64_t strips = (nvec + 255) / 256;
    uint64_t chunks = (sms * 6 + strips - 1) / strips;
    if (chunks > (rows + 3) / 4) chunks = (rows + 3) / 4;
    if (chunks > 65535) chunks = 65535;
    p.parts = static_cast<uint32_t>(chunks < 1 ? 1 : chunks);
    p.row_sums_bytes = (rows * sizeof(float2) + 255) / 256 * 256;
  }
  if (p.parts < 1) p.parts = 1;
  p.partial_bytes = p.parts > 1 ? static_cast<uint64_t>(p.parts) * 2 * cols * sizeof(float) : 0;
  return p;
}

template <typename T, int VW>
int launch(const T* dy, const T* x, const T* gamma, const float* mean, const float* rstd, T* dx, float* dgamma, float* dbeta,
           uint64_t rows, uint32_t cols, uint8_t* ws, uint64_t ws_bytes, cudaStream_t s) {
  const bool vec = cols % VW == 0 && aligned16(dy) && aligned16(x) && aligned16(gamma) && aligned16(dx);
  const Plan p = make_plan(rows, cols, sizeof(T), vec);
  if (p.row_sums_bytes + p.partial_bytes > ws_bytes)
    return fail(TCAB_ERR_INVALID_ARG, "layernorm_rows_backward: the workspace has %llu bytes, %llu are needed",
                static_cast<unsigned long long>(ws_bytes), static_cast<unsigned long long>(p.row_sums_bytes + p.partial_bytes));
  float* partial = reinterpret_cast<float*>(ws + p.row_sums_bytes);
  const Partials part = p.parts > 1 ? Partials{partial, partial + cols, 2 * static_cast<size_t>(cols)} : Partials{dgamma, dbeta, 0};
  const char* what = "ln_bwd";
  bool launched = false;
  if (p.kind == 0) {
#define TCAB_CASE(VV, TP, P)                                                                                         \
  if (!launched && p.tpr == TP && p.vpt == P) {                                                                      \
    ln_bwd_warp<T, VV, TP, P><<<p.parts, 256, 0, s>>>(dy, x, gamma, mean, rstd, dx, part, rows, cols);               \
    launched = true;                                                                                                 \
  }
    if (vec) {
      TCAB_CASE(VW, 8, 1) TCAB_CASE(VW, 16, 1) TCAB_CASE(VW, 32, 1) TCAB_CASE(VW, 32, 2) TCAB_CASE(VW, 32, 4)
    } else {
      TCAB_CASE(1, 8, 1) TCAB_CASE(1, 16, 1) TCAB_CASE(1, 32, 1) TCAB_CASE(1, 32, 2) TCAB_CASE(1, 32, 4)
    }
#undef TCAB_CASE
    what = "ln_bwd_warp";
  } else if (p.kind == 1) {
#define TCAB_CASE(VV, P)                                                                                             \
  if (!launched && p.vpt == P) {                                                                                     \
    ln_bwd_cta<T, VV, P><<<p.parts, p.threads, 0, s>>>(dy, x, gamma, mean, rstd, dx, part, rows, cols);              \
    launched = true;                                                                                                 \
  }
    if (vec) {
      TCAB_CASE(VW, 1) TCAB_CASE(VW, 2) TCAB_CASE(VW, 4)
    } else {
      TCAB_CASE(1, 4) TCAB_CASE(1, 8) TCAB_CASE(1, 16)
    }
#undef TCAB_CASE
    what = "ln_bwd_cta";
  } else {
    float2* row_sums = reinterpret_cast<float2*>(ws);
    const uint64_t most = static_cast<uint64_t>(sm_count()) * 4;
    const unsigned grid = static_cast<unsigned>(rows < most ? (rows ? rows : 1) : most);
    const uint32_t nvec = vec ? cols / VW : cols;
    const dim3 tiles((nvec + 255) / 256, p.parts);
    if (vec) {
      ln_bwd_sums<T, VW><<<grid, 512, 0, s>>>(dy, x, gamma, mean, rstd, row_sums, rows, cols);
      ln_bwd_tile<T, VW><<<tiles, 256, 0, s>>>(dy, x, gamma, mean, rstd, row_sums, dx, part, rows, cols);
    } else {
      ln_bwd_sums<T, 1><<<grid, 512, 0, s>>>(dy, x, gamma, mean, rstd, row_sums, rows, cols);
      ln_bwd_tile<T, 1><<<tiles, 256, 0, s>>>(dy, x, gamma, mean, rstd, row_sums, dx, part, rows, cols);
    }
    count_launch();
    launched = true;
    what = "ln_bwd_tile";
  }
  if (!launched) return fail(TCAB_ERR_UNSUPPORTED, "layernorm_rows_backward: no kernel for %u columns", cols);
  count_launch();
  const int rc = check_launch(what);
  if (rc != TCAB_OK || p.parts <= 1) return rc;
  ln_bwd_finish<<<static_cast<unsigned>((2ull * cols + 31) / 32), 256, 0, s>>>(partial, p.parts, cols, dgamma, dbeta);
  count_launch();
  return check_launch("ln_bwd_finish");
}

}  // namespace

uint64_t layernorm_backward_workspace(uint64_t rows, uint32_t cols, int elem_bytes) {
  const Plan a = make_plan(rows, cols, elem_bytes, false);
  uint64_t most = a.row_sums_bytes + a.partial_bytes;
  if (cols % (16 / elem_bytes) == 0) {
    const Plan b = make_plan(rows, cols, elem_bytes, true);
    if (b.row_sums_bytes + b.partial_bytes > most) most = b.row_sums_bytes + b.partial_bytes;
  }
  return most;
}

int launch_layernorm_backward_bf16(const __nv_bfloat16* dy, const __nv_bfloat16* x, const __nv_bfloat16* gamma, const float* mean,
                                   const float* rstd, __nv_bfloat16* dx, float* dgamma, float* dbeta, uint64_t rows, uint32_t cols,
                                   void* ws, uint64_t ws_bytes, cudaStream_t s) {
  return launch<__nv_bfloat16, 8>(dy, x, gamma, mean, rstd, dx, dgamma, dbeta, rows, cols, static_cast<uint8_t*>(ws), ws_bytes, s);
}

int launch_layernorm_backward_f32(const float* dy, const float* x, const float* gamma, const float* mean, const float* rstd,
                                  float* dx, float* dgamma, float* dbeta, uint64_t rows, uint32_t cols, void* ws,
                                  uint64_t ws_bytes, cudaStream_t s) {
  return launch<float, 4>(dy, x, gamma, mean, rstd, dx, dgamma, dbeta, rows, cols, static_cast<uint8_t*>(ws), ws_bytes, s);
}

}  // namespace tcab
