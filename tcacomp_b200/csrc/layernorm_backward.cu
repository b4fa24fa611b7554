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
//   ln_bwd_ring   rows of up to 16384 columns: a CTA per SM, chunks of consecutive rows brought to shared memory by bulk
//                 copies several chunks ahead, groups of 8 threads up to the whole CTA to a row
//   ln_bwd_sums + ln_bwd_tile   longer rows and operands off a 16-byte boundary: the two row sums first, then dx and the
//                 column sums over strips of columns
#include "f32x2.cuh"
#include "rowvec.cuh"
#include "sm100_ptx.cuh"

namespace tcab {
namespace {

constexpr int kMaxWarps = 16;  // 512 threads per CTA

__device__ int g_ln_bwd_status = 0;  // 1: a kernel gave up on a wait

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

// V consecutive elements as fp32 values: pairs, or a lone element as itself. load reads shared memory or (gamma) through
// L1; store writes global memory.
template <int BYTES>
struct RawOf;
template <>
struct RawOf<16> { typedef uint4 type; };
template <>
struct RawOf<8> { typedef uint2 type; };
template <>
struct RawOf<4> { typedef uint32_t type; };
template <>
struct RawOf<2> { typedef unsigned short type; };

__device__ __forceinline__ void words_of(const uint4& q, uint32_t (&w)[4]) { w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w; }
__device__ __forceinline__ void words_of(const uint2& q, uint32_t (&w)[2]) { w[0] = q.x; w[1] = q.y; }
__device__ __forceinline__ void words_of(const uint32_t& q, uint32_t (&w)[1]) { w[0] = q; }
__device__ __forceinline__ uint4 raw_of(const uint32_t (&w)[4]) { return make_uint4(w[0], w[1], w[2], w[3]); }
__device__ __forceinline__ uint2 raw_of(const uint32_t (&w)[2]) { return make_uint2(w[0], w[1]); }
__device__ __forceinline__ uint32_t raw_of(const uint32_t (&w)[1]) { return w[0]; }

template <typename T, int V>
struct Vals;
template <int V>
struct Vals<__nv_bfloat16, V> {  // V = 2, 4, 8: a word is a pair
  static constexpr int N = V / 2;
  typedef f32x2 Num;
  typedef typename RawOf<2 * V>::type Raw;
  static __device__ __forceinline__ void widen(const Raw& q, f32x2 (&v)[N]) {
    uint32_t w[N];
    words_of(q, w);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = pair_of_bf16(w[j]);
  }
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, f32x2 (&v)[N]) { widen(*reinterpret_cast<const Raw*>(p), v); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const f32x2 (&v)[N]) {
    uint32_t w[N];
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = bf16_of_pair(v[j]);
    __stcs(reinterpret_cast<Raw*>(p), raw_of(w));
  }
  static __device__ __forceinline__ void put(float* to, const f32x2 (&v)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) pair_to(v[j], to[2 * j], to[2 * j + 1]);
  }
};
template <int V>
struct Vals<float, V> {  // V = 2, 4: two words are a pair
  static constexpr int N = V / 2;
  typedef f32x2 Num;
  typedef typename RawOf<4 * V>::type Raw;
  static __device__ __forceinline__ void widen(const Raw& q, f32x2 (&v)[N]) {
    uint32_t w[V];
    words_of(q, w);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = pair_of(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
  }
  static __device__ __forceinline__ void load(const float* p, f32x2 (&v)[N]) { widen(*reinterpret_cast<const Raw*>(p), v); }
  static __device__ __forceinline__ void store(float* p, const f32x2 (&v)[N]) {
    uint32_t w[V];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float lo, hi;
      pair_to(v[j], lo, hi);
      w[2 * j] = __float_as_uint(lo);
      w[2 * j + 1] = __float_as_uint(hi);
    }
    __stcs(reinterpret_cast<Raw*>(p), raw_of(w));
  }
  static __device__ __forceinline__ void put(float* to, const f32x2 (&v)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) pair_to(v[j], to[2 * j], to[2 * j + 1]);
  }
};
template <>
struct Vals<__nv_bfloat16, 1> {
  static constexpr int N = 1;
  typedef float Num;
  typedef unsigned short Raw;
  static __device__ __forceinline__ void widen(const Raw& q, float (&v)[1]) { v[0] = __uint_as_float(static_cast<uint32_t>(q) << 16); }
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&v)[1]) { widen(*reinterpret_cast<const Raw*>(p), v); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&v)[1]) { *p = __float2bfloat16_rn(v[0]); }
  static __device__ __forceinline__ void put(float* to, const float (&v)[1]) { *to = v[0]; }
};
template <>
struct Vals<float, 1> {
  static constexpr int N = 1;
  typedef float Num;
  typedef uint32_t Raw;
  static __device__ __forceinline__ void widen(const Raw& q, float (&v)[1]) { v[0] = __uint_as_float(q); }
  static __device__ __forceinline__ void load(const float* p, float (&v)[1]) { v[0] = *p; }
  static __device__ __forceinline__ void store(float* p, const float (&v)[1]) { __stcs(p, v[0]); }
  static __device__ __forceinline__ void put(float* to, const float (&v)[1]) { *to = v[0]; }
};

constexpr uint32_t kRingBytes = 208 * 1024, kRingStages = 8;
constexpr int kSlots = kMaxWarps + 8;  // every group's warps, rounded up to pairs

// Chunks of `groups` RB consecutive rows go through a ring of `stages` shared-memory stages (x, then dy, of a chunk; each
// copied from the 16-byte boundary at or below its first byte, so rows need not be whole vectors). Group g of TPR threads
// takes rows g, g + groups, ... of a chunk, RB of them side by side; thread t owns the vectors t + i TPR of every row.
// TPR = 8, 16, 32: a template constant, sums by shuffles alone. TPR = 0: `tpr` threads (whole warps), sums over one named
// barrier per group and chunk. Thread 0 also issues the copies: a stage is refilled one chunk after it was read.
//
// Why the ring: the rows alone are too few bytes in flight. With the next row prefetched into registers (512 threads, one
// CTA per SM) bf16 rows of 4096 columns ran at 3.9 TB/s. Why pairs and RB: bf16 brings twice the elements per byte, and
// what is left is latency -- the sums of a row have to meet before its second half can start, and what a row costs a thread
// besides its elements. u and w are kept from the first half where the registers allow (KEEP: up to 16 values per thread).
// Measured (TB/s of 6 or 12 bytes per element): bf16 [65536, 8192] 5.2, [131072, 4096] 5.4, [524288, 512] 5.5; fp32
// [65536, 8192] 6.0, [262144, 1024] 5.8; rows of single elements (odd bf16 columns) 2.0-2.3.
template <typename T, int V, int VPT, int TPR_, int RB, bool KEEP>
__global__ void __launch_bounds__(512, 1)
ln_bwd_ring(const T* __restrict__ dy, const T* __restrict__ x, const T* __restrict__ gamma, const float* __restrict__ mean,
            const float* __restrict__ rstd, T* __restrict__ dx, Partials part, uint64_t rows, uint32_t cols, uint32_t tpr,
            uint32_t groups, uint32_t stages, uint32_t plane) {
  using A = Vals<T, V>;
  using Num = typename A::Num;
  constexpr int N = A::N;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ __align__(8) uint64_t bar_full[kRingStages], bar_empty[kRingStages];
  __shared__ __align__(16) float2 slots[2][RB][kSlots];
  __shared__ int abort_flag;
  volatile int* abort_p = &abort_flag;

  const uint32_t TPR = TPR_ > 0 ? TPR_ : tpr;
  const uint32_t g = threadIdx.x / TPR, t = threadIdx.x - g * TPR, nvec = cols / V;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t row_bytes = cols * sizeof(T);
  const uint64_t total = rows * row_bytes, chunk_bytes = static_cast<uint64_t>(groups) * RB * row_bytes;
  const uint64_t chunk_rows = static_cast<uint64_t>(groups) * RB, chunks = (rows + chunk_rows - 1) / chunk_rows;
  const float inv_n = 1.0f / static_cast<float>(cols);
  for (uint32_t k = threadIdx.x; k < 2 * RB * kSlots; k += blockDim.x) (&slots[0][0][0])[k] = make_float2(0.0f, 0.0f);
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (uint32_t s = 0; s < stages; ++s) {
      ptx::mbar_init(ptx::smem_u32(&bar_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&bar_empty[s]), blockDim.x / 32);
    }
    ptx::fence_barrier_init();
    ptx::fence_proxy_async();
  }
  __syncthreads();
  ptx::pdl_wait();
  ptx::pdl_launch();

  auto issue = [&](uint64_t chunk, uint32_t s) {  // thread 0
    const uint64_t from = chunk * chunk_bytes, start = from & ~15ull, end = from + chunk_bytes < total ? from + chunk_bytes : total;
    // Whole 16-byte granules that lie inside the tensor; the few bytes of the very last one come by plain loads.
    const uint64_t stop = ((end + 15) & ~15ull) <= total ? (end + 15) & ~15ull : total & ~15ull;
    uint8_t* dst = ring + s * 2 * plane;
    for (uint64_t at = stop; at < end; at += sizeof(T)) {
      *reinterpret_cast<T*>(dst + (at - start)) = *reinterpret_cast<const T*>(reinterpret_cast<const uint8_t*>(x) + at);
      *reinterpret_cast<T*>(dst + plane + (at - start)) = *reinterpret_cast<const T*>(reinterpret_cast<const uint8_t*>(dy) + at);
    }
    const uint32_t bytes = stop > start ? static_cast<uint32_t>(stop - start) : 0u;
    const uint32_t bar = ptx::smem_u32(&bar_full[s]);
    ptx::mbar_expect_tx(bar, 2 * bytes);
    if (bytes > 0) {
      ptx::bulk_load(ptx::smem_u32(dst), reinterpret_cast<const uint8_t*>(x) + start, bytes, bar);
      ptx::bulk_load(ptx::smem_u32(dst + plane), reinterpret_cast<const uint8_t*>(dy) + start, bytes, bar);
    }
  };
  if (threadIdx.x == 0)
    for (uint32_t s = 0; s < stages && blockIdx.x + static_cast<uint64_t>(s) * gridDim.x < chunks; ++s)
      issue(blockIdx.x + static_cast<uint64_t>(s) * gridDim.x, s);

  Num gm[KEEP ? VPT : 1][N], ag[VPT][N], ab[VPT][N];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const uint32_t idx = t + i * TPR;
    if constexpr (KEEP)
      if (idx < nvec) A::load(gamma + static_cast<size_t>(idx) * V, gm[i]);
#pragma unroll
    for (int j = 0; j < N; ++j) ag[i][j] = ab[i][j] = spread<Num>(0.0f);
  }
  float mu[RB], rs[RB];
  auto load_stats = [&](uint64_t chunk) {
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      const uint64_t row = chunk * chunk_rows + static_cast<uint64_t>(r) * groups + g;
      mu[r] = row < rows ? mean[row] : 0.0f;
      rs[r] = row < rows ? rstd[row] : 0.0f;
    }
  };
  load_stats(blockIdx.x);
  uint32_t stage = 0, phase = 0, parity = 0;
  uint32_t last_stage = 0, last_phase = 0;
  bool ok = true;
  for (uint64_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x, parity ^= 1u) {
    if (threadIdx.x == 0 && chunk != blockIdx.x) {  // refill the stage of the previous chunk
      const uint64_t next = chunk + (static_cast<uint64_t>(stages) - 1) * gridDim.x;
      if (next < chunks && ok) {
        if (ptx::mbar_wait(ptx::smem_u32(&bar_empty[last_stage]), last_phase, abort_p)) issue(next, last_stage);
        else ok = false;
      }
    }
    ok = ptx::mbar_wait(ptx::smem_u32(&bar_full[stage]), phase, abort_p) && ok;
    const uint32_t lead = static_cast<uint32_t>((chunk * chunk_bytes) & 15u);
    const uint8_t* base = ring + (stage * 2 * plane + lead + g * row_bytes);
    // which of this group's rows exist: the last chunk may be short
    const uint64_t left = rows - chunk * chunk_rows;
    bool live[RB];
    T* out_row[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      live[r] = g + r * groups < left;
      out_row[r] = dx + (chunk * chunk_rows + g + r * groups) * cols;
    }
    Num rs2[RB], shift[RB];
    float rs_row[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      rs_row[r] = rs[r];
      rs2[r] = spread<Num>(rs[r]);
      shift[r] = spread<Num>(-mu[r] * rs[r]);
    }
    load_stats(chunk + gridDim.x);  // the next rows' are under way
    Num u[KEEP ? RB : 1][KEEP ? VPT : 1][N], w[KEEP ? RB : 1][KEEP ? VPT : 1][N], s1[RB], s2[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) s1[r] = s2[r] = spread<Num>(0.0f);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const uint32_t idx = t + i * TPR;
      if (idx < nvec) {
        Num gi[N];
        if constexpr (!KEEP) A::load(gamma + idx * V, gi);
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          if (live[r]) {
            const T* xs = reinterpret_cast<const T*>(base + r * groups * row_bytes) + idx * V;
            Num d[N], uu[N], ww[N];
            A::load(xs, uu);
            A::load(reinterpret_cast<const T*>(reinterpret_cast<const uint8_t*>(xs) + plane), d);
#pragma unroll
            for (int j = 0; j < N; ++j) {
              if constexpr (KEEP) ww[j] = gm[i][j];
              else ww[j] = gi[j];
              uu[j] = fma_pair(uu[j], rs2[r], shift[r]);
              ww[j] = mul_pair(d[j], ww[j]);
              s1[r] = add_pair(s1[r], ww[j]);
              s2[r] = fma_pair(ww[j], uu[j], s2[r]);
              ag[i][j] = fma_pair(d[j], uu[j], ag[i][j]);
              ab[i][j] = add_pair(ab[i][j], d[j]);
              if constexpr (KEEP) {
                u[r][i][j] = uu[j];
                w[r][i][j] = ww[j];
              }
            }
          }
        }
      }
    }
    if (KEEP) {  // the stage has been read
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&bar_empty[stage]));
    }
    float t1[RB], t2[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      t1[r] = pair_sum(s1[r]);
      t2[r] = pair_sum(s2[r]);
    }
#pragma unroll
    for (int off = (TPR_ > 0 ? TPR_ : 32) / 2; off > 0; off >>= 1) {
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        t1[r] += __shfl_xor_sync(kFullMask, t1[r], off);
        t2[r] += __shfl_xor_sync(kFullMask, t2[r], off);
      }
    }
    if constexpr (TPR_ == 0) {
      const uint32_t nw = TPR >> 5, padded = (nw + 1) & ~1u;  // the slot of an odd group's missing warp stays zero
      if (lane == 0) {
#pragma unroll
        for (int r = 0; r < RB; ++r) slots[parity][r][g * padded + (warp - g * nw)] = make_float2(t1[r], t2[r]);
      }
      ptx::named_bar_sync(1 + g, TPR);
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const float4* q = reinterpret_cast<const float4*>(&slots[parity][r][g * padded]);
        t1[r] = t2[r] = 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < kMaxWarps / 2; ++k) {  // broadcast reads, the same order in every thread
          if (2 * k < nw) {
            const float4 v = q[k];
            t1[r] += v.x + v.z;
            t2[r] += v.y + v.w;
          }
        }
      }
    }
    Num a[RB], b[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      a[r] = spread<Num>(-rs_row[r] * (t1[r] * inv_n));
      b[r] = spread<Num>(-rs_row[r] * (t2[r] * inv_n));
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const uint32_t idx = t + i * TPR;
      if (idx < nvec && ok) {
        Num gi[N];
        if constexpr (!KEEP) A::load(gamma + idx * V, gi);
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          if (live[r]) {
            Num out[N];
            if constexpr (KEEP) {
#pragma unroll
              for (int j = 0; j < N; ++j) out[j] = fma_pair(u[r][i][j], b[r], fma_pair(w[r][i][j], rs2[r], a[r]));
            } else {
              const T* xs = reinterpret_cast<const T*>(base + r * groups * row_bytes) + idx * V;
              Num d[N], uu[N];
              A::load(xs, uu);
              A::load(reinterpret_cast<const T*>(reinterpret_cast<const uint8_t*>(xs) + plane), d);
#pragma unroll
              for (int j = 0; j < N; ++j)
                out[j] = fma_pair(fma_pair(uu[j], rs2[r], shift[r]), b[r], fma_pair(mul_pair(d[j], gi[j]), rs2[r], a[r]));
            }
            A::store(out_row[r] + idx * V, out);
          }
        }
      }
    }
    if (!KEEP) {
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&bar_empty[stage]));
    }
    last_stage = stage;
    last_phase = phase;
    if (++stage == stages) { stage = 0; phase ^= 1u; }
  }

  // The groups' column sums meet in shared memory (every copy has landed and been read), first dgamma's, then dbeta's.
  float* sums = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float* out = (which == 0 ? part.pg : part.pb) + blockIdx.x * part.stride;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const uint32_t idx = t + i * TPR;
      float* to = sums + static_cast<size_t>(g) * cols + static_cast<size_t>(idx) * V;
      if (idx < nvec) {
        if (which == 0) A::put(to, ag[i]);
        else A::put(to, ab[i]);
      }
    }
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < cols; c += blockDim.x) {
      float v = 0.0f;
      for (uint32_t k = 0; k < groups; ++k) v += sums[static_cast<size_t>(k) * cols + c];
      out[c] = v;
    }
  }
  if (threadIdx.x == 0 && abort_flag != 0) g_ln_bwd_status = 1;
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
  ptx::pdl_wait();
  ptx::pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t c = static_cast<uint64_t>(blockIdx.x) * 32 + lane, width = 2ull * cols;
  float v = 0.0f;
  if (c < width) {
#pragma unroll 16
    for (uint32_t p = warp; p < parts; p += 8) v += __ldcs(partial + p * width + c);
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
// for beforehand. `aligned`: x and dy start on 16-byte boundaries; `v`: elements per access.
struct Plan {
  int kind = 0;              // 0 ln_bwd_ring, 1 the two-pass form
  int values = 0;            // ln_bwd_ring: values per thread, 8, 16 or 32
  uint32_t tpr = 0, groups = 0, per_group = 1, stages = 0, plane = 0;  // per_group: rows side by side
  uint32_t parts = 1;        // CTAs that leave partial column sums
  uint64_t row_sums_bytes = 0, partial_bytes = 0;
};

// Rows a group takes side by side: two where a row is at most eight values per thread of bf16 ([2097152, 64]: 4.1 -> 5.5
// TB/s; four 3.4). With 16 values a second row would have to read its first half again (8192 columns: 5.2 -> 4.7).
constexpr int ring_rows(int es, int values) { return es == 2 && values == 8 ? 2 : 1; }

Plan make_plan(uint64_t rows, uint32_t cols, int es, bool aligned, int sm = sm_count()) {
  Plan p;
  const uint64_t sms = static_cast<uint64_t>(sm);
  const uint64_t row_bytes = static_cast<uint64_t>(cols) * es;
  if (aligned && cols <= 16384) {
    // 8 values per thread in groups of 8 to 32 threads, then 16, then (rows of more than 8192 columns) 32
    p.values = cols <= 256 ? 8 : cols <= 8192 ? 16 : 32;
    p.tpr = cols <= 64 ? 8 : cols <= 128 ? 16 : cols <= 512 ? 32 : (cols + 32 * p.values - 1) / (32 * p.values) * 32;
    p.groups = 512 / p.tpr;
    if (p.values == 16 && p.tpr > 32 && cols % 2 == 0) {
      // rows that leave many of the 512 threads idle at 16 values per thread: 32 where those keep more of them busy
      // (5120 columns: one group of 320 threads 3.8 TB/s, three of 160 with twice the values 4.7); at equal counts 16 is
      // ahead (8192 columns: 5.2 against 4.8), and so it is for rows of single elements (7001 columns 2.0 against 1.1)
      const uint32_t t32 = (cols + 1023) / 1024 * 32, busy16 = p.tpr * p.groups, busy32 = t32 * (512 / t32);
      if (busy32 > busy16 + 64) {
        p.values = 32;
        p.tpr = t32;
        p.groups = 512 / t32;
      }
    }
    p.per_group = ring_rows(es, p.values);
    if (p.tpr > 32 && rows < sms * p.groups * p.per_group) {  // few rows: over more SMs rather than side by side on one
      const uint64_t want = (rows + sms * p.per_group - 1) / (sms * p.per_group);
      p.groups = static_cast<uint32_t>(want < 1 ? 1 : want);
    }
    p.plane = static_cast<uint32_t>((p.groups * p.per_group * row_bytes + 32 + 127) / 128 * 128);
    p.stages = kRingBytes / (2 * p.plane);
    if (p.stages > kRingStages) p.stages = kRingStages;
  }
  if (p.stages >= 2) {
    const uint64_t chunk_rows = static_cast<uint64_t>(p.groups) * p.per_group, chunks = (rows + chunk_rows - 1) / chunk_rows;
    p.parts = static_cast<uint32_t>(chunks < sms ? chunks : sms);
  } else {
    p.kind = 1;
    const uint64_t strips = (static_cast<uint64_t>(cols) + 255) / 256;  // upper bound: V elements per thread make fewer
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

template <typename T>
struct Call {
  const T *dy, *x, *gamma;
  const float *mean, *rstd;
  T* dx;
  Partials part;
  uint64_t rows;
  uint32_t cols;
  cudaStream_t s;
};

template <typename T, int V, int VALUES, int TPR>
int launch_ring(const Plan& p, const Call<T>& c) {
  auto* fn = ln_bwd_ring<T, V, VALUES / V, TPR, ring_rows(sizeof(T), VALUES), VALUES <= 16>;
  uint32_t smem = 2 * p.plane * p.stages;
  const uint32_t sums = p.groups * c.cols * 4;  // the groups' column sums at the end
  if (smem < sums) smem = sums;
  TCAB_TRY_RC(reserve_smem("layernorm_rows_backward", reinterpret_cast<const void*>(fn), smem));
  launch_pdl(fn, dim3(p.parts), dim3(p.groups * p.tpr), smem, c.s, c.dy, c.x, c.gamma, c.mean, c.rstd, c.dx, c.part, c.rows,
             c.cols, p.tpr, p.groups, p.stages, p.plane);
  count_launch();
  return check_launch("ln_bwd_ring");
}

template <typename T, int V>
int launch_v(const Plan& p, const Call<T>& c) {
  if (p.values == 8) {
    if (p.tpr == 8) return launch_ring<T, V, 8, 8>(p, c);
    if (p.tpr == 16) return launch_ring<T, V, 8, 16>(p, c);
    return launch_ring<T, V, 8, 32>(p, c);
  }
  if (p.values == 16) {
    if (p.tpr == 32) return launch_ring<T, V, 16, 32>(p, c);
    return launch_ring<T, V, 16, 0>(p, c);
  }
  return launch_ring<T, V, 32, 0>(p, c);
}

template <typename T, int VW>
int launch_two_pass(const Plan& p, const Call<T>& c, float2* row_sums, bool vec) {
  const uint64_t most = static_cast<uint64_t>(sm_count()) * 4;
  const unsigned grid = static_cast<unsigned>(c.rows < most ? (c.rows ? c.rows : 1) : most);
  const uint32_t nvec = vec ? c.cols / VW : c.cols;
  const dim3 tiles((nvec + 255) / 256, p.parts);
  if (vec) {
    ln_bwd_sums<T, VW><<<grid, 512, 0, c.s>>>(c.dy, c.x, c.gamma, c.mean, c.rstd, row_sums, c.rows, c.cols);
    ln_bwd_tile<T, VW><<<tiles, 256, 0, c.s>>>(c.dy, c.x, c.gamma, c.mean, c.rstd, row_sums, c.dx, c.part, c.rows, c.cols);
  } else {
    ln_bwd_sums<T, 1><<<grid, 512, 0, c.s>>>(c.dy, c.x, c.gamma, c.mean, c.rstd, row_sums, c.rows, c.cols);
    ln_bwd_tile<T, 1><<<tiles, 256, 0, c.s>>>(c.dy, c.x, c.gamma, c.mean, c.rstd, row_sums, c.dx, c.part, c.rows, c.cols);
  }
  count_launch(2);
  return check_launch("ln_bwd_tile");
}

template <typename T, int VW>
int launch(const T* dy, const T* x, const T* gamma, const float* mean, const float* rstd, T* dx, float* dgamma, float* dbeta,
           uint64_t rows, uint32_t cols, uint8_t* ws, uint64_t ws_bytes, cudaStream_t s) {
  const bool aligned = aligned16(dy) && aligned16(x);
  const Plan p = make_plan(rows, cols, sizeof(T), aligned);
  if (p.row_sums_bytes + p.partial_bytes > ws_bytes)
    return fail(TCAB_ERR_INVALID_ARG, "layernorm_rows_backward: the workspace has %llu bytes, %llu are needed",
                static_cast<unsigned long long>(ws_bytes), static_cast<unsigned long long>(p.row_sums_bytes + p.partial_bytes));
  float* partial = reinterpret_cast<float*>(ws + p.row_sums_bytes);
  Partials part = {dgamma, dbeta, 0};
  if (p.parts > 1) {
    part.pg = partial;
    part.pb = partial + cols;
    part.stride = 2 * static_cast<size_t>(cols);
  }
  const Call<T> c = {dy, x, gamma, mean, rstd, dx, part, rows, cols, s};
  // elements per access: what divides the row and keeps dx and gamma aligned
  auto fits = [&](uint32_t v) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(gamma);
    return cols % v == 0 && a % (v * sizeof(T)) == 0;
  };
  int rc;
  if (p.kind == 1) {
    rc = launch_two_pass<T, VW>(p, c, reinterpret_cast<float2*>(ws), aligned && fits(VW));
  } else if (fits(VW)) {
    rc = launch_v<T, VW>(p, c);
  } else if (VW == 8 && fits(4)) {
    rc = launch_v<T, 4>(p, c);
  } else if (fits(2)) {
    rc = launch_v<T, 2>(p, c);
  } else {
    rc = launch_v<T, 1>(p, c);
  }
  if (rc != TCAB_OK || p.parts <= 1) return rc;
  launch_pdl(ln_bwd_finish, dim3(static_cast<unsigned>((2ull * cols + 31) / 32)), dim3(256), 0, s,
             static_cast<const float*>(partial), p.parts, cols, dgamma, dbeta);
  count_launch();
  return check_launch("ln_bwd_finish");
}

}  // namespace

uint64_t layernorm_backward_workspace(uint64_t rows, uint32_t cols, int elem_bytes) {
  const Plan a = make_plan(rows, cols, elem_bytes, false), b = make_plan(rows, cols, elem_bytes, true);
  const uint64_t na = a.row_sums_bytes + a.partial_bytes, nb = b.row_sums_bytes + b.partial_bytes;
  return na > nb ? na : nb;
}

void layernorm_backward_plan(uint64_t rows, uint32_t cols, int elem_bytes, int aligned, int sms, uint32_t* out) {
  const Plan p = make_plan(rows, cols, elem_bytes, aligned != 0, sms);
  const uint32_t v[8] = {static_cast<uint32_t>(p.kind), static_cast<uint32_t>(p.values), p.tpr, p.groups, p.per_group, p.stages, p.plane, p.parts};
  for (int i = 0; i < 8; ++i) out[i] = v[i];
}

int layernorm_backward_status(int* out) {
  if (cudaMemcpyFromSymbol(out, g_ln_bwd_status, sizeof(int)) != cudaSuccess) {
    cudaGetLastError();
    return fail(TCAB_ERR_CUDA, "device_status: cannot read the status word");
  }
  return TCAB_OK;
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
