// abi.cu -- the extern "C" surface declared in include/tcab.h: argument and shape
// validation, then one launch into the operator-class kernels.
//
// The checks stand where the reference's generated launcher derives every
// extent from its first tensor occurrence and TCA_REQUIREs the others to agree
// (internal/cg/cxx/launch.go:23-156), and where ValidateLaunch traps bad launch
// geometry (runtime/tca/launch.h:37-58). A failure is a status code plus a
// thread-local message; nothing throws across the boundary.
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <map>
#include <mutex>
#include <utility>

#include "../../include/tcab_tuning.h"
#include "common.cuh"
#include "ffn_gemm.h"
#include "rowvec.cuh"

namespace tcab {
namespace {

thread_local char g_err[512] = "";
std::atomic<uint64_t> g_launches{0};
Tune g_tune[kFamilies];

struct DevFacts {
  int sms = 0;
  int optin_smem = 0;
};
std::mutex g_mu;
std::map<int, DevFacts> g_dev;
std::map<std::pair<std::pair<int, const void*>, std::pair<int, size_t>>, int> g_occ;

int current_device() {
  int d = 0;
  if (cudaGetDevice(&d) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  return d;
}

const DevFacts& facts() {
  static const DevFacts none{};
  const int d = current_device();
  if (d < 0) return none;
  std::lock_guard<std::mutex> lk(g_mu);
  auto it = g_dev.find(d);
  if (it == g_dev.end()) {
    DevFacts f;
    cudaDeviceGetAttribute(&f.sms, cudaDevAttrMultiProcessorCount, d);
    cudaDeviceGetAttribute(&f.optin_smem, cudaDevAttrMaxSharedMemoryPerBlockOptin, d);
    it = g_dev.emplace(d, f).first;
  }
  return it->second;
}

}  // namespace

int fail(int status, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  std::vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return status;
}

void count_launch(unsigned n) { g_launches.fetch_add(n, std::memory_order_relaxed); }

int sm_count() {
  const int n = facts().sms;
  return n > 0 ? n : 1;
}

int max_optin_smem() { return facts().optin_smem; }

int check_launch(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(TCAB_ERR_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
  return TCAB_OK;
}

// The attribute belongs to the device's copy of the function and stays set; the largest size asked for is remembered.
int reserve_smem(const char* op, const void* fn, size_t bytes) {
  static std::map<std::pair<int, const void*>, size_t> reserved;
  const auto key = std::make_pair(current_device(), fn);
  std::lock_guard<std::mutex> lk(g_mu);
  size_t& have = reserved[key];
  if (have >= bytes) return TCAB_OK;
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(TCAB_ERR_CUDA, "%s: cannot reserve %zu bytes of shared memory: %s", op, bytes, cudaGetErrorString(e));
  }
  have = bytes;
  return TCAB_OK;
}

const Tune& tune(int family) { return g_tune[family]; }

int occupancy(const void* fn, int block, size_t smem) {
  const int d = current_device();
  const auto key = std::make_pair(std::make_pair(d, fn), std::make_pair(block, smem));
  {
    std::lock_guard<std::mutex> lk(g_mu);
    auto it = g_occ.find(key);
    if (it != g_occ.end()) return it->second;
  }
  int n = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, fn, block, smem) != cudaSuccess) {
    cudaGetLastError();
    n = 1;
  }
  std::lock_guard<std::mutex> lk(g_mu);
  g_occ[key] = n;
  return n;
}

namespace {
struct ScratchBuf {
  void* p = nullptr;
  size_t bytes = 0;
};
std::mutex g_scratch_mu;
std::map<std::pair<std::pair<int, cudaStream_t>, int>, ScratchBuf> g_scratch;
}  // namespace

void* stream_scratch(int kind, cudaStream_t stream, size_t bytes, bool grow, bool zero) {
  const int dev = current_device();
  if (dev < 0) return nullptr;
  std::lock_guard<std::mutex> lk(g_scratch_mu);
  ScratchBuf& b = g_scratch[{{dev, stream}, kind}];
  if (b.p != nullptr && b.bytes >= bytes) return b.p;
  if (b.p != nullptr) {
    if (!grow) return nullptr;
    cudaFree(b.p);
    b = ScratchBuf{};
  }
  if (cudaMalloc(&b.p, bytes) != cudaSuccess || (zero && cudaMemset(b.p, 0, bytes) != cudaSuccess)) {
    cudaGetLastError();
    if (b.p != nullptr) cudaFree(b.p);
    b = ScratchBuf{};
    return nullptr;
  }
  b.bytes = bytes;
  return b.p;
}

namespace {

// Frees the buffers of one (device, stream), or all of them. cudaFree waits for the device to go idle.
void release_scratch(bool all, int dev, cudaStream_t stream) {
  std::lock_guard<std::mutex> lk(g_scratch_mu);
  for (auto it = g_scratch.begin(); it != g_scratch.end();) {
    if (all || (it->first.first.first == dev && it->first.first.second == stream)) {
      if (it->second.p != nullptr) cudaFree(it->second.p);
      it = g_scratch.erase(it);
    } else {
      ++it;
    }
  }
  cudaGetLastError();
}

// ---- validation helpers ----------------------------------------------------

int check_tensor(const char* op, const char* name, const tcab_tensor* t, bool need_data = true) {
  if (t == nullptr) return fail(TCAB_ERR_INVALID_ARG, "%s: tensor '%s' is null", op, name);
  if (t->rank < 1 || t->rank > TCAB_MAX_RANK)
    return fail(TCAB_ERR_INVALID_ARG, "%s: tensor '%s' has rank %u (want 1..%d)", op, name, t->rank, TCAB_MAX_RANK);
  uint64_t n = 1;
  for (uint32_t i = 0; i < t->rank; ++i) {
    n *= t->dims[i];
    if (n >= (1ull << 32))
      return fail(TCAB_ERR_TOO_LARGE, "%s: tensor '%s' has 2^32 or more elements", op, name);
  }
  if (need_data && n > 0 && t->data == nullptr)
    return fail(TCAB_ERR_INVALID_ARG, "%s: tensor '%s' has a null data pointer", op, name);
  return TCAB_OK;
}

uint64_t count(const tcab_tensor* t, uint32_t from, uint32_t to) {
  uint64_t n = 1;
  for (uint32_t i = from; i < to; ++i) n *= t->dims[i];
  return n;
}

bool same_shape(const tcab_tensor* a, const tcab_tensor* b) {
  if (a->rank != b->rank) return false;
  for (uint32_t i = 0; i < a->rank; ++i)
    if (a->dims[i] != b->dims[i]) return false;
  return true;
}

int need_dtype(const char* op, const char* name, const tcab_tensor* t, int dtype, const char* spelled) {
  if (t->dtype != dtype) return fail(TCAB_ERR_DTYPE, "%s: tensor '%s' must be %s", op, name, spelled);
  return TCAB_OK;
}

int need_elem_align(const char* op, const char* name, const tcab_tensor* t, unsigned bytes) {
  if (reinterpret_cast<uintptr_t>(t->data) % bytes != 0)
    return fail(TCAB_ERR_ALIGNMENT, "%s: tensor '%s' is not %u-byte aligned", op, name, bytes);
  return TCAB_OK;
}

// Element types a lambda operand may have (the chain and map classes): 4-byte f32 / i32 / u32, 2-byte bf16.
int need_operand_dtype(const char* op, const char* name, const tcab_tensor* t) {
  if (t->dtype != TCAB_F32 && t->dtype != TCAB_BF16 && t->dtype != TCAB_I32 && t->dtype != TCAB_U32)
    return fail(TCAB_ERR_DTYPE, "%s: tensor '%s' must be f32, bf16, i32 or u32", op, name);
  return need_elem_align(op, name, t, t->dtype == TCAB_BF16 ? 2 : 4);
}

// How an operand of the iteration shape `full` (rank r) is indexed: 0 = by every axis (same shape), 1 = one value
// per row (full's extents with the innermost one = 1), 2 = one row shared by all rows (every extent 1 but the
// innermost), -1 = none of these. The reference lets an operand bind a subset of the live axes
// (pkg/chain.go checkOperand); these are the two subsets the innermost-axis kernels take.
int operand_indexing(const uint32_t* full, uint32_t rank, const tcab_tensor* t) {
  if (t->rank != rank) return -1;
  bool same = true, row = t->dims[rank - 1] == 1, col = t->dims[rank - 1] == full[rank - 1];
  for (uint32_t i = 0; i < rank; ++i) same = same && t->dims[i] == full[i];
  for (uint32_t i = 0; i + 1 < rank; ++i) {
    row = row && t->dims[i] == full[i];
    col = col && t->dims[i] == 1;
  }
  if (same) return 0;
  if (row) return 1;
  if (col && rank > 1) return 2;
  return -1;
}

int have_device(const char* op) {
  if (current_device() < 0) return fail(TCAB_ERR_CUDA, "%s: no CUDA device (this library has no CPU path)", op);
  return TCAB_OK;
}

#define TCAB_TRY(expr)              \
  do {                              \
    const int tcab_rc_ = (expr);    \
    if (tcab_rc_ != TCAB_OK) return tcab_rc_; \
  } while (0)

uint64_t tensor_bytes(const tcab_tensor* t) { return count(t, 0, t->rank) * (t->dtype == TCAB_BF16 ? 2 : 4); }

// Outputs against everything else a call touches: `outs` first, then the inputs. An output may be exactly the input
// may_be[i] where that is given. Null entries are skipped.
struct Named {
  const char* name;
  const tcab_tensor* t;
};
int need_disjoint(const char* op, const Named* outs, int n_outs, const Named* ins, int n_ins, const tcab_tensor* const* shareable = nullptr,
                  int n_shareable = 0) {
  auto overlap = [](const tcab_tensor* a, const tcab_tensor* b) {
    const uintptr_t pa = reinterpret_cast<uintptr_t>(a->data), pb = reinterpret_cast<uintptr_t>(b->data);
    const uint64_t na = tensor_bytes(a), nb = tensor_bytes(b);
    return na > 0 && nb > 0 && pa < pb + nb && pb < pa + na;
  };
  for (int i = 0; i < n_outs; ++i) {
    if (outs[i].t == nullptr) continue;
    for (int j = i + 1; j < n_outs; ++j)
      if (outs[j].t != nullptr && overlap(outs[i].t, outs[j].t))
        return fail(TCAB_ERR_INVALID_ARG, "%s: %s overlaps %s", op, outs[i].name, outs[j].name);
    for (int j = 0; j < n_ins; ++j) {
      if (ins[j].t == nullptr || !overlap(outs[i].t, ins[j].t)) continue;
      bool shared = false;  // the first output alone may be one of `shareable`, from the same address on
      for (int k = 0; i == 0 && k < n_shareable; ++k) shared = shared || (shareable[k] == ins[j].t && outs[i].t->data == ins[j].t->data);
      if (!shared) return fail(TCAB_ERR_INVALID_ARG, "%s: %s overlaps %s", op, outs[i].name, ins[j].name);
    }
  }
  return TCAB_OK;
}

// A workspace against the tensors of its call.
int need_apart(const char* op, const void* ws, uint64_t bytes, const Named* ts, int n) {
  const uintptr_t w = reinterpret_cast<uintptr_t>(ws);
  for (int i = 0; i < n && ws != nullptr && bytes > 0; ++i) {
    if (ts[i].t == nullptr) continue;
    const uintptr_t p = reinterpret_cast<uintptr_t>(ts[i].t->data);
    const uint64_t size = tensor_bytes(ts[i].t);
    if (size > 0 && (p >= w ? p - w < bytes : w - p < size))
      return fail(TCAB_ERR_INVALID_ARG, "%s: the workspace overlaps %s", op, ts[i].name);
  }
  return TCAB_OK;
}

// Extents are walked in 32 bits, a stride past the end included, and are coordinates of tensor maps.
int need_extent(const char* op, const char* name, uint32_t extent) {
  if (extent > 0x7fffffffu) return fail(TCAB_ERR_TOO_LARGE, "%s: an extent of %s is 2^31 or more", op, name);
  return TCAB_OK;
}

// mean / rstd of x's rows: f32, the extents of x without the innermost one (rank-1 x: extent 1).
int check_row_stats(const char* op, const char* name, const tcab_tensor* t, const tcab_tensor* x) {
  TCAB_TRY(check_tensor(op, name, t));
  TCAB_TRY(need_dtype(op, name, t, TCAB_F32, "f32"));
  bool ok = x->rank == 1 ? (t->rank == 1 && t->dims[0] == 1) : t->rank == x->rank - 1;
  for (uint32_t i = 0; ok && x->rank > 1 && i + 1 < x->rank; ++i) ok = t->dims[i] == x->dims[i];
  if (!ok) return fail(TCAB_ERR_SHAPE, "%s: %s must have the extents of x without the innermost one", op, name);
  return need_elem_align(op, name, t, 4);
}

int check_row_param(const char* op, const char* name, const tcab_tensor* t, uint32_t cols, int dtype, const char* spelled) {
  TCAB_TRY(check_tensor(op, name, t));
  TCAB_TRY(need_dtype(op, name, t, dtype, spelled));
  if (t->rank != 1 || t->dims[0] != cols)
    return fail(TCAB_ERR_SHAPE, "%s: %s must be rank 1 with extent %u (the innermost extent of x)", op, name, cols);
  return need_elem_align(op, name, t, dtype == TCAB_F32 ? 4 : 2);
}

// x of the layer-norm forms with statistics.
int check_norm_rows(const char* op, const tcab_tensor* x) {
  TCAB_TRY(check_tensor(op, "x", x));
  if (x->dtype != TCAB_F32 && x->dtype != TCAB_BF16) return fail(TCAB_ERR_DTYPE, "%s: x must be f32 or bf16", op);
  if (x->dims[x->rank - 1] == 0) return fail(TCAB_ERR_SHAPE, "%s: the innermost extent of x must be positive", op);
  TCAB_TRY(need_extent(op, "x", x->dims[x->rank - 1]));
  return need_elem_align(op, "x", x, x->dtype == TCAB_F32 ? 4 : 2);
}

int check_like_x(const char* op, const char* name, const tcab_tensor* t, const tcab_tensor* x) {
  TCAB_TRY(check_tensor(op, name, t));
  if (t->dtype != x->dtype) return fail(TCAB_ERR_DTYPE, "%s: %s must have the element type of x", op, name);
  if (!same_shape(t, x)) return fail(TCAB_ERR_SHAPE, "%s: %s must have the shape of x", op, name);
  return need_elem_align(op, name, t, x->dtype == TCAB_F32 ? 4 : 2);
}

// A bf16 [rows, cols] operand of the feed-forward contractions; optional ones may be null.
int check_matrix(const char* op, const char* name, const tcab_tensor* t, uint32_t rows, uint32_t cols) {
  TCAB_TRY(check_tensor(op, name, t));
  TCAB_TRY(need_dtype(op, name, t, TCAB_BF16, "bf16"));
  if (t->rank != 2 || t->dims[0] != rows || t->dims[1] != cols)
    return fail(TCAB_ERR_SHAPE, "%s: %s must be [%u, %u]", op, name, rows, cols);
  return need_elem_align(op, name, t, 16);
}
int check_matrix_opt(const char* op, const char* name, const tcab_tensor* t, uint32_t rows, uint32_t cols) {
  return t == nullptr ? TCAB_OK : check_matrix(op, name, t, rows, cols);
}
int check_bias_opt(const char* op, const char* name, const tcab_tensor* t, uint32_t n) {
  if (t == nullptr) return TCAB_OK;
  TCAB_TRY(check_tensor(op, name, t));
  TCAB_TRY(need_dtype(op, name, t, TCAB_F32, "f32"));
  if (t->rank != 1 || t->dims[0] != n) return fail(TCAB_ERR_SHAPE, "%s: %s must be [%u]", op, name, n);
  return need_elem_align(op, name, t, 4);
}
// The first two operands of a contraction, a [M,K] and b [K,N]: they name the extents.
int check_contraction(const char* op, const char* an, const tcab_tensor* a, const char* bn, const tcab_tensor* b, uint32_t* m,
                      uint32_t* k, uint32_t* n) {
  TCAB_TRY(check_tensor(op, an, a));
  TCAB_TRY(check_tensor(op, bn, b));
  TCAB_TRY(need_dtype(op, an, a, TCAB_BF16, "bf16"));
  TCAB_TRY(need_dtype(op, bn, b, TCAB_BF16, "bf16"));
  if (a->rank != 2 || b->rank != 2) return fail(TCAB_ERR_SHAPE, "%s: %s and %s must be rank 2", op, an, bn);
  if (b->dims[0] != a->dims[1]) return fail(TCAB_ERR_SHAPE, "%s: %s.Dim(0) must equal %s.Dim(1) (dim k)", op, bn, an);
  *m = a->dims[0];
  *k = a->dims[1];
  *n = b->dims[1];
  for (int i = 0; i < 2; ++i) {
    TCAB_TRY(need_extent(op, an, a->dims[i]));
    TCAB_TRY(need_extent(op, bn, b->dims[i]));
  }
  if (*k % 8 != 0 || *n % 8 != 0)
    return fail(TCAB_ERR_ALIGNMENT, "%s: K and N must be multiples of 8 (16-byte rows for the tensor maps)", op);
  TCAB_TRY(need_elem_align(op, an, a, 16));
  return need_elem_align(op, bn, b, 16);
}
int check_workspace(const char* op, const void* ws, uint64_t have, uint64_t need) {
  if (have < need || (need > 0 && ws == nullptr))
    return fail(TCAB_ERR_INVALID_ARG, "%s: the workspace has %llu bytes, %llu are needed", op,
                static_cast<unsigned long long>(ws != nullptr ? have : 0), static_cast<unsigned long long>(need));
  if (reinterpret_cast<uintptr_t>(ws) % 16 != 0) return fail(TCAB_ERR_ALIGNMENT, "%s: the workspace is not 16-byte aligned", op);
  return TCAB_OK;
}
uint64_t round256(uint64_t b) { return (b + 255) / 256 * 256; }

__nv_bfloat16* bf16_of(const tcab_tensor* t) { return t != nullptr ? static_cast<__nv_bfloat16*>(t->data) : nullptr; }
float* f32_of(const tcab_tensor* t) { return t != nullptr ? static_cast<float*>(t->data) : nullptr; }

}  // namespace
}  // namespace tcab

using namespace tcab;

extern "C" {

const char* tcab_last_error(void) { return g_err; }

const char* tcab_status_string(int status) {
  switch (status) {
    case TCAB_OK: return "ok";
    case TCAB_ERR_INVALID_ARG: return "invalid argument";
    case TCAB_ERR_SHAPE: return "shape mismatch";
    case TCAB_ERR_DTYPE: return "unsupported element type";
    case TCAB_ERR_ALIGNMENT: return "misaligned operand";
    case TCAB_ERR_UNSUPPORTED: return "unsupported by this build";
    case TCAB_ERR_CUDA: return "CUDA failure";
    case TCAB_ERR_TOO_LARGE: return "extent too large";
    default: return "unknown status";
  }
}

int tcab_abi_version(void) { return TCAB_ABI_VERSION; }

uint64_t tcab_launch_count(void) { return g_launches.load(std::memory_order_relaxed); }

int tcab_device_status(int* status) {
  if (status == nullptr) return fail(TCAB_ERR_INVALID_ARG, "device_status: null output");
  TCAB_TRY(have_device("device_status"));
  int gemm = 0, rows = 0, ffn = 0, norm = 0;
  TCAB_TRY(gemm_device_status(&gemm));
  TCAB_TRY(rows_smem_status(&rows));
  TCAB_TRY(ffn_device_status(&ffn));
  TCAB_TRY(layernorm_backward_status(&norm));
  // 1..5: a kernel of gemm_bias_act.cu, 8: one of ffn_gemm.cuh, 16: a shared-memory row kernel, 32: ln_bwd_ring
  *status = gemm != 0 ? gemm : ffn != 0 ? 8 : rows != 0 ? 16 : (norm != 0 ? 32 : 0);
  return TCAB_OK;
}

int tcab_release_stream(void* stream) {
  TCAB_TRY(have_device("release_stream"));
  release_scratch(false, current_device(), static_cast<cudaStream_t>(stream));
  return TCAB_OK;
}

int tcab_release_all(void) {
  release_scratch(true, 0, nullptr);
  return TCAB_OK;
}

namespace {
int prepare_common(const char* op, const tcab_chain* chain, const int32_t* in_dtypes, uint32_t n_ins, int use, int out_dtype,
                   PreparedChain* pc);
}

int tcab_compile_check(const tcab_chain* chain, const int32_t* in_dtypes, uint32_t n_ins, int use, int out_dtype,
                       int row_value_mask, int shared_row_mask, int cell_value_mask) {
  PreparedChain pc;
  TCAB_TRY(prepare_common("compile_check", chain, in_dtypes, n_ins, use, out_dtype, &pc));
  JitSpec sp = pc.spec;
  sp.rb_mask = row_value_mask;
  sp.cb_mask = shared_row_mask;
  sp.cell_mask = cell_value_mask;
  return jit_compile_check(sp);
}

int tcab_chain_prepare(const tcab_chain* chain, const int32_t* in_dtypes, uint32_t n_ins, int use, int out_dtype) {
  const char* op = "chain_prepare";
  PreparedChain pc;
  TCAB_TRY(prepare_common(op, chain, in_dtypes, n_ins, use, out_dtype, &pc));
  TCAB_TRY(have_device(op));
  return warm_chain(pc);
}

namespace {
int prepare_common(const char* op, const tcab_chain* chain, const int32_t* in_dtypes, uint32_t n_ins, int use, int out_dtype,
                   PreparedChain* pcp) {
  PreparedChain& pc = *pcp;
  if (chain == nullptr || chain->map_expr == nullptr)
    return fail(TCAB_ERR_INVALID_ARG, "%s: chain and map_expr are required", op);
  if (use != TCAB_USE_REDUCE && use != TCAB_USE_CONTRACT && use != TCAB_USE_MAP && use != TCAB_USE_REDUCE_BATCHED)
    return fail(TCAB_ERR_INVALID_ARG, "%s: unknown use %d", op, use);
  if (use != TCAB_USE_MAP && chain->combine_expr == nullptr) return fail(TCAB_ERR_INVALID_ARG, "%s: combine_expr is required", op);
  if (chain->n_captures > TCAB_MAX_CAPTURES)
    return fail(TCAB_ERR_INVALID_ARG, "%s: %u captures (at most %d)", op, chain->n_captures, TCAB_MAX_CAPTURES);
  if (n_ins < 1 || n_ins > TCAB_MAX_INPUTS || (use == TCAB_USE_CONTRACT && n_ins != 2))
    return fail(TCAB_ERR_INVALID_ARG, "%s: bad operand count %u", op, n_ins);
  int types[TCAB_MAX_INPUTS] = {};  // TCAB_F32 == 0
  for (uint32_t i = 0; i < n_ins && in_dtypes != nullptr; ++i) {
    if (in_dtypes[i] < TCAB_F32 || in_dtypes[i] > TCAB_U32) return fail(TCAB_ERR_DTYPE, "%s: in_dtypes[%u] is not a tcab_dtype", op, i);
    types[i] = in_dtypes[i];
  }
  if (use == TCAB_USE_MAP && (out_dtype < TCAB_F32 || out_dtype > TCAB_U32)) return fail(TCAB_ERR_DTYPE, "%s: out_dtype is not a tcab_dtype", op);
  TCAB_TRY(prepare_chain(chain, n_ins, &pc, use == TCAB_USE_MAP ? 'M' : use == TCAB_USE_CONTRACT ? 'C' : 'R', types,
                         use == TCAB_USE_MAP ? out_dtype : TCAB_F32));
  if (use == TCAB_USE_REDUCE_BATCHED) pc.spec.kind = 'B';
  return TCAB_OK;
}
}  // namespace

int tcab_tune(const char* family, int p0, int p1, int p2, int p3) {
  static const char* names[kFamilies] = {"softmax", "layernorm", "reduce_inner", "reduce_outer", "gemm", "ffn"};
  if (family == nullptr) return fail(TCAB_ERR_INVALID_ARG, "tune: null family");
  for (int i = 0; i < kFamilies; ++i) {
    if (std::strcmp(family, names[i]) == 0) {
      g_tune[i].p0 = p0 > 0 ? p0 : 0;
      g_tune[i].p1 = p1 > 0 ? p1 : 0;
      g_tune[i].p2 = p2 > 0 ? p2 : 0;
      g_tune[i].p3 = p3 > 0 ? p3 : 0;
      return TCAB_OK;
    }
  }
  return fail(TCAB_ERR_INVALID_ARG, "tune: unknown family '%s'", family);
}

int tcab_plan_outer_split(uint64_t tiles, uint64_t cells, uint32_t nk, uint64_t resident_ctas, int sms, int forced,
                          uint32_t* ranges, uint32_t* klen) {
  if (ranges == nullptr || klen == nullptr) return fail(TCAB_ERR_INVALID_ARG, "plan_outer_split: null output");
  if (sms < 1) return fail(TCAB_ERR_INVALID_ARG, "plan_outer_split: sms must be positive");
  plan_outer_ranges(plan_outer_splits(tiles, cells, nk, resident_ctas, sms, forced), nk, ranges, klen);
  return TCAB_OK;
}

int tcab_plan_row_kernels(uint64_t rows_or_batches, uint32_t nk, uint32_t nc, int sms, uint32_t nvec, uint32_t per_step,
                          int prefer_three, int n_in, uint32_t* outer_flat_g, uint32_t* stream_cluster, uint32_t* rows32) {
  if (outer_flat_g == nullptr || stream_cluster == nullptr || rows32 == nullptr)
    return fail(TCAB_ERR_INVALID_ARG, "plan_row_kernels: null output");
  if (sms < 1 || per_step < 1) return fail(TCAB_ERR_INVALID_ARG, "plan_row_kernels: sms and per_step must be positive");
  *outer_flat_g = outer_flat_groups(rows_or_batches, nk, nc, sms, nc % 4 == 0);
  *stream_cluster = stream_cluster_size(nvec, per_step, prefer_three != 0);
  *rows32 = rows32_warps(nvec, n_in);
  return TCAB_OK;
}

int tcab_plan_row_shape(int op, int elem_bytes, uint32_t nvec, uint32_t* threads_per_row, uint32_t* slots_per_thread) {
  if (threads_per_row == nullptr || slots_per_thread == nullptr) return fail(TCAB_ERR_INVALID_ARG, "plan_row_shape: null output");
  if ((op != 0 && op != 1) || (elem_bytes != 2 && elem_bytes != 4) || (op == 0 && elem_bytes != 4))
    return fail(TCAB_ERR_INVALID_ARG, "plan_row_shape: op 0 (softmax, 4-byte elements) or 1 (layer-norm, 2 or 4)");
  int t = 0, v = 0;
  const bool fits = op == 0 ? tcab::softmax_row_shape(nvec, true, &t, &v) : tcab::layernorm_row_shape(nvec, true, elem_bytes, &t, &v);
  *threads_per_row = fits ? static_cast<uint32_t>(t) : 0;
  *slots_per_thread = fits ? static_cast<uint32_t>(v) : 0;
  return TCAB_OK;
}

int tcab_plan_outer_flat_ranges(uint64_t batches, uint32_t nk, uint32_t nc, int sms, uint64_t max_partials,
                                uint32_t* groups, uint32_t* ranges, uint32_t* klen) {
  if (groups == nullptr || ranges == nullptr || klen == nullptr)
    return fail(TCAB_ERR_INVALID_ARG, "plan_outer_flat_ranges: null output");
  if (sms < 1) return fail(TCAB_ERR_INVALID_ARG, "plan_outer_flat_ranges: sms must be positive");
  *groups = outer_flat_groups(batches, nk, nc, sms, nc % 4 == 0);
  *ranges = 1;
  *klen = nk;
  if (*groups != 0) *ranges = outer_flat_ranges(batches, nk, nc, *groups, nc % 4 == 0, sms, max_partials, klen);
  return TCAB_OK;
}

int tcab_plan_ffn(int form, uint32_t m, uint32_t n, uint32_t k, uint32_t pairs, int sms, uint32_t* rows, uint32_t* cols, uint32_t* ranges,
                  uint32_t* blocks) {
  if (rows == nullptr || cols == nullptr || ranges == nullptr || blocks == nullptr) return fail(TCAB_ERR_INVALID_ARG, "plan_ffn: null output");
  if (form < kFfnFwd || form > kFfnDw || pairs < 1 || pairs > 2 || sms < 1)
    return fail(TCAB_ERR_INVALID_ARG, "plan_ffn: form 0..3, one or two pairs, a positive SM count");
  ffn_plan(form, m, n, k, pairs, sms, rows, cols, ranges, blocks);
  return TCAB_OK;
}

int tcab_plan_layernorm_backward(uint64_t rows, uint32_t cols, int elem_bytes, int aligned, int sms, uint32_t* out) {
  if (out == nullptr) return fail(TCAB_ERR_INVALID_ARG, "plan_layernorm_backward: null output");
  if (cols < 1 || sms < 1 || (elem_bytes != 2 && elem_bytes != 4))
    return fail(TCAB_ERR_INVALID_ARG, "plan_layernorm_backward: positive cols and sms, elements of 2 or 4 bytes");
  layernorm_backward_plan(rows, cols, elem_bytes, aligned, sms, out);
  return TCAB_OK;
}

int tcab_softmax_rows(const tcab_tensor* x, const tcab_tensor* y, void* stream) {
  const char* op = "softmax_rows";
  TCAB_TRY(check_tensor(op, "x", x));
  TCAB_TRY(check_tensor(op, "y", y));
  TCAB_TRY(need_dtype(op, "x", x, TCAB_F32, "f32"));
  TCAB_TRY(need_dtype(op, "y", y, TCAB_F32, "f32"));
  if (!same_shape(x, y)) return fail(TCAB_ERR_SHAPE, "%s: y must have the shape of x", op);
  TCAB_TRY(need_elem_align(op, "x", x, 4));
  TCAB_TRY(need_elem_align(op, "y", y, 4));
  TCAB_TRY(have_device(op));
  const uint32_t cols = x->dims[x->rank - 1];
  return launch_softmax_rows(static_cast<const float*>(x->data), static_cast<float*>(y->data),
                             count(x, 0, x->rank - 1), cols, static_cast<cudaStream_t>(stream));
}

int tcab_layernorm_rows(const tcab_tensor* x, const tcab_tensor* gamma, const tcab_tensor* beta, float eps,
                        const tcab_tensor* y, void* stream) {
  const char* op = "layernorm_rows";
  TCAB_TRY(check_tensor(op, "x", x));
  TCAB_TRY(check_tensor(op, "gamma", gamma));
  TCAB_TRY(check_tensor(op, "beta", beta));
  TCAB_TRY(check_tensor(op, "y", y));
  if (x->dtype != TCAB_F32 && x->dtype != TCAB_BF16) return fail(TCAB_ERR_DTYPE, "%s: x must be f32 or bf16", op);
  if (y->dtype != x->dtype || gamma->dtype != x->dtype || beta->dtype != x->dtype)
    return fail(TCAB_ERR_DTYPE, "%s: gamma, beta and y must have the element type of x", op);
  if (!same_shape(x, y)) return fail(TCAB_ERR_SHAPE, "%s: y must have the shape of x", op);
  const uint32_t cols = x->dims[x->rank - 1];
  if (gamma->rank != 1 || gamma->dims[0] != cols)
    return fail(TCAB_ERR_SHAPE, "%s: gamma must be rank 1 with extent %u (the innermost extent of x)", op, cols);
  if (beta->rank != 1 || beta->dims[0] != cols)
    return fail(TCAB_ERR_SHAPE, "%s: beta must be rank 1 with extent %u (the innermost extent of x)", op, cols);
  const unsigned es = x->dtype == TCAB_F32 ? 4 : 2;
  TCAB_TRY(need_elem_align(op, "x", x, es));
  TCAB_TRY(need_elem_align(op, "y", y, es));
  TCAB_TRY(need_elem_align(op, "gamma", gamma, es));
  TCAB_TRY(need_elem_align(op, "beta", beta, es));
  TCAB_TRY(have_device(op));
  const uint64_t rows = count(x, 0, x->rank - 1);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (x->dtype == TCAB_BF16)
    return launch_layernorm_rows_bf16(static_cast<const __nv_bfloat16*>(x->data),
                                      static_cast<const __nv_bfloat16*>(gamma->data),
                                      static_cast<const __nv_bfloat16*>(beta->data), eps,
                                      static_cast<__nv_bfloat16*>(y->data), RowStats{}, rows, cols, s);
  return launch_layernorm_rows_f32(static_cast<const float*>(x->data), static_cast<const float*>(gamma->data),
                                   static_cast<const float*>(beta->data), eps, static_cast<float*>(y->data), RowStats{}, rows,
                                   cols, s);
}

int tcab_reduce_outer(const tcab_tensor* t, const tcab_tensor* sum, const tcab_tensor* max,
                      const tcab_tensor* argmax, void* stream) {
  const char* op = "reduce_outer";
  TCAB_TRY(check_tensor(op, "t", t));
  TCAB_TRY(need_dtype(op, "t", t, TCAB_F32, "f32"));
  if (t->rank != 3) return fail(TCAB_ERR_SHAPE, "%s: t must be rank 3 [b, k, c]", op);
  if (sum == nullptr && max == nullptr && argmax == nullptr)
    return fail(TCAB_ERR_INVALID_ARG, "%s: at least one of sum, max, argmax is required", op);
  const tcab_tensor* outs[3] = {sum, max, argmax};
  const char* names[3] = {"sum", "max", "argmax"};
  for (int i = 0; i < 3; ++i) {
    if (outs[i] == nullptr) continue;
    TCAB_TRY(check_tensor(op, names[i], outs[i]));
    TCAB_TRY(need_dtype(op, names[i], outs[i], i == 2 ? TCAB_I32 : TCAB_F32, i == 2 ? "i32" : "f32"));
    if (outs[i]->rank != 2 || outs[i]->dims[0] != t->dims[0] || outs[i]->dims[1] != t->dims[2])
      return fail(TCAB_ERR_SHAPE, "%s: %s must be [%u, %u]", op, names[i], t->dims[0], t->dims[2]);
    TCAB_TRY(need_elem_align(op, names[i], outs[i], 4));
  }
  TCAB_TRY(need_elem_align(op, "t", t, 4));
  TCAB_TRY(have_device(op));
  return launch_reduce_outer(static_cast<const float*>(t->data), sum ? static_cast<float*>(sum->data) : nullptr,
                             max ? static_cast<float*>(max->data) : nullptr,
                             argmax ? static_cast<int32_t*>(argmax->data) : nullptr, t->dims[0], t->dims[1],
                             t->dims[2], static_cast<cudaStream_t>(stream));
}

int tcab_chain_reduce(const tcab_chain* chain, const tcab_tensor* ins, uint32_t n_ins, uint32_t reduce_axis,
                      const tcab_tensor* out, void* stream) {
  const char* op = "chain_reduce";
  if (chain == nullptr || chain->map_expr == nullptr || chain->combine_expr == nullptr)
    return fail(TCAB_ERR_INVALID_ARG, "%s: chain, map_expr and combine_expr are required", op);
  if (chain->n_captures > TCAB_MAX_CAPTURES)
    return fail(TCAB_ERR_INVALID_ARG, "%s: %u captures (at most %d)", op, chain->n_captures, TCAB_MAX_CAPTURES);
  if (ins == nullptr || n_ins < 1 || n_ins > TCAB_MAX_INPUTS)
    return fail(TCAB_ERR_INVALID_ARG, "%s: between 1 and %d operands are required", op, TCAB_MAX_INPUTS);
  const float* ptrs[TCAB_MAX_INPUTS] = {};
  int types[TCAB_MAX_INPUTS] = {};  // TCAB_F32 == 0
  for (uint32_t i = 0; i < n_ins; ++i) {
    char name[16];
    std::snprintf(name, sizeof(name), "ins[%u]", i);
    TCAB_TRY(check_tensor(op, name, &ins[i]));
    TCAB_TRY(need_operand_dtype(op, name, &ins[i]));
    if (ins[i].rank != ins[0].rank) return fail(TCAB_ERR_SHAPE, "%s: %s must have the rank of ins[0]", op, name);
    ptrs[i] = static_cast<const float*>(ins[i].data);
    types[i] = ins[i].dtype;
  }
  // the iteration shape: per axis the largest extent among the operands; an operand may have extent 1 along the
  // innermost axis (one value per row) or along every other axis (one row shared by all rows)
  tcab_tensor full = ins[0];
  for (uint32_t i = 1; i < n_ins; ++i)
    for (uint32_t d = 0; d < full.rank; ++d)
      if (ins[i].dims[d] > full.dims[d]) full.dims[d] = ins[i].dims[d];
  if (reduce_axis >= full.rank) return fail(TCAB_ERR_INVALID_ARG, "%s: reduce_axis %u out of range", op, reduce_axis);
  int rb = 0, cb = 0, cells = 0;
  for (uint32_t i = 0; i < n_ins; ++i) {
    int how = operand_indexing(full.dims, full.rank, &ins[i]);
    if (how != 0 && reduce_axis != full.rank - 1) {
      // a middle-axis reduction: an operand may lack the REDUCED axis (extent 1 there, the common extents elsewhere):
      // one value per output cell
      bool cell = ins[i].dims[reduce_axis] == 1;
      for (uint32_t d = 0; cell && d < full.rank; ++d) cell = d == reduce_axis || ins[i].dims[d] == full.dims[d];
      if (!cell)
        return fail(TCAB_ERR_SHAPE, "%s: ins[%u] must have the operands' common shape, or extent 1 along the reduced axis", op, i);
      cells |= 1 << i;
      continue;
    }
    if (how < 0)
      return fail(TCAB_ERR_SHAPE, "%s: ins[%u] must have the operands' common shape, or extent 1 along the innermost axis, "
                  "or extent 1 along every other axis", op, i);
    rb |= (how == 1) << i;
    cb |= (how == 2) << i;
  }
  const tcab_tensor* t = &full;
  TCAB_TRY(check_tensor(op, "out", out));
  TCAB_TRY(need_dtype(op, "out", out, TCAB_F32, "f32"));
  TCAB_TRY(need_elem_align(op, "out", out, 4));
  // out = the operands' extents minus the reduced axis (rank 1 -> [1]).
  uint32_t want[TCAB_MAX_RANK], wr = 0;
  for (uint32_t i = 0; i < t->rank; ++i)
    if (i != reduce_axis) want[wr++] = t->dims[i];
  if (wr == 0) want[wr++] = 1;
  bool ok = out->rank == wr;
  for (uint32_t i = 0; ok && i < wr; ++i) ok = out->dims[i] == want[i];
  if (!ok) return fail(TCAB_ERR_SHAPE, "%s: out must have the operands' extents without axis %u", op, reduce_axis);
  PreparedChain pc;
  TCAB_TRY(prepare_chain(chain, n_ins, &pc, 'R', types, TCAB_F32, rb, cb, cells));
  TCAB_TRY(have_device(op));
  return launch_chain_reduce(pc, ptrs, count(t, 0, reduce_axis), t->dims[reduce_axis],
                             count(t, reduce_axis + 1, t->rank), static_cast<float*>(out->data),
                             static_cast<cudaStream_t>(stream));
}

int tcab_chain_reduce_batched(const tcab_chain* chain, const tcab_tensor* ins, uint32_t n_ins, uint32_t n_problems,
                              const tcab_tensor* outs, void* stream) {
  const char* op = "chain_reduce_batched";
  if (chain == nullptr || chain->map_expr == nullptr || chain->combine_expr == nullptr)
    return fail(TCAB_ERR_INVALID_ARG, "%s: chain, map_expr and combine_expr are required", op);
  if (chain->n_captures > TCAB_MAX_CAPTURES)
    return fail(TCAB_ERR_INVALID_ARG, "%s: %u captures (at most %d)", op, chain->n_captures, TCAB_MAX_CAPTURES);
  if (ins == nullptr || outs == nullptr || n_ins < 1 || n_ins > TCAB_MAX_INPUTS)
    return fail(TCAB_ERR_INVALID_ARG, "%s: between 1 and %d operands per problem are required", op, TCAB_MAX_INPUTS);
  if (n_problems < 1 || n_problems > TCAB_MAX_BATCH)
    return fail(TCAB_ERR_TOO_LARGE, "%s: %u problems (between 1 and %d per call)", op, n_problems, TCAB_MAX_BATCH);
  const float* ptrs[TCAB_MAX_BATCH * TCAB_MAX_INPUTS] = {};
  float* optrs[TCAB_MAX_BATCH] = {};
  int types[TCAB_MAX_INPUTS] = {};  // TCAB_F32 == 0
  const tcab_tensor* t0 = &ins[0];
  for (uint32_t b = 0; b < n_problems; ++b) {
    for (uint32_t i = 0; i < n_ins; ++i) {
      const tcab_tensor* t = &ins[b * n_ins + i];
      char name[32];
      std::snprintf(name, sizeof(name), "ins[%u][%u]", b, i);
      TCAB_TRY(check_tensor(op, name, t));
      TCAB_TRY(need_operand_dtype(op, name, t));
      if (!same_shape(t0, t)) return fail(TCAB_ERR_SHAPE, "%s: %s must have the shape of ins[0][0]", op, name);
      if (b == 0) types[i] = t->dtype;
      else if (t->dtype != types[i]) return fail(TCAB_ERR_DTYPE, "%s: %s must have the element type of ins[0][%u]", op, name, i);
      ptrs[b * n_ins + i] = static_cast<const float*>(t->data);
    }
    const tcab_tensor* o = &outs[b];
    char name[32];
    std::snprintf(name, sizeof(name), "outs[%u]", b);
    TCAB_TRY(check_tensor(op, name, o));
    TCAB_TRY(need_dtype(op, name, o, TCAB_F32, "f32"));
    TCAB_TRY(need_elem_align(op, name, o, 4));
    bool ok = t0->rank == 1 ? (o->rank == 1 && o->dims[0] == 1) : o->rank == t0->rank - 1;
    for (uint32_t i = 0; ok && t0->rank > 1 && i + 1 < t0->rank; ++i) ok = o->dims[i] == t0->dims[i];
    if (!ok) return fail(TCAB_ERR_SHAPE, "%s: %s must have the operands' extents without the innermost axis", op, name);
    optrs[b] = static_cast<float*>(o->data);
  }
  PreparedChain pc;
  TCAB_TRY(prepare_chain(chain, n_ins, &pc, 'R', types));
  TCAB_TRY(have_device(op));
  return launch_chain_reduce_batched(pc, ptrs, optrs, n_problems, static_cast<uint32_t>(count(t0, 0, t0->rank - 1)),
                                     t0->dims[t0->rank - 1], static_cast<cudaStream_t>(stream));
}

int tcab_chain_reduce_noalloc(const tcab_chain* chain, const tcab_tensor* ins, uint32_t n_ins,
                              const tcab_tensor* out, void* stream) {
  const char* op = "chain_reduce_noalloc";
  if (chain == nullptr || chain->map_expr == nullptr || chain->combine_expr == nullptr)
    return fail(TCAB_ERR_INVALID_ARG, "%s: chain, map_expr and combine_expr are required", op);
  if (chain->n_captures > TCAB_MAX_CAPTURES)
    return fail(TCAB_ERR_INVALID_ARG, "%s: %u captures (at most %d)", op, chain->n_captures, TCAB_MAX_CAPTURES);
  if (ins == nullptr || n_ins < 1 || n_ins > TCAB_MAX_INPUTS)
    return fail(TCAB_ERR_INVALID_ARG, "%s: between 1 and %d operands are required", op, TCAB_MAX_INPUTS);
  const float* ptrs[TCAB_MAX_INPUTS] = {};
  int types[TCAB_MAX_INPUTS] = {};  // TCAB_F32 == 0
  for (uint32_t i = 0; i < n_ins; ++i) {
    char name[16];
    std::snprintf(name, sizeof(name), "ins[%u]", i);
    TCAB_TRY(check_tensor(op, name, &ins[i]));
    TCAB_TRY(need_operand_dtype(op, name, &ins[i]));
    if (i > 0 && !same_shape(&ins[0], &ins[i]))
      return fail(TCAB_ERR_SHAPE, "%s: %s must have the shape of ins[0]", op, name);
    ptrs[i] = static_cast<const float*>(ins[i].data);
    types[i] = ins[i].dtype;
  }
  const tcab_tensor* t = &ins[0];
  TCAB_TRY(check_tensor(op, "out", out));
  TCAB_TRY(need_dtype(op, "out", out, TCAB_F32, "f32"));
  TCAB_TRY(need_elem_align(op, "out", out, 4));
  const uint64_t rows = count(t, 0, t->rank - 1);
  bool ok = t->rank == 1 ? (out->rank == 1 && out->dims[0] == 1) : out->rank == t->rank - 1;
  for (uint32_t i = 0; ok && t->rank > 1 && i + 1 < t->rank; ++i) ok = out->dims[i] == t->dims[i];
  if (!ok) return fail(TCAB_ERR_SHAPE, "%s: out must have the operands' extents without the innermost axis", op);
  if (rows > TCAB_NOALLOC_MAX_ROWS)
    return fail(TCAB_ERR_TOO_LARGE,
                "%s: %llu rows exceed TCAB_NOALLOC_MAX_ROWS = %d (the fixed scratch array); use tcab_chain_reduce",
                op, static_cast<unsigned long long>(rows), TCAB_NOALLOC_MAX_ROWS);
  PreparedChain pc;
  TCAB_TRY(prepare_chain(chain, n_ins, &pc, 'R', types));
  TCAB_TRY(have_device(op));
  return launch_chain_reduce_noalloc(pc, ptrs, rows, t->dims[t->rank - 1], static_cast<float*>(out->data),
                                     static_cast<cudaStream_t>(stream));
}

int tcab_map(const tcab_chain* chain, const tcab_tensor* ins, uint32_t n_ins, const tcab_tensor* out, void* stream) {
  const char* op = "map";
  if (chain == nullptr || chain->map_expr == nullptr) return fail(TCAB_ERR_INVALID_ARG, "%s: chain and map_expr are required", op);
  if (chain->n_captures > TCAB_MAX_CAPTURES)
    return fail(TCAB_ERR_INVALID_ARG, "%s: %u captures (at most %d)", op, chain->n_captures, TCAB_MAX_CAPTURES);
  if (ins == nullptr || n_ins < 1 || n_ins > TCAB_MAX_INPUTS)
    return fail(TCAB_ERR_INVALID_ARG, "%s: between 1 and %d operands are required", op, TCAB_MAX_INPUTS);
  TCAB_TRY(check_tensor(op, "out", out));
  TCAB_TRY(need_operand_dtype(op, "out", out));
  const void* ptrs[TCAB_MAX_INPUTS] = {};
  int types[TCAB_MAX_INPUTS] = {};  // TCAB_F32 == 0
  int rb = 0, cb = 0;
  for (uint32_t i = 0; i < n_ins; ++i) {
    char name[16];
    std::snprintf(name, sizeof(name), "ins[%u]", i);
    TCAB_TRY(check_tensor(op, name, &ins[i]));
    TCAB_TRY(need_operand_dtype(op, name, &ins[i]));
    const int how = operand_indexing(out->dims, out->rank, &ins[i]);
    if (how < 0)
      return fail(TCAB_ERR_SHAPE, "%s: %s must have the shape of out, or extent 1 along the innermost axis (one value per "
                  "row), or extent 1 along every other axis (one row shared by all rows)", op, name);
    rb |= (how == 1) << i;
    cb |= (how == 2) << i;
    ptrs[i] = ins[i].data;
    types[i] = ins[i].dtype;
  }
  PreparedChain pc;
  TCAB_TRY(prepare_chain(chain, n_ins, &pc, 'M', types, out->dtype, rb, cb));
  TCAB_TRY(have_device(op));
  return launch_chain_map(pc, ptrs, out->data, count(out, 0, out->rank), out->dims[out->rank - 1],
                          static_cast<cudaStream_t>(stream));
}

int tcab_chain_contract(const tcab_chain* chain, const tcab_tensor* lhs, const tcab_tensor* rhs, int rhs_is_nk,
                        const tcab_tensor* out, void* stream) {
  const char* op = "chain_contract";
  if (chain == nullptr || chain->map_expr == nullptr || chain->combine_expr == nullptr)
    return fail(TCAB_ERR_INVALID_ARG, "%s: chain, map_expr and combine_expr are required", op);
  if (chain->n_captures > TCAB_MAX_CAPTURES)
    return fail(TCAB_ERR_INVALID_ARG, "%s: %u captures (at most %d)", op, chain->n_captures, TCAB_MAX_CAPTURES);
  TCAB_TRY(check_tensor(op, "lhs", lhs));
  TCAB_TRY(check_tensor(op, "rhs", rhs));
  TCAB_TRY(check_tensor(op, "out", out));
  TCAB_TRY(need_operand_dtype(op, "lhs", lhs));
  TCAB_TRY(need_operand_dtype(op, "rhs", rhs));
  TCAB_TRY(need_dtype(op, "out", out, TCAB_F32, "f32"));
  if (lhs->rank != 2 || rhs->rank != 2 || out->rank != 2)
    return fail(TCAB_ERR_SHAPE, "%s: lhs, rhs and out must be rank 2", op);
  const uint32_t m = lhs->dims[0], k = lhs->dims[1];
  const uint32_t rk = rhs_is_nk ? rhs->dims[1] : rhs->dims[0], n = rhs_is_nk ? rhs->dims[0] : rhs->dims[1];
  if (rk != k) return fail(TCAB_ERR_SHAPE, "%s: rhs.Dim(%d) must equal lhs.Dim(1) (dim k)", op, rhs_is_nk ? 1 : 0);
  if (out->dims[0] != m || out->dims[1] != n) return fail(TCAB_ERR_SHAPE, "%s: out must be [%u, %u]", op, m, n);
  TCAB_TRY(need_elem_align(op, "out", out, 4));
  const int types[2] = {lhs->dtype, rhs->dtype};
  PreparedChain pc;
  TCAB_TRY(prepare_chain(chain, 2, &pc, 'C', types));
  TCAB_TRY(have_device(op));
  return launch_chain_contract(pc, static_cast<const float*>(lhs->data), static_cast<const float*>(rhs->data),
                               rhs_is_nk ? 1 : 0, static_cast<float*>(out->data), m, n, k,
                               static_cast<cudaStream_t>(stream));
}

int tcab_gemm_bias_act(const tcab_tensor* a, const tcab_tensor* b, const tcab_tensor* bias, int act,
                       const tcab_tensor* c, void* stream) {
  const char* op = "gemm_bias_act";
  TCAB_TRY(check_tensor(op, "a", a));
  TCAB_TRY(check_tensor(op, "b", b));
  TCAB_TRY(check_tensor(op, "c", c));
  TCAB_TRY(need_dtype(op, "a", a, TCAB_BF16, "bf16"));
  TCAB_TRY(need_dtype(op, "b", b, TCAB_BF16, "bf16"));
  TCAB_TRY(need_dtype(op, "c", c, TCAB_BF16, "bf16"));
  if (a->rank != 2 || b->rank != 2 || c->rank != 2) return fail(TCAB_ERR_SHAPE, "%s: a, b and c must be rank 2", op);
  const uint32_t m = a->dims[0], k = a->dims[1], n = b->dims[1];
  if (b->dims[0] != k) return fail(TCAB_ERR_SHAPE, "%s: b.Dim(0) must equal a.Dim(1) (dim k)", op);
  if (c->dims[0] != m || c->dims[1] != n) return fail(TCAB_ERR_SHAPE, "%s: c must be [%u, %u]", op, m, n);
  if (bias != nullptr) {
    TCAB_TRY(check_tensor(op, "bias", bias));
    TCAB_TRY(need_dtype(op, "bias", bias, TCAB_F32, "f32"));
    if (bias->rank != 1 || bias->dims[0] != n) return fail(TCAB_ERR_SHAPE, "%s: bias must be [%u]", op, n);
    TCAB_TRY(need_elem_align(op, "bias", bias, 4));
  }
  if (act != TCAB_ACT_NONE && act != TCAB_ACT_RELU) return fail(TCAB_ERR_INVALID_ARG, "%s: unknown activation %d", op, act);
  if (k % 8 != 0 || n % 8 != 0)
    return fail(TCAB_ERR_ALIGNMENT, "%s: K and N must be multiples of 8 (16-byte rows for the tensor maps)", op);
  TCAB_TRY(need_elem_align(op, "a", a, 16));
  TCAB_TRY(need_elem_align(op, "b", b, 16));
  TCAB_TRY(need_elem_align(op, "c", c, 16));
  TCAB_TRY(have_device(op));
  return launch_gemm_bias_act(static_cast<const __nv_bfloat16*>(a->data), static_cast<const __nv_bfloat16*>(b->data),
                              bias ? static_cast<const float*>(bias->data) : nullptr, act,
                              static_cast<__nv_bfloat16*>(c->data), m, n, k, static_cast<cudaStream_t>(stream));
}

int tcab_layernorm_rows_stats(const tcab_tensor* x, const tcab_tensor* gamma, const tcab_tensor* beta, float eps,
                              const tcab_tensor* y, const tcab_tensor* mean, const tcab_tensor* rstd, void* stream) {
  const char* op = "layernorm_rows_stats";
  TCAB_TRY(check_norm_rows(op, x));
  const uint32_t cols = x->dims[x->rank - 1];
  TCAB_TRY(check_like_x(op, "y", y, x));
  TCAB_TRY(check_row_param(op, "gamma", gamma, cols, x->dtype, "the element type of x"));
  TCAB_TRY(check_row_param(op, "beta", beta, cols, x->dtype, "the element type of x"));
  TCAB_TRY(check_row_stats(op, "mean", mean, x));
  TCAB_TRY(check_row_stats(op, "rstd", rstd, x));
  const Named outs[] = {{"y", y}, {"mean", mean}, {"rstd", rstd}}, ins[] = {{"x", x}, {"gamma", gamma}, {"beta", beta}};
  const tcab_tensor* may_be[] = {x};
  TCAB_TRY(need_disjoint(op, outs, 3, ins, 3, may_be, 1));
  TCAB_TRY(have_device(op));
  const uint64_t rows = count(x, 0, x->rank - 1);
  const RowStats st = {f32_of(mean), f32_of(rstd)};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (x->dtype == TCAB_BF16)
    return launch_layernorm_rows_bf16(bf16_of(x), bf16_of(gamma), bf16_of(beta), eps, bf16_of(y), st, rows, cols, s);
  return launch_layernorm_rows_f32(f32_of(x), f32_of(gamma), f32_of(beta), eps, f32_of(y), st, rows, cols, s);
}

uint64_t tcab_layernorm_rows_backward_workspace(const tcab_tensor* x) {
  if (x == nullptr || x->rank < 1 || x->rank > TCAB_MAX_RANK || (x->dtype != TCAB_F32 && x->dtype != TCAB_BF16)) return 0;
  const uint32_t cols = x->dims[x->rank - 1];
  return cols == 0 ? 0 : layernorm_backward_workspace(count(x, 0, x->rank - 1), cols, x->dtype == TCAB_F32 ? 4 : 2);
}

int tcab_layernorm_rows_backward(const tcab_tensor* dy, const tcab_tensor* x, const tcab_tensor* gamma, const tcab_tensor* mean,
                                 const tcab_tensor* rstd, const tcab_tensor* dx, const tcab_tensor* dgamma,
                                 const tcab_tensor* dbeta, void* workspace, uint64_t workspace_bytes, void* stream) {
  const char* op = "layernorm_rows_backward";
  TCAB_TRY(check_norm_rows(op, x));
  const uint32_t cols = x->dims[x->rank - 1];
  TCAB_TRY(check_like_x(op, "dy", dy, x));
  TCAB_TRY(check_like_x(op, "dx", dx, x));
  TCAB_TRY(check_row_param(op, "gamma", gamma, cols, x->dtype, "the element type of x"));
  TCAB_TRY(check_row_stats(op, "mean", mean, x));
  TCAB_TRY(check_row_stats(op, "rstd", rstd, x));
  TCAB_TRY(check_row_param(op, "dgamma", dgamma, cols, TCAB_F32, "f32"));
  TCAB_TRY(check_row_param(op, "dbeta", dbeta, cols, TCAB_F32, "f32"));
  const Named outs[] = {{"dx", dx}, {"dgamma", dgamma}, {"dbeta", dbeta}};
  const Named ins[] = {{"dy", dy}, {"x", x}, {"gamma", gamma}, {"mean", mean}, {"rstd", rstd}};
  const tcab_tensor* may_be[] = {dy, x};
  TCAB_TRY(need_disjoint(op, outs, 3, ins, 5, may_be, 2));
  TCAB_TRY(need_apart(op, workspace, workspace_bytes, outs, 3));
  TCAB_TRY(need_apart(op, workspace, workspace_bytes, ins, 5));
  TCAB_TRY(have_device(op));
  TCAB_TRY(check_workspace(op, workspace, workspace_bytes, tcab_layernorm_rows_backward_workspace(x)));
  const uint64_t rows = count(x, 0, x->rank - 1);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (x->dtype == TCAB_BF16)
    return launch_layernorm_backward_bf16(bf16_of(dy), bf16_of(x), bf16_of(gamma), f32_of(mean), f32_of(rstd), bf16_of(dx),
                                          f32_of(dgamma), f32_of(dbeta), rows, cols, workspace, workspace_bytes, s);
  return launch_layernorm_backward_f32(f32_of(dy), f32_of(x), f32_of(gamma), f32_of(mean), f32_of(rstd), f32_of(dx),
                                       f32_of(dgamma), f32_of(dbeta), rows, cols, workspace, workspace_bytes, s);
}

int tcab_gemm_bias_act_residual(const tcab_tensor* a, const tcab_tensor* b, const tcab_tensor* bias, const tcab_tensor* residual,
                                int act, const tcab_tensor* preact, const tcab_tensor* c, void* stream) {
  const char* op = "gemm_bias_act_residual";
  uint32_t m = 0, k = 0, n = 0;
  TCAB_TRY(check_contraction(op, "a", a, "b", b, &m, &k, &n));
  TCAB_TRY(check_matrix(op, "c", c, m, n));
  TCAB_TRY(check_matrix_opt(op, "residual", residual, m, n));
  TCAB_TRY(check_matrix_opt(op, "preact", preact, m, n));
  TCAB_TRY(check_bias_opt(op, "bias", bias, n));
  if (act < TCAB_ACT_NONE || act > TCAB_ACT_GELU_TANH) return fail(TCAB_ERR_INVALID_ARG, "%s: unknown activation %d", op, act);
  const Named outs[] = {{"c", c}, {"preact", preact}}, ins[] = {{"a", a}, {"b", b}, {"bias", bias}, {"residual", residual}};
  const tcab_tensor* may_be[] = {residual};
  TCAB_TRY(need_disjoint(op, outs, 2, ins, 4, may_be, residual != nullptr ? 1 : 0));
  TCAB_TRY(have_device(op));
  FfnProblem p;
  p.a[0] = bf16_of(a);
  p.b[0] = bf16_of(b);
  p.c[0] = bf16_of(c);
  p.z[0] = bf16_of(preact);
  p.bias[0] = f32_of(bias);
  p.residual = bf16_of(residual);
  p.M = m;
  p.N = n;
  p.K = k;
  p.act = act;
  return launch_ffn_gemm(op, kFfnFwd, p, static_cast<cudaStream_t>(stream));
}

uint64_t tcab_gemm_bias_act_backward_workspace(uint32_t m, uint32_t n, int act, int with_dbias) {
  const uint64_t dz = act == TCAB_ACT_NONE ? 0 : round256(2ull * m * n);
  return dz + (with_dbias ? round256(act_backward_workspace(m, n, 0)) : 0);
}

int tcab_gemm_bias_act_backward(const tcab_tensor* dc, const tcab_tensor* a, const tcab_tensor* b, const tcab_tensor* preact,
                                int act, const tcab_tensor* da, const tcab_tensor* db, const tcab_tensor* dbias,
                                void* workspace, uint64_t workspace_bytes, void* stream) {
  const char* op = "gemm_bias_act_backward";
  uint32_t m = 0, k = 0, n = 0;
  TCAB_TRY(check_contraction(op, "a", a, "b", b, &m, &k, &n));
  TCAB_TRY(check_matrix(op, "dc", dc, m, n));
  if (act < TCAB_ACT_NONE || act > TCAB_ACT_GELU_TANH) return fail(TCAB_ERR_INVALID_ARG, "%s: unknown activation %d", op, act);
  if (act != TCAB_ACT_NONE && preact == nullptr)
    return fail(TCAB_ERR_INVALID_ARG, "%s: preact is required for every activation but none", op);
  TCAB_TRY(check_matrix_opt(op, "preact", preact, m, n));
  TCAB_TRY(check_matrix_opt(op, "da", da, m, k));
  TCAB_TRY(check_matrix_opt(op, "db", db, k, n));
  TCAB_TRY(check_bias_opt(op, "dbias", dbias, n));
  const Named outs[] = {{"da", da}, {"db", db}, {"dbias", dbias}}, ins[] = {{"dc", dc}, {"a", a}, {"b", b}, {"preact", preact}};
  TCAB_TRY(need_disjoint(op, outs, 3, ins, 4));
  TCAB_TRY(need_apart(op, workspace, workspace_bytes, outs, 3));
  TCAB_TRY(need_apart(op, workspace, workspace_bytes, ins, 4));
  TCAB_TRY(have_device(op));
  TCAB_TRY(check_workspace(op, workspace, workspace_bytes, tcab_gemm_bias_act_backward_workspace(m, n, act, dbias != nullptr)));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const __nv_bfloat16* dz = bf16_of(dc);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const bool contract = da != nullptr || db != nullptr;
  bool beside = false;  // the last launch of this call so far, if there is one, does not write dz
  if (act != TCAB_ACT_NONE && (contract || dbias != nullptr)) {
    __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(ws);
    TCAB_TRY(launch_act_backward(op, act, dz, bf16_of(preact), contract ? to : nullptr, f32_of(dbias), m, n, ws + round256(2ull * m * n), s));
    dz = to;
    beside = dbias != nullptr && n > 0 && act_backward_finishes(m, n, 0);
  } else if (dbias != nullptr) {
    TCAB_TRY(launch_act_backward(op, TCAB_ACT_NONE, dz, nullptr, nullptr, f32_of(dbias), m, n, ws, s));
    beside = n > 0;
  }
  FfnTaken taken;
  if (da != nullptr) {
    FfnProblem p;
    p.a[0] = dz;
    p.b[0] = bf16_of(b);
    p.c[0] = bf16_of(da);
    p.M = m;
    p.N = k;
    p.K = n;
    p.beside = beside;
    TCAB_TRY(launch_ffn_gemm(op, kFfnDx, p, s, &taken));
    beside = beside || (m > 0 && k > 0);
  }
  if (db != nullptr) {
    FfnProblem p;
    p.a[0] = bf16_of(a);
    p.b[0] = dz;
    p.c[0] = bf16_of(db);
    p.M = k;
    p.N = n;
    p.K = m;
    p.beside = beside;
    p.taken = taken.sms;
    p.taken_us = taken.us;
    TCAB_TRY(launch_ffn_gemm(op, kFfnDw, p, s));
  }
  return TCAB_OK;
}

int tcab_gated_gemm(const tcab_tensor* x, const tcab_tensor* w_gate, const tcab_tensor* w_up, const tcab_tensor* bias_gate,
                    const tcab_tensor* bias_up, int act, const tcab_tensor* gate, const tcab_tensor* up, const tcab_tensor* h,
                    void* stream) {
  const char* op = "gated_gemm";
  uint32_t m = 0, k = 0, n = 0;
  TCAB_TRY(check_contraction(op, "x", x, "w_gate", w_gate, &m, &k, &n));
  TCAB_TRY(check_matrix(op, "w_up", w_up, k, n));
  TCAB_TRY(check_matrix(op, "h", h, m, n));
  if ((gate == nullptr) != (up == nullptr)) return fail(TCAB_ERR_INVALID_ARG, "%s: gate and up are stored both or neither", op);
  if ((bias_gate == nullptr) != (bias_up == nullptr)) return fail(TCAB_ERR_INVALID_ARG, "%s: bias_gate and bias_up come both or neither", op);
  TCAB_TRY(check_matrix_opt(op, "gate", gate, m, n));
  TCAB_TRY(check_matrix_opt(op, "up", up, m, n));
  TCAB_TRY(check_bias_opt(op, "bias_gate", bias_gate, n));
  TCAB_TRY(check_bias_opt(op, "bias_up", bias_up, n));
  if (act < TCAB_ACT_RELU || act > TCAB_ACT_SIGMOID) return fail(TCAB_ERR_INVALID_ARG, "%s: unknown activation %d", op, act);
  const Named outs[] = {{"h", h}, {"gate", gate}, {"up", up}};
  const Named ins[] = {{"x", x}, {"w_gate", w_gate}, {"w_up", w_up}, {"bias_gate", bias_gate}, {"bias_up", bias_up}};
  TCAB_TRY(need_disjoint(op, outs, 3, ins, 5));
  TCAB_TRY(have_device(op));
  FfnProblem p;
  p.a[0] = bf16_of(x);
  p.b[0] = bf16_of(w_gate);
  p.b[1] = bf16_of(w_up);
  p.c[0] = bf16_of(h);
  p.z[0] = bf16_of(gate);
  p.z[1] = bf16_of(up);
  p.bias[0] = f32_of(bias_gate);
  p.bias[1] = f32_of(bias_up);
  p.M = m;
  p.N = n;
  p.K = k;
  p.act = act;
  return launch_ffn_gemm(op, kFfnGated, p, static_cast<cudaStream_t>(stream));
}

uint64_t tcab_gated_gemm_backward_workspace(uint32_t m, uint32_t n, int with_dbias) {
  return 2 * round256(2ull * m * n) + (with_dbias ? round256(act_backward_workspace(m, n, 1)) : 0);
}

int tcab_gated_gemm_backward(const tcab_tensor* dh, const tcab_tensor* x, const tcab_tensor* w_gate, const tcab_tensor* w_up,
                             const tcab_tensor* gate, const tcab_tensor* up, int act, const tcab_tensor* dx,
                             const tcab_tensor* dw_gate, const tcab_tensor* dw_up, const tcab_tensor* dbias_gate,
                             const tcab_tensor* dbias_up, void* workspace, uint64_t workspace_bytes, void* stream) {
  const char* op = "gated_gemm_backward";
  uint32_t m = 0, k = 0, n = 0;
  TCAB_TRY(check_contraction(op, "x", x, "w_gate", w_gate, &m, &k, &n));
  TCAB_TRY(check_matrix(op, "w_up", w_up, k, n));
  TCAB_TRY(check_matrix(op, "dh", dh, m, n));
  TCAB_TRY(check_matrix(op, "gate", gate, m, n));
  TCAB_TRY(check_matrix(op, "up", up, m, n));
  if (act < TCAB_ACT_RELU || act > TCAB_ACT_SIGMOID) return fail(TCAB_ERR_INVALID_ARG, "%s: unknown activation %d", op, act);
  if ((dw_gate == nullptr) != (dw_up == nullptr)) return fail(TCAB_ERR_INVALID_ARG, "%s: dw_gate and dw_up come both or neither", op);
  if ((dbias_gate == nullptr) != (dbias_up == nullptr))
    return fail(TCAB_ERR_INVALID_ARG, "%s: dbias_gate and dbias_up come both or neither", op);
  TCAB_TRY(check_matrix_opt(op, "dx", dx, m, k));
  TCAB_TRY(check_matrix_opt(op, "dw_gate", dw_gate, k, n));
  TCAB_TRY(check_matrix_opt(op, "dw_up", dw_up, k, n));
  TCAB_TRY(check_bias_opt(op, "dbias_gate", dbias_gate, n));
  TCAB_TRY(check_bias_opt(op, "dbias_up", dbias_up, n));
  const Named outs[] = {{"dx", dx}, {"dw_gate", dw_gate}, {"dw_up", dw_up}, {"dbias_gate", dbias_gate}, {"dbias_up", dbias_up}};
  const Named ins[] = {{"dh", dh}, {"x", x}, {"w_gate", w_gate}, {"w_up", w_up}, {"gate", gate}, {"up", up}};
  TCAB_TRY(need_disjoint(op, outs, 5, ins, 6));
  TCAB_TRY(need_apart(op, workspace, workspace_bytes, outs, 5));
  TCAB_TRY(need_apart(op, workspace, workspace_bytes, ins, 6));
  TCAB_TRY(have_device(op));
  TCAB_TRY(check_workspace(op, workspace, workspace_bytes, tcab_gated_gemm_backward_workspace(m, n, dbias_gate != nullptr)));
  if (dx == nullptr && dw_gate == nullptr && dbias_gate == nullptr) return TCAB_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const uint64_t plane = round256(2ull * m * n);
  __nv_bfloat16* dgate = reinterpret_cast<__nv_bfloat16*>(ws);
  __nv_bfloat16* dup = reinterpret_cast<__nv_bfloat16*>(ws + plane);
  TCAB_TRY(launch_gated_backward(op, act, bf16_of(dh), bf16_of(gate), bf16_of(up), dgate, dup, f32_of(dbias_gate), f32_of(dbias_up),
                                 m, n, ws + 2 * plane, s));
  bool beside = dbias_gate != nullptr && n > 0;  // the last launch of this call so far, if there is one, writes neither
  FfnTaken taken;
  if (dx != nullptr) {
    FfnProblem p;
    p.a[0] = dgate;
    p.a[1] = dup;
    p.b[0] = bf16_of(w_gate);
    p.b[1] = bf16_of(w_up);
    p.c[0] = bf16_of(dx);
    p.M = m;
    p.N = k;
    p.K = n;
    p.beside = beside;
    TCAB_TRY(launch_ffn_gemm(op, kFfnDx, p, s, &taken));
    beside = beside || (m > 0 && k > 0);
  }
  if (dw_gate != nullptr) {
    FfnProblem p;
    p.a[0] = bf16_of(x);
    p.b[0] = dgate;
    p.b[1] = dup;
    p.c[0] = bf16_of(dw_gate);
    p.c[1] = bf16_of(dw_up);
    p.M = k;
    p.N = n;
    p.K = m;
    p.beside = beside;
    p.taken = taken.sms;
    p.taken_us = taken.us;
    TCAB_TRY(launch_ffn_gemm(op, kFfnDw, p, s));
  }
  return TCAB_OK;
}

}  // extern "C"
