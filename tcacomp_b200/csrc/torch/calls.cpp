// calls.cpp -- the feed-forward operators' host path from torch tensors to the C ABI (include/tcab.h), as a Python extension
// module: five to eleven tensors per call are viewed, one to four outputs and a workspace allocated from torch's allocator.
// The functions take every argument by position; ops.py gives them their names, defaults and activation codes.
//
// Why native: with ctypes views a call of one launch cost 10 to 13 us of host time, 3 to 4 of which were the C ABI with
// the launch itself (a library product through torch: 8.7), and that time is what a step over few tokens is made of.
//
// What is refused is refused by the Python checks: a tensor that the fast view does not take goes to `slow` (ops.py), which
// raises or, for one that is only unusual (empty), returns its view as bytes. The library's own status codes raise through
// `check`. Nothing is linked against libtcab.so: bind() receives the addresses that the one loaded copy has.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>

#include "../../../include/tcab.h"

namespace {

PyObject *g_slow = nullptr, *g_check = nullptr;

struct Table {
  decltype(&tcab_layernorm_rows_stats) ln_stats;
  decltype(&tcab_layernorm_rows_backward) ln_backward;
  decltype(&tcab_layernorm_rows_backward_workspace) ln_backward_ws;
  decltype(&tcab_gemm_bias_act_residual) gemm;
  decltype(&tcab_gemm_bias_act_backward) gemm_backward;
  decltype(&tcab_gemm_bias_act_backward_workspace) gemm_backward_ws;
  decltype(&tcab_gated_gemm) gated;
  decltype(&tcab_gated_gemm_backward) gated_backward;
  decltype(&tcab_gated_gemm_backward_workspace) gated_backward_ws;
} g_fn = {};

struct Raised {};  // a Python exception is set

// A view of one operand; null where it is None.
struct View {
  tcab_tensor v;
  bool given = false;
  const tcab_tensor* ptr() const { return given ? &v : nullptr; }
};

bool fill(const at::Tensor& t, int dev, tcab_tensor* v) {
  if (!t.defined() || t.layout() != c10::kStrided || !t.is_cuda() || t.get_device() != dev || !t.is_contiguous()) return false;
  const auto type = t.scalar_type();
  if (type != at::kBFloat16 && type != at::kFloat) return false;
  const int64_t n = t.numel(), rank = t.dim();
  if (n <= 0 || n >= (int64_t{1} << 32) || rank < 1 || rank > TCAB_MAX_RANK) return false;
  v->data = t.data_ptr();
  v->dtype = type == at::kFloat ? TCAB_F32 : TCAB_BF16;
  v->rank = static_cast<uint32_t>(rank);
  for (int64_t i = 0; i < rank; ++i) v->dims[i] = static_cast<uint32_t>(t.size(i));
  return true;
}

void slow(PyObject* o, const char* name, int dev, tcab_tensor* v) {
  PyObject* b = PyObject_CallFunction(g_slow, "Osi", o, name, dev);
  if (b == nullptr) throw Raised();
  const bool ok = PyBytes_Check(b) && PyBytes_GET_SIZE(b) == static_cast<Py_ssize_t>(sizeof(tcab_tensor));
  if (ok) std::memcpy(v, PyBytes_AS_STRING(b), sizeof(tcab_tensor));
  Py_DECREF(b);
  if (!ok) {
    PyErr_SetString(PyExc_RuntimeError, "a tensor's view is not one tcab_tensor");
    throw Raised();
  }
}

View view(PyObject* o, const char* name, int dev) {
  View w;
  if (o == Py_None) return w;
  w.given = true;
  if (!THPVariable_Check(o) || !fill(THPVariable_Unpack(o), dev, &w.v)) slow(o, name, dev, &w.v);
  return w;
}
// An operand that may not be None: `slow` refuses that.
View need(PyObject* o, const char* name, int dev) {
  View w;
  w.given = true;
  if (!THPVariable_Check(o) || !fill(THPVariable_Unpack(o), dev, &w.v)) slow(o, name, dev, &w.v);
  return w;
}

// The device of a call's first operand.
int device_of(PyObject* o, const char* name) {
  if (THPVariable_Check(o)) {
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.is_cuda()) return static_cast<int>(t.get_device());
  }
  tcab_tensor v;
  slow(o, name, 0, &v);  // raises
  PyErr_Format(PyExc_ValueError, "%s must live on a CUDA device", name);
  throw Raised();
}

// An output: the caller's, a new one for True (or, where `always`, for None), none for None.
struct Output {
  View w;
  at::Tensor made;
  PyObject* given = nullptr;
  PyObject* take() const {
    if (made.defined()) return THPVariable_Wrap(made);
    PyObject* o = given != nullptr ? given : Py_None;
    Py_INCREF(o);
    return o;
  }
};

at::Tensor make(const int64_t* dims, int rank, at::ScalarType type, int dev) {
  int64_t strides[TCAB_MAX_RANK];
  int64_t s = 1;
  for (int i = rank - 1; i >= 0; --i) {
    strides[i] = s;
    s *= dims[i] > 0 ? dims[i] : 1;
  }
  return at::detail::empty_strided_cuda(at::IntArrayRef(dims, rank), at::IntArrayRef(strides, rank), type,
                                        c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(dev)));
}

Output output(PyObject* o, const char* name, const int64_t* dims, int rank, at::ScalarType type, int dev, bool always) {
  Output r;
  if (o == Py_True || (always && o == Py_None)) {
    r.made = make(dims, rank, type, dev);
    r.w.given = true;
    if (!fill(r.made, dev, &r.w.v)) {  // empty, or 2^32 elements and more
      PyObject* t = THPVariable_Wrap(r.made);
      if (t == nullptr) throw Raised();
      try {
        slow(t, name, dev, &r.w.v);
      } catch (...) {
        Py_DECREF(t);
        throw;
      }
      Py_DECREF(t);
    }
  } else if (o != Py_None) {
    r.given = o;
    r.w = need(o, name, dev);
  }
  return r;
}

void matrices(const View& a, const char* an, const View& b, const char* bn) {
  if (a.v.rank == 2 && b.v.rank == 2) return;
  PyErr_Format(PyExc_ValueError, "%s must be a rank-2 tensor", a.v.rank != 2 ? an : bn);
  throw Raised();
}

at::ScalarType type_of(const View& x) { return x.v.dtype == TCAB_F32 ? at::kFloat : at::kBFloat16; }

// A workspace for the call's length: it belongs to the current stream, which the call's work is on.
struct Workspace {
  at::Tensor t;
  uint64_t bytes;
  Workspace(uint64_t n, int dev) : bytes(n) {
    const int64_t dims[1] = {static_cast<int64_t>(n)};
    if (n > 0) t = make(dims, 1, at::kByte, dev);
  }
  void* ptr() const { return bytes > 0 ? t.data_ptr() : nullptr; }
};

template <typename F>
void run(F&& f) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f();
  Py_END_ALLOW_THREADS
  if (rc == TCAB_OK) return;
  PyObject* r = PyObject_CallFunction(g_check, "i", rc);
  if (r != nullptr) {
    Py_DECREF(r);
    PyErr_Format(PyExc_RuntimeError, "status %d", rc);
  }
  throw Raised();
}

void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream(); }

PyObject* tuple_of(std::initializer_list<const Output*> outs) {
  PyObject* t = PyTuple_New(static_cast<Py_ssize_t>(outs.size()));
  if (t == nullptr) throw Raised();
  Py_ssize_t i = 0;
  for (const Output* o : outs) {
    PyObject* v = o->take();
    if (v == nullptr) {
      Py_DECREF(t);
      throw Raised();
    }
    PyTuple_SET_ITEM(t, i++, v);
  }
  return t;
}

int code_of(PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised();
  return static_cast<int>(v);
}

struct Stats {
  int64_t dims[TCAB_MAX_RANK];
  int rank;
};
Stats stats_shape(const View& x) {
  Stats s;
  s.rank = x.v.rank > 1 ? static_cast<int>(x.v.rank) - 1 : 1;
  s.dims[0] = 1;
  for (uint32_t i = 0; i + 1 < x.v.rank; ++i) s.dims[i] = x.v.dims[i];
  return s;
}

// (x, gamma, beta, eps, out, mean, rstd) -> (out, mean, rstd)
PyObject* ln_stats(PyObject* const* a) {
  const int dev = device_of(a[0], "x");
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  const View x = need(a[0], "x", dev), gamma = need(a[1], "gamma", dev), beta = need(a[2], "beta", dev);
  const double eps = PyFloat_AsDouble(a[3]);
  if (eps == -1.0 && PyErr_Occurred()) throw Raised();
  int64_t dims[TCAB_MAX_RANK];
  for (uint32_t i = 0; i < x.v.rank; ++i) dims[i] = x.v.dims[i];
  const Stats s = stats_shape(x);
  const Output y = output(a[4], "out", dims, static_cast<int>(x.v.rank), type_of(x), dev, true);
  const Output mean = output(a[5], "mean", s.dims, s.rank, at::kFloat, dev, true);
  const Output rstd = output(a[6], "rstd", s.dims, s.rank, at::kFloat, dev, true);
  void* st = stream_of(dev);
  run([&] {
    return g_fn.ln_stats(x.ptr(), gamma.ptr(), beta.ptr(), static_cast<float>(eps), y.w.ptr(), mean.w.ptr(), rstd.w.ptr(), st);
  });
  return tuple_of({&y, &mean, &rstd});
}

// (dy, x, gamma, mean, rstd, dx, dgamma, dbeta) -> (dx, dgamma, dbeta)
PyObject* ln_backward(PyObject* const* a) {
  const int dev = device_of(a[1], "x");
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  const View x = need(a[1], "x", dev), dy = need(a[0], "dy", dev), gamma = need(a[2], "gamma", dev);
  const View mean = need(a[3], "mean", dev), rstd = need(a[4], "rstd", dev);
  int64_t dims[TCAB_MAX_RANK];
  for (uint32_t i = 0; i < x.v.rank; ++i) dims[i] = x.v.dims[i];
  const int64_t cols[1] = {dims[x.v.rank - 1]};
  const Output dx = output(a[5], "dx", dims, static_cast<int>(x.v.rank), type_of(x), dev, true);
  const Output dgamma = output(a[6], "dgamma", cols, 1, at::kFloat, dev, true);
  const Output dbeta = output(a[7], "dbeta", cols, 1, at::kFloat, dev, true);
  const Workspace ws(g_fn.ln_backward_ws(x.ptr()), dev);
  void* st = stream_of(dev);
  run([&] {
    return g_fn.ln_backward(dy.ptr(), x.ptr(), gamma.ptr(), mean.ptr(), rstd.ptr(), dx.w.ptr(), dgamma.w.ptr(), dbeta.w.ptr(), ws.ptr(),
                            ws.bytes, st);
  });
  return tuple_of({&dx, &dgamma, &dbeta});
}

// (a, b, bias, residual, act, out, preact) -> out
PyObject* gemm(PyObject* const* p) {
  const int dev = device_of(p[0], "a");
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  const View a = need(p[0], "a", dev), b = need(p[1], "b", dev);
  matrices(a, "a", b, "b");
  const View bias = view(p[2], "bias", dev), residual = view(p[3], "residual", dev), preact = view(p[6], "preact", dev);
  const int act = code_of(p[4]);
  const int64_t dims[2] = {a.v.dims[0], b.v.dims[1]};
  const Output c = output(p[5], "out", dims, 2, at::kBFloat16, dev, true);
  void* st = stream_of(dev);
  run([&] { return g_fn.gemm(a.ptr(), b.ptr(), bias.ptr(), residual.ptr(), act, preact.ptr(), c.w.ptr(), st); });
  return c.take();
}

// (dc, a, b, preact, act, da, db, dbias) -> (da, db, dbias); an output is given, asked for (True) or not wanted (None)
PyObject* gemm_backward(PyObject* const* p) {
  const int dev = device_of(p[1], "a");
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  const View a = need(p[1], "a", dev), b = need(p[2], "b", dev);
  matrices(a, "a", b, "b");
  const View dc = need(p[0], "dc", dev), preact = view(p[3], "preact", dev);
  const int act = code_of(p[4]);
  const int64_t m = a.v.dims[0], k = a.v.dims[1], n = b.v.dims[1], mk[2] = {m, k}, kn[2] = {k, n};
  const Output da = output(p[5], "da", mk, 2, at::kBFloat16, dev, false), db = output(p[6], "db", kn, 2, at::kBFloat16, dev, false);
  const Output dbias = output(p[7], "dbias", &n, 1, at::kFloat, dev, false);
  const Workspace ws(g_fn.gemm_backward_ws(a.v.dims[0], b.v.dims[1], act, dbias.w.given), dev);
  void* st = stream_of(dev);
  run([&] {
    return g_fn.gemm_backward(dc.ptr(), a.ptr(), b.ptr(), preact.ptr(), act, da.w.ptr(), db.w.ptr(), dbias.w.ptr(), ws.ptr(), ws.bytes, st);
  });
  return tuple_of({&da, &db, &dbias});
}

// (x, w_gate, w_up, bias_gate, bias_up, act, out, gate, up) -> out
PyObject* gated(PyObject* const* p) {
  const int dev = device_of(p[0], "x");
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  const View x = need(p[0], "x", dev), wg = need(p[1], "w_gate", dev);
  matrices(x, "x", wg, "w_gate");
  const View wu = need(p[2], "w_up", dev), bg = view(p[3], "bias_gate", dev), bu = view(p[4], "bias_up", dev);
  const View gate = view(p[7], "gate", dev), up = view(p[8], "up", dev);
  const int act = code_of(p[5]);
  const int64_t dims[2] = {x.v.dims[0], wg.v.dims[1]};
  const Output h = output(p[6], "out", dims, 2, at::kBFloat16, dev, true);
  void* st = stream_of(dev);
  run([&] { return g_fn.gated(x.ptr(), wg.ptr(), wu.ptr(), bg.ptr(), bu.ptr(), act, gate.ptr(), up.ptr(), h.w.ptr(), st); });
  return h.take();
}

// (dh, x, w_gate, w_up, gate, up, act, dx, dw_gate, dw_up, dbias_gate, dbias_up) -> the last five
PyObject* gated_backward(PyObject* const* p) {
  const int dev = device_of(p[1], "x");
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  const View x = need(p[1], "x", dev), wg = need(p[2], "w_gate", dev);
  matrices(x, "x", wg, "w_gate");
  const View dh = need(p[0], "dh", dev), wu = need(p[3], "w_up", dev), gate = need(p[4], "gate", dev), up = need(p[5], "up", dev);
  const int act = code_of(p[6]);
  const int64_t m = x.v.dims[0], k = x.v.dims[1], n = wg.v.dims[1], mk[2] = {m, k}, kn[2] = {k, n};
  const Output dx = output(p[7], "dx", mk, 2, at::kBFloat16, dev, false);
  const Output dwg = output(p[8], "dw_gate", kn, 2, at::kBFloat16, dev, false), dwu = output(p[9], "dw_up", kn, 2, at::kBFloat16, dev, false);
  const Output dbg = output(p[10], "dbias_gate", &n, 1, at::kFloat, dev, false), dbu = output(p[11], "dbias_up", &n, 1, at::kFloat, dev, false);
  const Workspace ws(g_fn.gated_backward_ws(x.v.dims[0], wg.v.dims[1], dbg.w.given || dbu.w.given), dev);
  void* st = stream_of(dev);
  run([&] {
    return g_fn.gated_backward(dh.ptr(), x.ptr(), wg.ptr(), wu.ptr(), gate.ptr(), up.ptr(), act, dx.w.ptr(), dwg.w.ptr(), dwu.w.ptr(),
                               dbg.w.ptr(), dbu.w.ptr(), ws.ptr(), ws.bytes, st);
  });
  return tuple_of({&dx, &dwg, &dwu, &dbg, &dbu});
}

// One Python entry: the argument count, and C++ exceptions turned into Python's.
template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) return PyErr_Format(PyExc_TypeError, "%zd arguments, %zd expected", n, N);
  HANDLE_TH_ERRORS
  try {
    return F(args);
  } catch (const Raised&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// bind(slow, check, address, ...): the addresses in the order of Table
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  constexpr Py_ssize_t kN = sizeof(Table) / sizeof(void*);
  if (n != 2 + kN) return PyErr_Format(PyExc_TypeError, "%zd arguments, %zd expected", n, 2 + kN);
  void* at[kN];
  for (Py_ssize_t i = 0; i < kN; ++i) {
    at[i] = PyLong_AsVoidPtr(args[2 + i]);
    if (at[i] == nullptr) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "a null address");
  }
  std::memcpy(&g_fn, at, sizeof(g_fn));
  Py_INCREF(args[0]);
  Py_INCREF(args[1]);
  Py_XSETREF(g_slow, args[0]);
  Py_XSETREF(g_check, args[1]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind)), METH_FASTCALL, nullptr},
#define TCAB_ENTRY(F, N) {#F, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<F, N>)), METH_FASTCALL, nullptr}
    TCAB_ENTRY(ln_stats, 7), TCAB_ENTRY(ln_backward, 8), TCAB_ENTRY(gemm, 7), TCAB_ENTRY(gemm_backward, 8), TCAB_ENTRY(gated, 9),
    TCAB_ENTRY(gated_backward, 12),
#undef TCAB_ENTRY
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
