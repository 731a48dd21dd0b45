// binding.cpp -- the Python side of the small operators (ecad_amd/_ops.so): argument checks of EcadEngine.op_quantize_int8 / op_gemm_int8 / op_gate_norm / op_rope_table / op_rope and the
// call into libecad_hip.so.  These launches take 3 to 5 us on the device; the same checks in Python took 8 to 15 us a call (a dozen tensors at half a microsecond each,
// two allocations at 1.6), here 1 to 2.  Everything that a call may not be given is refused here or in the library: what torch keeps beside a tensor's memory (gradients,
// tangents, traces, lazy signs) does not get past check().  Host code only: the operators are the library's, reached through the C ABI of include/ecad_hip.h.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/TracerMode.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

#include <chrono>
#include <cstdarg>
#include <memory>
#include <string>
#include <thread>
#include <utility>

#include "../../include/ecad_hip.h"

namespace {

using at::Tensor;

// What an engine gives its calls: the library's entry points, its handle, dtype and device.
struct Engine {
  decltype(&ecad_op_quantize_int8) quantize;
  decltype(&ecad_op_gemm_int8) gemm;
  decltype(&ecad_op_gate_norm) norm;
  decltype(&ecad_op_rope_table) table;
  decltype(&ecad_op_rope) rope;
  decltype(&ecad_last_error) last_error;
  EcadEngine* handle;
  at::ScalarType dtype;
  c10::Device device{c10::DeviceType::CPU};
  PyObject* stream_of;  // callable(device index) -> hipStream_t as an integer
  PyObject* index;
  int running = 0;      // calls in the library; read and written with the interpreter's lock
  bool closed = false;
};
const char* const ENGINE = "ecad_amd._ops.Engine";

struct Refused {
  std::string message;
};
[[noreturn]] void refuse(const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  throw Refused{buf};
}
std::string text(at::IntArrayRef v) {
  std::string s = "(";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + (v.size() == 1 ? ",)" : ")");
}

// ---- arguments ---------------------------------------------------------------------------------------------------------------------------------------------------

// These calls pass torch's dispatcher by: a tracer would see the allocation of a result and nothing that fills it.
void refuse_tracing() {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  const bool recorded = Modes::any_modes_set() && (Modes::get_mode(Key::PROXY) || Modes::get_mode(Key::FAKE) || Modes::get_mode(Key::FUNCTIONAL));
  if (recorded || at::tracer::impl::is_dispatch_enabled()) throw std::runtime_error("this op cannot be traced: it is a call into the library that a recorded graph would not hold");
}

Engine& held(PyObject* o) {
  void* p = PyCapsule_GetPointer(o, ENGINE);
  if (!p) throw python_error();
  return *static_cast<Engine*>(p);
}
bool dual_level;  // as the call came in, some thread differentiates forward: only then is there a tangent to look for (read and written with the interpreter's lock)

Engine& engine_of(PyObject* o) {
  refuse_tracing();
  Engine* const e = o == Py_None ? nullptr : &held(o);
  if (!e || e->closed) throw std::runtime_error("the engine is closed");
  dual_level = torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;
  return *e;
}
const Tensor* maybe(PyObject* o, const char* name) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) refuse("%s must be a tensor, got %s", name, Py_TYPE(o)->tp_name);
  return &THPVariable_Unpack(o);
}
const Tensor& tensor(PyObject* o, const char* name) {
  const Tensor* t = maybe(o, name);
  if (!t) refuse("%s is needed", name);
  return *t;
}
const Tensor& matrix(PyObject* o, const char* name) {
  const Tensor& t = tensor(o, name);
  if (t.dim() != 2) refuse("%s must be a tensor of two dimensions", name);
  return t;
}
int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
int32_t integer32(PyObject* o, const char* name) {
  const int64_t v = integer(o);
  if (v < INT32_MIN || v > INT32_MAX) refuse("%s %lld is out of range", name, (long long)v);
  return (int32_t)v;
}
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v;
}

enum Dense { WHOLE, LAST };  // contiguous, or the last dimension only

bool dense(const Tensor& t, Dense how) { return how == WHOLE ? t.is_contiguous() : t.dim() == 0 || t.size(-1) <= 1 || t.stride(-1) == 1; }

// a tangent of forward-mode differentiation (of the tensor, or of what it is a view of); none where that mode is switched off
bool has_tangent(const Tensor& t) { return dual_level && t._fw_grad(0).defined(); }

using Keys = c10::DispatchKeySet;
using Key = c10::DispatchKey;
// a tensor of another kind that stands for values it does not hold itself (fake, wrapped by a transform, a subclass with a dispatch of its own)
constexpr Keys STANDS_IN({Key::Python, Key::Functionalize, Key::FuncTorchGradWrapper, Key::FuncTorchBatched, Key::Batched});
// values that are not what the memory says: the lazily negated ones of x.conj().imag, the zeros without memory of forward-mode differentiation
constexpr Keys LAZY({Key::Negative, Key::ZeroTensor});

// on the engine's device, of that type and shape, with memory of its own; gradients are not recorded by these operators, tangents not carried on
void check(const Engine& e, const Tensor& t, const char* name, at::ScalarType type, at::IntArrayRef shape, Dense how) {
  if (t.scalar_type() == type && t.device() == e.device && t.sizes() == shape && dense(t, how) && !(t.requires_grad() && c10::GradMode::is_enabled()) && !has_tangent(t) && !t.key_set().has_any(STANDS_IN | LAZY)) return;
  if (t.key_set().has_any(STANDS_IN)) throw std::runtime_error(std::string(name) + " is a tensor that holds no values itself (traced, transformed, or a subclass with a dispatch of its own)");
  if (t.device() != e.device) refuse("%s is on %s, this engine on %s", name, t.device().str().c_str(), e.device.str().c_str());
  if (t.scalar_type() != type) {
    auto of = [](at::ScalarType s) { return s == at::kHalf ? "torch.float16" : s == at::kBFloat16 ? "torch.bfloat16" : s == at::kFloat ? "torch.float32" : s == at::kChar ? "torch.int8" : s == at::kInt ? "torch.int32" : at::toString(s); };
    refuse("%s must be %s, got %s", name, of(type), of(t.scalar_type()));
  }
  if (t.sizes() != shape) refuse("%s must have shape %s, got %s", name, text(shape).c_str(), text(t.sizes()).c_str());
  if (!dense(t, how)) refuse("%s must %s, got strides %s", name, how == WHOLE ? "be contiguous" : "have a dense last dimension", text(t.strides()).c_str());
  if (t.key_set().has_any(LAZY)) refuse("%s is lazily negated or a zero without memory: its memory does not hold its values (resolve_neg(), or clone it)", name);
  if (has_tangent(t)) refuse("%s has a forward-mode tangent: this op carries none on (take unpack_dual(...).primal, or switch forward gradients off)", name);
  refuse("%s requires a gradient: this op has none (detach it, or call under torch.no_grad())", name);
}
// a row stride (one row: the width, whatever the tensor says)
int64_t rows(const Engine& e, const Tensor& t, const char* name, at::ScalarType type, int64_t M, int64_t N) {
  check(e, t, name, type, {M, N}, LAST);
  return M > 1 ? t.stride(0) : N;
}
// the stride of 8-bit rows (one row: the next multiple of 16)
int64_t int8_rows(const Engine& e, const Tensor& t, const char* name, int64_t M, int64_t N) {
  check(e, t, name, at::kChar, {M, N}, LAST);
  return M > 1 ? t.stride(0) : (N + 15) & ~(int64_t)15;
}
const float* vector(const Engine& e, PyObject* o, const char* name, int64_t n) {
  const Tensor* t = maybe(o, name);
  if (!t) return nullptr;
  check(e, *t, name, at::kFloat, {n}, WHOLE);
  return static_cast<const float*>(t->data_ptr());
}
// modulations [samples, N] that cover M rows, and the stride between samples: 0 where the rows are one sample's, or where all samples share one (an expanded view)
struct Mod {
  const void* p = nullptr;
  int64_t stride = 0;
};
Mod modulation(const Engine& e, PyObject* o, const char* name, int64_t M, int64_t N, int64_t rows_per_batch) {
  if (o == Py_None) return {};
  const Tensor& t = matrix(o, name);
  const int64_t samples = t.size(0);
  check(e, t, name, e.dtype, {samples, N}, LAST);
  if (rows_per_batch < 1) refuse("rows_per_batch must be at least 1, got %lld", (long long)rows_per_batch);
  if (M > samples * rows_per_batch) refuse("%s has %lld samples of %lld rows, %lld rows are given", name, (long long)samples, (long long)rows_per_batch, (long long)M);
  return {t.data_ptr(), M > rows_per_batch ? t.stride(0) : 0};
}
int32_t size32(int64_t v, const char* what) {
  if (v > INT32_MAX) refuse("%s %lld is more than these operators index", what, (long long)v);
  return (int32_t)v;
}

// ---- results -----------------------------------------------------------------------------------------------------------------------------------------------------

Tensor fresh(const Engine& e, at::IntArrayRef shape, at::ScalarType type) { return at::empty(shape, at::TensorOptions().dtype(type).device(e.device)); }

// behind the launch: a tensor of the caller's has other values now, and whoever has saved it for a backward pass is told so (inference tensors count no versions)
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// an output: the caller's tensor, or a new one
struct Out {
  PyObject* given = nullptr;
  Tensor made;
  const Tensor& t() const { return given ? THPVariable_Unpack(given) : made; }
  PyObject* object() {  // once, behind the launch
    if (given) {
      written(t());
      Py_INCREF(given);
      return given;
    }
    return THPVariable_Wrap(std::move(made));
  }
};
Out out_rows(const Engine& e, PyObject* given, const char* name, at::ScalarType type, int64_t M, int64_t N, int64_t& stride) {
  Out o;
  if (given != Py_None) {
    stride = rows(e, tensor(given, name), name, type, M, N);
    o.given = given;
  } else {
    o.made = fresh(e, {M, N}, type);
    stride = N;
  }
  return o;
}
// 8-bit rows on 16 bytes and their scales
struct Int8Out {
  Out q, scale;
  int64_t stride;
};
Int8Out out_int8(const Engine& e, PyObject* given, const char* name, int64_t M, int64_t N) {
  Int8Out o;
  if (given != Py_None) {
    if (!PyTuple_Check(given) || PyTuple_GET_SIZE(given) != 2) refuse("%s must be a pair (q, scale)", name);
    o.q.given = PyTuple_GET_ITEM(given, 0);
    o.scale.given = PyTuple_GET_ITEM(given, 1);
    o.stride = int8_rows(e, tensor(o.q.given, "q"), "q", M, N);
    if (o.scale.given == Py_None) refuse("%s must come with its scale", name);
    (void)vector(e, o.scale.given, "scale", M);
  } else {
    o.stride = (N + 15) & ~(int64_t)15;
    Tensor rows = fresh(e, {M, o.stride}, at::kChar);
    o.q.made = o.stride == N ? std::move(rows) : rows.narrow(1, 0, N);
    o.scale.made = fresh(e, {M}, at::kFloat);
  }
  return o;
}
PyObject* pair(PyObject* a, PyObject* b) {  // takes both references
  PyObject* t = a && b ? PyTuple_New(2) : nullptr;
  if (!t) {
    Py_XDECREF(a);
    Py_XDECREF(b);
    throw python_error();
  }
  PyTuple_SET_ITEM(t, 0, a);
  PyTuple_SET_ITEM(t, 1, b);
  return t;
}

void* stream(const Engine& e) {
  PyObject* r = PyObject_CallFunctionObjArgs(e.stream_of, e.index, nullptr);
  if (!r) throw python_error();
  void* s = PyLong_AsVoidPtr(r);
  Py_DECREF(r);
  if (!s && PyErr_Occurred()) throw python_error();
  return s;
}
// f: the entry point alone, without the interpreter's lock: a launch waits where the device's queue is full, and the other threads do not.  close() waits for it.
template <typename F> void launch(Engine& e, F&& f) {
  void* const s = stream(e);
  if (e.closed) throw std::runtime_error("the engine is closed");  // (by a thread that ran meanwhile)
  ++e.running;
  PyThreadState* const state = PyEval_SaveThread();
  const int rc = f(s);
  PyEval_RestoreThread(state);
  --e.running;
  if (rc == ECAD_OK) return;
  const char* m = e.last_error(e.handle);  // this thread's own
  const std::string message = m && *m ? m : "error " + std::to_string(rc);
  if (rc == ECAD_E_INVALID || rc == ECAD_E_UNSUPPORTED) throw Refused{message};
  throw std::runtime_error(message);
}

void arguments(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) refuse("%lld arguments, %lld are wanted", (long long)n, (long long)want);
}
template <typename F> PyObject* guarded(F&& f) {
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const Refused& r) {
    PyErr_SetString(PyExc_ValueError, r.message.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// ---- operators -----------------------------------------------------------------------------------------------------------------------------------------------------

// (engine, x, out)
PyObject* quantize_int8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arguments(n, 3);
    Engine& e = engine_of(a[0]);
    const Tensor& x = matrix(a[1], "x");
    const int64_t M = x.size(0), K = x.size(1), ldx = rows(e, x, "x", e.dtype, M, K);
    const int32_t m = size32(M, "row count"), k = size32(K, "width");
    Int8Out o = out_int8(e, a[2], "out", M, K);
    int8_t* q = static_cast<int8_t*>(o.q.t().data_ptr());
    float* scale = static_cast<float*>(o.scale.t().data_ptr());
    const void* xp = x.data_ptr();
    launch(e, [&](void* s) { return e.quantize(e.handle, xp, ldx, q, o.stride, scale, m, k, s); });
    return pair(o.q.object(), o.scale.object());
  });
}

// (engine, epi, a, a_scale, w, w_scale, bias, resid, gate_table, gate_mod, rows_per_batch, out, resid_out, kernel)
PyObject* gemm_int8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arguments(n, 14);
    Engine& e = engine_of(a[0]);
    const Tensor &A = matrix(a[2], "a"), &W = matrix(a[4], "w");
    const int64_t M = A.size(0), K = A.size(1), N = W.size(0);
    EcadInt8Gemm g{};
    g.epi = integer32(a[1], "epi");
    g.lda = int8_rows(e, A, "a", M, K), g.A = static_cast<const int8_t*>(A.data_ptr()), g.ldw = int8_rows(e, W, "w", N, K), g.W = static_cast<const int8_t*>(W.data_ptr());
    g.a_scale = vector(e, a[3], "a_scale", M), g.w_scale = vector(e, a[5], "w_scale", N), g.bias = vector(e, a[6], "bias", N);
    if (a[3] == Py_None || a[5] == Py_None) refuse("a_scale and w_scale are needed");
    PyObject *resid = a[7], *out = a[11], *resid_out = a[12];
    g.rows_per_batch = integer32(a[10], "rows_per_batch");
    Out o;
    if (g.epi == 3) {
      if (resid == Py_None) refuse("epilogue 3 needs resid");
      if (resid_out == Py_None) resid_out = resid;
      const Tensor &r = tensor(resid, "resid"), &ro = tensor(resid_out, "resid_out");
      g.ldr = rows(e, r, "resid", e.dtype, M, N), g.resid = r.data_ptr();
      g.ldro = rows(e, ro, "resid_out", e.dtype, M, N), g.resid_out = ro.data_ptr();
      g.gate_table = vector(e, a[8], "gate_table", N);
      const Mod m = modulation(e, a[9], "gate_mod", M, N, g.rows_per_batch);
      g.gate_mod = m.p, g.gate_mod_stride = m.stride;
      if (out != Py_None) o = out_rows(e, out, "out", e.dtype, M, N, g.ldo);
    } else {
      if (resid != Py_None || a[8] != Py_None || a[9] != Py_None || resid_out != Py_None) refuse("resid and gates belong to epilogue 3");
      o = out_rows(e, out, "out", e.dtype, M, N, g.ldo);
    }
    const bool kept = o.given || o.made.defined();
    if (kept) g.out = o.t().data_ptr();
    g.M = size32(M, "row count"), g.N = size32(N, "width"), g.K = size32(K, "depth"), g.kernel = integer32(a[13], "kernel");
    launch(e, [&](void* s) { return e.gemm(e.handle, &g, s); });
    if (g.epi == 3) written(THPVariable_Unpack(resid_out));
    if (kept) return o.object();
    Py_RETURN_NONE;
  });
}

// (engine, h, y, pre, post, pre_weight, post_weight, gate_table, gate_mod, table_shift, table_scale, mod_shift, mod_scale, rows_per_batch, resid_scale, eps, quantize, out_h, out_n)
PyObject* gate_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arguments(n, 19);
    Engine& e = engine_of(a[0]);
    const Tensor& h = matrix(a[1], "h");
    const Tensor* y = maybe(a[2], "y");
    const int64_t M = h.size(0), D = h.size(1);
    EcadGateNorm g{};
    g.ldh = rows(e, h, "h", e.dtype, M, D), g.h = h.data_ptr();
    g.pre = integer32(a[3], "pre"), g.post = integer32(a[4], "post"), g.rows_per_batch = integer32(a[13], "rows_per_batch");
    const bool quantize = truth(a[16]);
    if (y) g.ldy = rows(e, *y, "y", e.dtype, M, D), g.y = y->data_ptr();
    g.pre_weight = vector(e, a[5], "pre_weight", D), g.post_weight = vector(e, a[6], "post_weight", D), g.gate_table = vector(e, a[7], "gate_table", D);
    g.table_shift = vector(e, a[9], "table_shift", D), g.table_scale = vector(e, a[10], "table_scale", D);
    const Mod gm = modulation(e, a[8], "gate_mod", M, D, g.rows_per_batch), ms = modulation(e, a[11], "mod_shift", M, D, g.rows_per_batch), mc = modulation(e, a[12], "mod_scale", M, D, g.rows_per_batch);
    g.gate_mod = gm.p, g.gate_mod_stride = gm.stride, g.mod_shift = ms.p, g.mod_scale = mc.p;
    if (ms.p && mc.p && ms.stride != mc.stride) refuse("mod_shift and mod_scale must have the same stride between samples, got %lld and %lld (one that all samples share may be a table)", (long long)ms.stride, (long long)mc.stride);
    g.mod_stride = ms.p ? ms.stride : mc.stride;
    Out nh, nn;
    Int8Out q;
    if (y) {
      nh = out_rows(e, a[17], "out_h", e.dtype, M, D, g.ldho);
      g.h_out = nh.t().data_ptr();
    } else if (a[17] != Py_None) {
      refuse("out_h without y: h' is h");
    }
    if (g.pre == ECAD_NORM_NONE) {
      if (a[18] != Py_None || quantize) refuse("out_n or quantize without a pre-norm");
    } else if (quantize) {
      q = out_int8(e, a[18], "out_n", M, D);
      g.q = static_cast<int8_t*>(q.q.t().data_ptr()), g.ldq = q.stride, g.q_scale = static_cast<float*>(q.scale.t().data_ptr());
    } else {
      nn = out_rows(e, a[18], "out_n", e.dtype, M, D, g.ldn);
      g.n_out = nn.t().data_ptr();
    }
    g.M = size32(M, "row count"), g.D = size32(D, "width"), g.resid_scale = (float)real(a[14]), g.eps = (float)real(a[15]);
    launch(e, [&](void* s) { return e.norm(e.handle, &g, s); });
    PyObject* first;
    if (y) {
      first = nh.object();
    } else {
      Py_INCREF(a[1]);
      first = a[1];
    }
    PyObject* second;
    if (g.pre == ECAD_NORM_NONE) {
      Py_INCREF(Py_None);
      second = Py_None;
    } else {
      second = quantize ? pair(q.q.object(), q.scale.object()) : nn.object();
    }
    return pair(first, second);
  });
}

// (engine, positions, dims, theta, scaling, factor, original_length, beta_fast, beta_slow, out)
PyObject* rope_table(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arguments(n, 10);
    Engine& e = engine_of(a[0]);
    const Tensor& p = tensor(a[1], "positions");
    const bool floats = p.scalar_type() == at::kFloat;
    if ((p.dim() != 1 && p.dim() != 2) || (!floats && p.scalar_type() != at::kInt)) refuse("positions must be an int32 or float32 tensor of shape (S,) or (S, axes)");
    if (!PyTuple_Check(a[2])) refuse("axes_dims must be an int or a tuple of them");
    int32_t dims[64];
    const Py_ssize_t axes = PyTuple_GET_SIZE(a[2]);
    if (axes < 1 || axes > 64 || axes != (p.dim() == 2 ? p.size(1) : 1)) refuse("positions of shape %s for %lld axes", text(p.sizes()).c_str(), (long long)axes);
    int64_t pairs = 0;
    for (Py_ssize_t i = 0; i < axes; ++i) {
      dims[i] = integer32(PyTuple_GET_ITEM(a[2], i), "axes_dims");
      if (dims[i] < 2 || dims[i] % 2 || dims[i] > 65536) refuse("axes_dims must be even and positive, got %d", dims[i]);
      pairs += dims[i] / 2;
    }
    check(e, p, "positions", p.scalar_type(), p.sizes(), WHOLE);
    const int64_t S = p.size(0);
    Out o;
    if (a[9] != Py_None) {
      check(e, tensor(a[9], "out"), "out", at::kFloat, {S, pairs, 2}, WHOLE);
      o.given = a[9];
    } else {
      o.made = fresh(e, {S, pairs, 2}, at::kFloat);
    }
    const double theta = real(a[3]), factor = real(a[5]), length = real(a[6]), fast = real(a[7]), slow = real(a[8]);
    const int32_t scaling = integer32(a[4], "scaling");
    const int32_t count = size32(S, "position count");
    const void* pp = p.data_ptr();
    float* table = static_cast<float*>(o.t().data_ptr());
    launch(e, [&](void* s) { return e.table(e.handle, pp, floats, dims, (int)axes, count, scaling, theta, factor, length, fast, slow, table, s); });
    return o.object();
  });
}

// (engine, q, k, table, half, index, inverse, q_out, k_out)
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arguments(n, 9);
    Engine& e = engine_of(a[0]);
    const Tensor& q = tensor(a[1], "q");
    if (q.dim() != 4) refuse("q must have shape (samples, tokens, heads, elements)");
    const int64_t B = q.size(0), S = q.size(1), D = q.size(3);
    const Tensor* k = maybe(a[2], "k");
    if (k && (k->dim() != 4 || k->size(0) != B || k->size(1) != S || k->size(2) < 1 || k->size(3) != D)) refuse("k of shape %s for q of shape %s", text(k->sizes()).c_str(), text(q.sizes()).c_str());
    const Tensor& t = tensor(a[3], "table");
    if (t.dim() != 3 || t.size(2) != 2) refuse("table must have shape (rows, pairs, 2)");
    check(e, t, "table", at::kFloat, t.sizes(), WHOLE);
    EcadRope g{};
    if (const Tensor* x = maybe(a[5], "index")) {
      const bool each = x->dim() == 2;
      if (!(x->dim() == 1 && x->size(0) == S) && !(each && x->size(0) == B && x->size(1) == S)) refuse("index must have shape (%lld,) or (%lld, %lld)", (long long)S, (long long)B, (long long)S);
      check(e, *x, "index", at::kInt, x->sizes(), LAST);
      g.index = static_cast<const int32_t*>(x->data_ptr()), g.index_stride = each && B > 1 ? x->stride(0) : 0;
    }
    if (a[7] != Py_None && (a[2] == Py_None) != (a[8] == Py_None)) refuse("out must be (q_out, k_out), k_out None where k is None");
    auto heads = [&](const Tensor& x, const char* name, PyObject* given, const char* out_name, Out& o) {
      check(e, x, name, e.dtype, x.sizes(), LAST);
      EcadRopeHeads h{};
      h.x = x.data_ptr(), h.sample = x.stride(0), h.token = x.stride(1), h.head = x.stride(2), h.H = x.size(2);
      if (a[7] != Py_None) {
        check(e, tensor(given, out_name), out_name, e.dtype, x.sizes(), LAST);
        o.given = given;
      } else {
        o.made = fresh(e, x.sizes(), e.dtype);
      }
      const Tensor& out = o.t();
      h.out = out.data_ptr(), h.out_sample = out.stride(0), h.out_token = out.stride(1), h.out_head = out.stride(2);
      return h;
    };
    Out qo, ko;
    g.q = heads(q, "q", a[7], "q_out", qo);
    if (k) g.k = heads(*k, "k", a[8], "k_out", ko);
    g.table = static_cast<const float*>(t.data_ptr()), g.table_rows = size32(t.size(0), "table rows"), g.rot = size32(2 * t.size(1), "turned elements");
    g.B = size32(B, "sample count"), g.S = size32(S, "token count"), g.D = size32(D, "head size"), g.half = truth(a[4]), g.inverse = truth(a[6]);
    launch(e, [&](void* s) { return e.rope(e.handle, &g, s); });
    PyObject* second;
    if (k) {
      second = ko.object();
    } else {
      Py_INCREF(Py_None);
      second = Py_None;
    }
    return pair(qo.object(), second);
  });
}

// ---- module ----------------------------------------------------------------------------------------------------------------------------------------------------------

void forget(PyObject* capsule) {
  Engine* e = static_cast<Engine*>(PyCapsule_GetPointer(capsule, ENGINE));
  if (!e) return;
  Py_XDECREF(e->stream_of);
  Py_XDECREF(e->index);
  delete e;
}

// (engine): no call starts behind this one, and those that run have left the library when it returns
PyObject* close(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arguments(n, 1);
    Engine& e = held(a[0]);
    e.closed = true;
    while (e.running) {
      PyThreadState* const state = PyEval_SaveThread();
      std::this_thread::sleep_for(std::chrono::microseconds(50));
      PyEval_RestoreThread(state);
    }
    Py_RETURN_NONE;
  });
}

// (addresses of the six entry points, engine handle, dtype: 0 fp16 / 1 bf16, device index or -1 for the CPU, stream_of)
PyObject* engine(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arguments(n, 5);
    if (!PyTuple_Check(a[0]) || PyTuple_GET_SIZE(a[0]) != 6) refuse("six entry points are wanted");
    void* f[6];
    for (int i = 0; i < 6; ++i) {
      f[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(a[0], i));
      if (!f[i]) refuse("entry point %d is missing", i);
    }
    auto e = std::make_unique<Engine>();
    e->quantize = reinterpret_cast<decltype(e->quantize)>(f[0]);
    e->gemm = reinterpret_cast<decltype(e->gemm)>(f[1]);
    e->norm = reinterpret_cast<decltype(e->norm)>(f[2]);
    e->table = reinterpret_cast<decltype(e->table)>(f[3]);
    e->rope = reinterpret_cast<decltype(e->rope)>(f[4]);
    e->last_error = reinterpret_cast<decltype(e->last_error)>(f[5]);
    e->handle = static_cast<EcadEngine*>(PyLong_AsVoidPtr(a[1]));
    if (PyErr_Occurred()) throw python_error();
    e->dtype = integer(a[2]) == ECAD_DTYPE_F16 ? at::kHalf : at::kBFloat16;
    const int64_t index = integer(a[3]);
    e->device = index < 0 ? c10::Device(c10::DeviceType::CPU) : c10::Device(c10::DeviceType::CUDA, (c10::DeviceIndex)index);
    e->stream_of = a[4];
    e->index = a[3];
    PyObject* capsule = PyCapsule_New(e.get(), ENGINE, forget);
    if (!capsule) throw python_error();
    Py_INCREF(a[4]);
    Py_INCREF(a[3]);
    e.release();
    return capsule;
  });
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)> PyCFunction fast() { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(F)); }

PyMethodDef methods[] = {{"engine", fast<engine>(), METH_FASTCALL, "What an engine gives its calls."},
                         {"close", fast<close>(), METH_FASTCALL, "No more calls on an engine; waits for those that run."},
                         {"quantize_int8", fast<quantize_int8>(), METH_FASTCALL, "EcadEngine.op_quantize_int8"},
                         {"gemm_int8", fast<gemm_int8>(), METH_FASTCALL, "EcadEngine.op_gemm_int8"},
                         {"gate_norm", fast<gate_norm>(), METH_FASTCALL, "EcadEngine.op_gate_norm"},
                         {"rope_table", fast<rope_table>(), METH_FASTCALL, "EcadEngine.op_rope_table"},
                         {"rope", fast<rope>(), METH_FASTCALL, "EcadEngine.op_rope"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops", "Argument checks and calls of the operators of an 8-bit transformer block.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops(void) { return PyModule_Create(&module); }
