// nb_torch: the host side of the training operators for torch: the checks of the arguments, the outputs and workspaces
// from torch's allocator, and the calls of libnabla_g1's C entries on torch's current stream. It is compiled because a
// call's time on the host is what a small layer or a list of many small gradients costs.
//
// Every function raises TypeError for a tensor it cannot take, NotImplementedError for one with a forward-mode tangent
// and ValueError for an option out of range, before any launch; nothing is cast or copied.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

#include "../../include/nabla_g1.h"

namespace {

using at::Tensor;

constexpr const char* WHERE = "nablaengine_b200.torch_ffi: ";

// Thrown by a call that a dispatch mode (a trace, say) has to see: it returns None, and torch_ffi calls its custom op.
struct Dispatched {};

void leave_to_dispatcher() {
  if (c10::impl::dispatch_mode_enabled()) throw Dispatched{};
}

struct Refused {
  PyObject* kind;
  std::string text;
};

// What the caller passed, in torch_ffi's words.
std::string describe(PyObject* x) {
  std::string text = "?";
  PyObject* module = PyImport_ImportModule("nablaengine_b200.torch_ffi");
  PyObject* r = module ? PyObject_CallMethod(module, "_describe", "O", x) : nullptr;
  const char* s = r ? PyUnicode_AsUTF8(r) : nullptr;
  if (s) text = s;
  PyErr_Clear();
  Py_XDECREF(r);
  Py_XDECREF(module);
  return text;
}

[[noreturn]] void refuse(PyObject* kind, const std::string& text) { throw Refused{kind, WHERE + text}; }

int code_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: return -1;
  }
}

// A tensor argument: its tensor if it is one on a GPU of a value type whose memory holds its values (no lazy negation),
// else null. One that carries a forward-mode tangent is refused: the calls here read memory past the dispatcher and
// would drop it.
const Tensor* gpu_tensor(PyObject* x) {
  if (!THPVariable_Check(x)) return nullptr;
  const Tensor& t = THPVariable_Unpack(x);
  if (t._fw_grad(0).defined()) refuse(PyExc_NotImplementedError, "forward-mode derivatives are not available");
  const bool plain = t.is_cuda() && t.layout() == at::kStrided && !t.is_neg() && !t._is_zerotensor();
  return plain && code_of(t) >= 0 ? &t : nullptr;
}

int gpu_of(const Tensor& t) { return t.get_device(); }

void* at_or_null(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

void check(int rc, const char* entry) {
  if (rc == 0) return;
  refuse(PyExc_RuntimeError, std::string(entry) + " failed (CUDA error " + std::to_string(rc) + ")");
}

double number(PyObject* x) {
  const double v = PyFloat_AsDouble(x);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}

// ---- layer norm ---------------------------------------------------------------------------------------------------
struct Rows {
  const Tensor* t;
  int64_t rows, cols, stride;
};

// Rows one stride apart with dense columns.
Rows rows_of(const char* name, PyObject* x) {
  const Tensor* t = gpu_tensor(x);
  if (t && t->dim() >= 1 && t->size(-1) >= 1) {
    Rows r = {t, 0, t->size(-1), t->size(-1)};
    r.rows = t->numel() / r.cols;
    if (t->is_contiguous()) return r;
    if (r.cols == 1 || t->stride(-1) == 1) {
      bool uniform = true;
      int64_t span = -1;
      for (int64_t d = t->dim() - 2; d >= 0; d--) {
        if (t->size(d) == 1) continue;
        if (span < 0) r.stride = t->stride(d);
        else uniform = uniform && t->stride(d) == span;
        span = t->stride(d) * t->size(d);
      }
      if (uniform) return r;
    }
  }
  refuse(PyExc_TypeError, std::string(name) + " must be a float32, bfloat16 or float16 CUDA tensor (..., columns) with "
                          "dense columns and rows one stride apart, got " + describe(x));
}

// A parameter (or an undefined tensor for None): (columns,), dense, x's type or float32, x's device.
Tensor param(const char* name, PyObject* p, const Tensor& x) {
  if (p == Py_None) return Tensor();
  const Tensor* t = gpu_tensor(p);
  if (!t || !(t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat) || t->dim() != 1 ||
      t->size(0) != x.size(-1) || !t->is_contiguous() || gpu_of(*t) != gpu_of(x))
    refuse(PyExc_TypeError, std::string(name) + " must be a contiguous (" + std::to_string(x.size(-1)) +
                                ",) tensor of x's type or float32 on x's device, got " + describe(p));
  return *t;
}

int param_code(const Tensor& w, const Tensor& b, const Tensor& x) {
  if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type())
    refuse(PyExc_TypeError, "weight and bias must have one type");
  return code_of(w.defined() ? w : b.defined() ? b : x);
}

Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

// (x, weight, bias, eps) -> (y, mean, rstd)
std::vector<Tensor> layer_norm(PyObject* const* a) {
  leave_to_dispatcher();
  const Rows r = rows_of("x", a[0]);
  const Tensor& x = *r.t;
  const Tensor w = param("weight", a[1], x), b = param("bias", a[2], x);
  const int wcode = param_code(w, b, x);
  const double eps = number(a[3]);
  if (!std::isfinite(eps) || eps < 0 || !std::isfinite((float)eps))
    refuse(PyExc_ValueError, "eps must be finite and >= 0, got " + std::to_string(eps));
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  const Tensor y = empty(x.sizes(), x.scalar_type(), x), mean = empty(lead, at::kFloat, x),
               rstd = empty(lead, at::kFloat, x);
  if (r.rows)
    check(nb_g1_layer_norm_forward(c10::cuda::getCurrentCUDAStream(gpu_of(x)), r.rows, r.cols, r.stride, code_of(x),
                                   x.data_ptr(), wcode, at_or_null(w), at_or_null(b), (float)eps, y.data_ptr(),
                                   mean.data_ptr<float>(), rstd.data_ptr<float>()),
          "nb_g1_layer_norm_forward");
  return {y, mean, rstd};
}

const Tensor& statistic(const char* name, PyObject* p, const Tensor& x) {
  const Tensor* t = gpu_tensor(p);
  if (!t || t->scalar_type() != at::kFloat || t->sizes() != x.sizes().slice(0, x.dim() - 1) || !t->is_contiguous() ||
      gpu_of(*t) != gpu_of(x))
    refuse(PyExc_TypeError, std::string(name) + " must be a contiguous torch.float32 tensor of x's leading dimensions "
                            "on x's device, got " + describe(p));
  return *t;
}

// (g_y, x, mean, rstd, weight, bias, want_x, want_weight, want_bias) -> (g_x, g_weight, g_bias), None where not wanted
std::vector<Tensor> layer_norm_backward(PyObject* const* a) {
  leave_to_dispatcher();
  const Rows r = rows_of("x", a[1]), g = rows_of("g_y", a[0]);
  const Tensor& x = *r.t;
  if (g.t->sizes() != x.sizes() || g.t->scalar_type() != x.scalar_type() || gpu_of(*g.t) != gpu_of(x))
    refuse(PyExc_TypeError, "g_y must be like x (" + describe(a[1]) + "), got " + describe(a[0]));
  const Tensor &mean = statistic("mean", a[2], x), &rstd = statistic("rstd", a[3], x);
  const Tensor w = param("weight", a[4], x), b = param("bias", a[5], x);
  const int wcode = param_code(w, b, x);
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  Tensor gx, gw, gb, work;
  if (a[6] == Py_True) gx = empty(x.sizes(), x.scalar_type(), x);
  if (a[7] == Py_True && w.defined()) gw = empty(w.sizes(), w.scalar_type(), x);
  if (a[8] == Py_True && b.defined()) gb = empty(b.sizes(), b.scalar_type(), x);
  if (gw.defined() || gb.defined())
    work = empty({(int64_t)nb_g1_layer_norm_work_bytes(r.rows, r.cols)}, at::kByte, x);
  if (r.rows || work.defined())
    check(nb_g1_layer_norm_backward(c10::cuda::getCurrentCUDAStream(gpu_of(x)), r.rows, r.cols, g.stride, r.stride,
                                    code_of(x), g.t->data_ptr(), x.data_ptr(), mean.data_ptr<float>(),
                                    rstd.data_ptr<float>(), wcode, at_or_null(w), at_or_null(gx), at_or_null(gw),
                                    at_or_null(gb), at_or_null(work)),
          "nb_g1_layer_norm_backward");
  return {gx, gw, gb};
}

// ---- the gradient list --------------------------------------------------------------------------------------------
// True when t's values fill one span of memory, in any order of its dimensions.
bool dense(const Tensor& t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

struct List {
  std::vector<const Tensor*> t;
  std::vector<const void*> at;
  std::vector<long long> sizes;
  std::vector<int> types;
  int device = -1;
};

List list_of(const char* name, PyObject* x) {
  if (!PyList_Check(x) && !PyTuple_Check(x))
    refuse(PyExc_TypeError, std::string(name) + " must be a list or tuple of tensors, got " + describe(x));
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(x);
  PyObject** items = PySequence_Fast_ITEMS(x);
  List l;
  l.t.reserve(n), l.at.reserve(n), l.sizes.reserve(n), l.types.reserve(n);
  for (Py_ssize_t i = 0; i < n; i++) {
    const Tensor* t = gpu_tensor(items[i]);
    if (!t || !dense(*t))
      refuse(PyExc_TypeError, std::string(name) + "[" + std::to_string(i) + "] must be a dense float32, bfloat16 or "
                              "float16 CUDA tensor, got " + describe(items[i]));
    if (l.device < 0) l.device = gpu_of(*t);
    if (gpu_of(*t) != l.device)
      refuse(PyExc_TypeError, std::string(name) + "[" + std::to_string(i) + "] is on cuda:" +
                                  std::to_string(gpu_of(*t)) + ", " + name + "[0] on cuda:" +
                                  std::to_string(l.device));
    l.t.push_back(t);
    l.at.push_back(t->data_ptr());
    l.sizes.push_back(t->numel());
    l.types.push_back(code_of(*t));
  }
  if (l.device < 0) l.device = c10::cuda::current_device();
  return l;
}

// The outputs of a list: like the gradients, each of its gradient's type or float32.
List outs_of(PyObject* x, PyObject* grads, const List& g) {
  List o = list_of("out", x);
  if (o.t.size() != g.t.size())
    refuse(PyExc_TypeError, "out must have as many tensors as grads (" + std::to_string(g.t.size()) + "), got " +
                                std::to_string(o.t.size()));
  for (size_t i = 0; i < o.t.size(); i++) {
    const Tensor &a = *o.t[i], &b = *g.t[i];
    if (a.sizes() != b.sizes() || gpu_of(a) != gpu_of(b) || (o.types[i] != g.types[i] && o.types[i] != 0) ||
        !((a.is_contiguous() && b.is_contiguous()) || a.strides() == b.strides()))
      refuse(PyExc_TypeError, "out[" + std::to_string(i) + "] must be like grads[" + std::to_string(i) + "] (" +
                                  describe(PySequence_Fast_GET_ITEM(grads, i)) + ") or its float32 form, got " +
                                  describe(PySequence_Fast_GET_ITEM(x, i)));
  }
  return o;
}

// The result of a clip's entry: it refuses outputs that share memory, which is told as such; anything else is an error.
void check_clip(int rc, const char* entry, const List& g, const List* o) {
  if (rc == 0) return;
  const auto meet = [](const List& a, size_t i, const List& b, size_t k) {
    const char *x = static_cast<const char*>(a.at[i]), *y = static_cast<const char*>(b.at[k]);
    return x < y + b.t[k]->nbytes() && y < x + a.t[i]->nbytes();
  };
  for (size_t i = 0; o && i < g.t.size(); i++)
    for (size_t k = 0; k < g.t.size(); k++) {
      const bool own = i == k && g.at[i] == o->at[i] && g.types[i] == o->types[i];
      if ((!own && meet(*o, i, g, k)) || (i != k && meet(*o, i, *o, k)))
        refuse(PyExc_ValueError, "out[" + std::to_string(i) + "] and " + std::to_string(k) + ": a clipped gradient may "
                                 "not share memory with another gradient or output (but may be its own gradient)");
    }
  check(rc, entry);
}

Tensor empty_on(int device, at::IntArrayRef sizes, at::ScalarType type) {
  return at::detail::empty_cuda(sizes, type, at::Device(at::kCUDA, (c10::DeviceIndex)device), std::nullopt);
}

Tensor work_for(const List& g) {
  return empty_on(g.device, {(int64_t)nb_g1_grad_work_bytes((int)g.t.size())}, at::kByte);
}

// The two calls below write in place and have no operation that a trace could hold: it would hold their results.
void refuse_trace() {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  if (!c10::impl::dispatch_mode_enabled()) return;
  if (TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY) ||
      TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FAKE))
    refuse(PyExc_NotImplementedError, "grad_norm and clip_grad_norm cannot be traced");
}

// (grads, zero) -> stats (2,) float64: the sum of squares and the number of non-finite values
std::vector<Tensor> grad_sumsq(PyObject* const* a) {
  refuse_trace();
  const List g = list_of("grads", a[0]);
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)g.device);
  const Tensor work = work_for(g), stats = empty_on(g.device, {2}, at::kDouble);
  check(nb_g1_grad_sumsq(c10::cuda::getCurrentCUDAStream(g.device), (int)g.t.size(), g.at.data(), g.sizes.data(),
                         g.types.data(), a[1] == Py_True, work.data_ptr(), stats.data_ptr<double>()),
        "nb_g1_grad_sumsq");
  return {stats};
}

// (grads, outs or None, max_norm, eps, zero, stats or None) -> (norm, bad): by grads' own sums, or by stats'
std::vector<Tensor> grad_clip(PyObject* const* a) {
  refuse_trace();
  const List g = list_of("grads", a[0]);
  const double max_norm = number(a[2]), eps = number(a[3]);
  if (!(max_norm >= 0) || !(eps >= 0) || !std::isfinite(eps))
    refuse(PyExc_ValueError, "max_norm and eps must be >= 0 (eps finite), got " + std::to_string(max_norm) + ", " +
                                 std::to_string(eps));
  List other;
  if (a[1] != Py_None && a[1] != a[0]) other = outs_of(a[1], a[0], g);
  const List& o = a[1] == a[0] ? g : other;
  void* const* outs = a[1] == Py_None ? nullptr : const_cast<void* const*>(o.at.data());
  const int count = (int)g.t.size(), zero = a[4] == Py_True;
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)g.device);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(g.device);
  const Tensor norm = empty_on(g.device, {}, at::kFloat), bad = empty_on(g.device, {}, at::kLong);
  long long* badp = reinterpret_cast<long long*>(bad.data_ptr<int64_t>());
  if (a[5] == Py_None) {
    long long values = 0;
    for (long long n : g.sizes) values += n;
    Tensor work;
    if (count > NB_G1_GRAD_SMALL_TENSORS || values > NB_G1_GRAD_SMALL_VALUES) work = work_for(g);
    check_clip(nb_g1_grad_clip(stream, count, g.at.data(), outs, g.sizes.data(), g.types.data(), o.types.data(), zero,
                               max_norm, eps, at_or_null(work), norm.data_ptr<float>(), badp),
               "nb_g1_grad_clip", g, outs ? &o : nullptr);
  } else {
    const Tensor& stats = THPVariable_Unpack(a[5]);
    check_clip(nb_g1_grad_scale(stream, count, g.at.data(), outs, g.sizes.data(), g.types.data(), o.types.data(), zero,
                                max_norm, eps, stats.data_ptr<double>(), norm.data_ptr<float>(), badp),
               "nb_g1_grad_scale", g, outs ? &o : nullptr);
  }
  if (outs)
    for (const Tensor* t : o.t)
      if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return {norm, bad};
}

// ---- the module -----------------------------------------------------------------------------------------------------
template <std::vector<Tensor> (*F)(PyObject* const*), int N>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments are wanted, got %zd", N, n);
    return nullptr;
  }
  try {
    const std::vector<Tensor> r = F(args);
    PyObject* t = PyTuple_New((Py_ssize_t)r.size());
    if (!t) return nullptr;
    for (size_t i = 0; i < r.size(); i++) {
      PyObject* x = r[i].defined() ? THPVariable_Wrap(r[i]) : Py_NewRef(Py_None);
      if (!x) {
        Py_DECREF(t);
        return nullptr;
      }
      PyTuple_SET_ITEM(t, (Py_ssize_t)i, x);
    }
    return t;
  } catch (const Dispatched&) {
    return Py_NewRef(Py_None);
  } catch (const Refused& e) {
    PyErr_SetString(e.kind, e.text.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyMethodDef METHODS[] = {
    {"layer_norm", (PyCFunction)(void (*)())call<layer_norm, 4>, METH_FASTCALL, "x, weight, bias, eps"},
    {"layer_norm_backward", (PyCFunction)(void (*)())call<layer_norm_backward, 9>, METH_FASTCALL,
     "g_y, x, mean, rstd, weight, bias, want_x, want_weight, want_bias"},
    {"grad_sumsq", (PyCFunction)(void (*)())call<grad_sumsq, 2>, METH_FASTCALL, "grads, zero"},
    {"grad_clip", (PyCFunction)(void (*)())call<grad_clip, 6>, METH_FASTCALL,
     "grads, outs, max_norm, eps, zero, stats"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef MODULE = {PyModuleDef_HEAD_INIT, "nb_torch", nullptr, -1, METHODS, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_nb_torch() { return PyModule_Create(&MODULE); }
