// The int8 operators' checks of their tensors and the calls of b200_quantize_act_int8,
// b200_rmsnorm_int8 and b200_linear_int8, for int8.py, which has their signatures, what they do and
// the stream. Here because a small call is host time: a launch takes 2 us, and the same checks in
// Python with ctypes' conversion of the arguments took up to 6 more. One token, calls back to back:
// codes 5.6 -> 3.0 us, norm 6.4 -> 3.0, linear 7.8 -> 3.6.
//
// Every function takes tensors (or None), then numbers, and returns the entry point's status. What
// the entry points cannot see (types, devices, shapes, strides that do not fit) raises ValueError.
#include <Python.h>

#include <climits>
#include <exception>

#include <torch/csrc/autograd/python_variable.h>

#include "strands_b200.h"

namespace {

decltype(&b200_quantize_act_int8) g_quantize = nullptr;
decltype(&b200_rmsnorm_int8) g_rmsnorm = nullptr;
decltype(&b200_linear_int8) g_linear = nullptr;

struct Raised {};  // a Python exception is set

template <typename... A>
[[noreturn]] void refuse(const char* format, A... a) {
  PyErr_Format(PyExc_ValueError, format, a...);
  throw Raised{};
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a tensor", name);
    throw Raised{};
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.layout() != c10::kStrided) refuse("%s: b200 kernels take CUDA tensors only", name);
  return t;
}

int32_t small(int64_t v, const char* name) {
  if (v > INT32_MAX || v < INT32_MIN) refuse("%s: a size or stride is past 2^31", name);
  return int32_t(v);
}

int64_t number(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}

// The tensor an operator goes by: its device, rows and columns.
struct Place {
  int device;
  int32_t rows, k;
};
Place place(const at::Tensor& t, const char* name) {
  if (t.dim() != 2) refuse("%s must be 2-D", name);
  return {int(t.get_device()), small(t.size(0), name), small(t.size(1), name)};
}

// The row stride in elements of a tensor that must be `type` [rows, k] with contiguous rows.
int32_t row_stride(const at::Tensor& t, const char* name, at::ScalarType type, const Place& p, int64_t k) {
  if (t.scalar_type() != type || t.get_device() != p.device || t.dim() != 2 || t.size(0) != p.rows || t.size(1) != k)
    refuse("%s must be %s of shape (%d, %lld) on cuda:%d", name, c10::toString(type), int(p.rows), (long long)k, p.device);
  if (k > 1 && t.stride(1) != 1) refuse("%s's rows must be contiguous", name);
  return small(p.rows > 1 ? t.stride(0) : k, name);
}

const float* vector(const at::Tensor& t, const char* name, const Place& p, int64_t n) {
  if (t.scalar_type() != at::kFloat || t.get_device() != p.device || t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
    refuse("%s must be a contiguous fp32 tensor of %lld on cuda:%d", name, (long long)n, p.device);
  return static_cast<const float*>(t.data_ptr());
}

int32_t act_type(const at::Tensor& t, const char* name) {
  if (t.scalar_type() == at::kFloat) return B200_ACT_F32;
  if (t.scalar_type() != at::kBFloat16) refuse("%s must be float32 or bfloat16, not %s", name, c10::toString(t.scalar_type()));
  return B200_ACT_BF16;
}

template <typename F>
PyObject* launch(F f) {
  PyThreadState* const state = PyEval_SaveThread();  // a full launch queue makes the call wait
  const int status = f();
  PyEval_RestoreThread(state);
  return PyLong_FromLong(status);
}

// Runs an operator's body; C++ exceptions (torch's own among them) become Python's.
template <typename F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F body) {
  if (n != want) return PyErr_Format(PyExc_TypeError, "expected %zd arguments, not %zd", want, n);
  if (!g_linear) return PyErr_Format(PyExc_RuntimeError, "the entry points are not bound");
  try {
    return body();
  } catch (const Raised&) {
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// x, lo, out, scale, stream
PyObject* quantize_act(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 5, [&] {
    const at::Tensor& x = tensor(a[0], "x");
    const Place p = place(x, "x");
    const int32_t type = act_type(x, "x"), ldx = row_stride(x, "x", x.scalar_type(), p, p.k);
    const uint16_t* lo = nullptr;
    if (a[1] != Py_None) {
      const at::Tensor& t = tensor(a[1], "lo");
      if (type != B200_ACT_BF16) refuse("a low plane belongs to bfloat16 activations");
      if (row_stride(t, "lo", at::kBFloat16, p, p.k) != ldx) refuse("x and lo must have the same row stride");
      lo = static_cast<const uint16_t*>(t.data_ptr());
    }
    const at::Tensor &q = tensor(a[2], "out"), &s = tensor(a[3], "scale");
    const int32_t ldq = row_stride(q, "out", at::kChar, p, p.k);
    float* scale = const_cast<float*>(vector(s, "scale", p, p.rows));
    const void* xp = x.data_ptr();
    auto* qp = static_cast<int8_t*>(q.data_ptr());
    void* stream = reinterpret_cast<void*>(number(a[4]));
    return launch([&] { return g_quantize(xp, lo, type, p.rows, p.k, ldx, qp, ldq, scale, stream); });
  });
}

// x, w, eps, delta, resid_out, out, scale, stream
PyObject* rmsnorm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 8, [&] {
    const at::Tensor& x = tensor(a[0], "x");
    const Place p = place(x, "x");
    const int32_t ldx = row_stride(x, "x", at::kFloat, p, p.k);
    const float* w = vector(tensor(a[1], "w"), "w", p, p.k);
    const double eps = PyFloat_AsDouble(a[2]);
    if (eps == -1.0 && PyErr_Occurred()) throw Raised{};
    const void* delta = nullptr;
    float* sum = nullptr;
    int32_t type = B200_ACT_F32, ldd = 0, lds = 0;
    if (a[3] != Py_None) {
      const at::Tensor& t = tensor(a[3], "delta");
      type = act_type(t, "delta");
      ldd = row_stride(t, "delta", t.scalar_type(), p, p.k);
      delta = t.data_ptr();
    }
    if (a[4] != Py_None) {
      if (!delta) refuse("resid_out needs a delta");
      const at::Tensor& t = tensor(a[4], "resid_out");
      lds = row_stride(t, "resid_out", at::kFloat, p, p.k);
      sum = static_cast<float*>(t.data_ptr());
    }
    const at::Tensor &q = tensor(a[5], "out"), &s = tensor(a[6], "scale");
    const int32_t ldq = row_stride(q, "out", at::kChar, p, p.k);
    float* scale = const_cast<float*>(vector(s, "scale", p, p.rows));
    const auto* xp = static_cast<const float*>(x.data_ptr());
    auto* qp = static_cast<int8_t*>(q.data_ptr());
    void* stream = reinterpret_cast<void*>(number(a[7]));
    return launch([&] {
      return g_rmsnorm(xp, ldx, delta, type, ldd, sum, lds, p.rows, p.k, w, float(eps), qp, ldq, scale, stream);
    });
  });
}

// q, scale, codes, row_scale, out, lo, n, k, n_valid, epilogue, stream
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 11, [&] {
    const at::Tensor& q = tensor(a[0], "q");
    const Place p = place(q, "q");
    const int32_t ldx = row_stride(q, "q", at::kChar, p, p.k);
    const float* xs = vector(tensor(a[1], "scale"), "scale", p, p.rows);
    const int32_t wn = small(number(a[6]), "the weight"), wk = small(number(a[7]), "the weight");
    const int32_t valid = small(number(a[8]), "n_valid"), epilogue = small(number(a[9]), "epilogue");
    const at::Tensor& codes = tensor(a[2], "the weight");
    if (row_stride(codes, "the weight", at::kChar, {p.device, wn, wk}, wk) != wk)
      refuse("the weight must hold contiguous int8 codes");
    b200_qweight w = {};
    w.format = B200_W_INT8;
    w.n = wn;
    w.k = wk;
    w.data = codes.data_ptr();
    w.row_scale = vector(tensor(a[3], "the weight's row scales"), "the weight's row scales", p, wn);
    const bool swiglu = epilogue == B200_EP_SWIGLU;
    if (swiglu && valid % 2) refuse("a SwiGLU has as many up as gate features");
    const int64_t cols = swiglu ? valid / 2 : valid;
    const at::Tensor& out = tensor(a[4], "out");
    b200_linear_out o = {};
    o.epilogue = epilogue;
    o.n_valid = valid;
    o.out = out.data_ptr();
    o.ldo = row_stride(out, "out", swiglu ? at::kBFloat16 : at::kFloat, p, cols);
    if (a[5] != Py_None) {
      const at::Tensor& lo = tensor(a[5], "lo");
      const at::ScalarType type = lo.scalar_type();
      if (!swiglu || (type != at::kBFloat16 && type != at::kByte && type != at::kFloat8_e4m3fn))
        refuse("a low plane belongs to the SwiGLU, in bfloat16 or e4m3 bytes");
      if (row_stride(lo, "lo", type, p, cols) != o.ldo) refuse("out and lo must have the same row stride");
      const int64_t gap = reinterpret_cast<intptr_t>(lo.data_ptr()) - reinterpret_cast<intptr_t>(o.out);
      if (gap == 0 || gap % 2) refuse("lo must be a tensor of its own, a whole number of bf16 from out");
      o.lo_offset = gap / 2;
      o.lo_format = type == at::kBFloat16 ? B200_LO_BF16 : B200_LO_E4M3;
    }
    const auto* qp = static_cast<const int8_t*>(q.data_ptr());
    void* stream = reinterpret_cast<void*>(number(a[10]));
    return launch([&] { return g_linear(qp, xs, p.rows, p.k, ldx, &w, &o, stream); });
  });
}

// The addresses of b200_quantize_act_int8, b200_rmsnorm_int8 and b200_linear_int8 in the loaded library.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3) return PyErr_Format(PyExc_TypeError, "expected 3 addresses");
  try {
    const int64_t f[3] = {number(a[0]), number(a[1]), number(a[2])};
    g_quantize = reinterpret_cast<decltype(g_quantize)>(f[0]);
    g_rmsnorm = reinterpret_cast<decltype(g_rmsnorm)>(f[1]);
    g_linear = reinterpret_cast<decltype(g_linear)>(f[2]);
  } catch (const Raised&) {
    return nullptr;
  }
  Py_RETURN_NONE;
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(bind), FAST(quantize_act), FAST(rmsnorm), FAST(linear), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_int8_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__int8_ops() { return PyModule_Create(&module); }
