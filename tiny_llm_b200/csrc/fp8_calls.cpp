// The 8-bit operators' calls without the interpreter: reads the tensors, checks that the call is an ordinary one and launches it through
// the C entry points of the kernels' libraries.  Read attribute by attribute from Python, a call of five tensors took longer than the
// small kernels run (8.5 us a call, 4.0 this way).
//
// Every function returns True if it launched the call and False, having done nothing, if the call is not one of the ordinary ones or its
// entry point refused it: the Python function then goes through its own checks, which have the words for what does not fit.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>

#include "fp8_calls.h"

namespace {

int (*g_quantize)(const QuantizeCall*) = nullptr;
int (*g_rms_norm)(const RmsNormCall*) = nullptr;
int (*g_quantize_weight)(const QuantizeWeightCall*) = nullptr;
int (*g_linear)(const LinearFp8Call*) = nullptr;

constexpr int F32 = 0, BF16 = 1;
constexpr int OUT_BF16 = 0, OUT_F32 = 1, OUT_ADD = 2, OUT_FP8 = 3;
constexpr int64_t MOST = INT32_MAX - 4095;

// A matrix of rows on the wanted device; false: not an ordinary one.
struct Matrix { void* data; int64_t rows, cols, ld; c10::ScalarType type; };
bool matrix(PyObject* o, int device, Matrix& m) {
  if (!THPVariable_Check(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.get_device() != device || t.layout() != at::kStrided || t.dim() != 2) return false;
  m.rows = t.size(0);
  m.cols = t.size(1);
  if (m.rows < 1 || m.cols < 1 || m.rows > MOST || m.cols > MOST || (m.cols > 1 && t.stride(1) != 1)) return false;
  m.ld = m.rows > 1 ? t.stride(0) : (m.cols + 15) / 16 * 16;      // (the stride of a single row means nothing)
  if (m.ld < m.cols) return false;
  m.data = t.data_ptr();
  m.type = t.scalar_type();
  return true;
}
bool float_vector(PyObject* o, int device, int64_t n, void** data) {
  if (!THPVariable_Check(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.get_device() != device || t.scalar_type() != at::kFloat || t.numel() != n || !t.is_contiguous()) return false;
  *data = t.data_ptr();
  return true;
}
int64_t groups(int64_t n) { return (n + 127) / 128; }
bool values8(const Matrix& m) { return m.type == at::ScalarType::Float8_e4m3fn && m.ld % 16 == 0 && reinterpret_cast<uintptr_t>(m.data) % 16 == 0; }
bool row_scales(const Matrix& s, const Matrix& of) { return s.type == at::ScalarType::Float8_e8m0fnu && s.rows == of.rows && s.cols == groups(of.cols); }
bool weight_scales(const Matrix& s, const Matrix& of) {
  return s.type == at::kFloat && s.rows == groups(of.rows) && s.cols == groups(of.cols) && (s.rows == 1 || s.ld == s.cols);
}
int float_code(c10::ScalarType t) { return t == at::kFloat ? F32 : t == at::kBFloat16 ? BF16 : -1; }

// The launch, with the interpreter let go (a full queue makes it wait).
template <typename Call>
bool launch(int (*entry)(const Call*), const Call& c) {
  int rc = -1;
  Py_BEGIN_ALLOW_THREADS;
  rc = entry(&c);
  Py_END_ALLOW_THREADS;
  return rc == 0;
}
// Tensors that cannot give an address or a size throw; to the caller such a call is not an ordinary one.
template <typename Function>
PyObject* answer(Function call) {
  bool launched = false;
  try {
    launched = call();
  } catch (...) {
  }
  return PyBool_FromLong(launched);
}
bool number(PyObject* o, long long& v) {
  v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) { PyErr_Clear(); return false; }
  return true;
}

// (x, out, scales, device, stream)
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return answer([&] {
    long long device, stream;
    Matrix x, out, sc;
    if (n != 5 || !number(a[3], device) || !number(a[4], stream) || !matrix(a[0], (int)device, x) || !matrix(a[1], (int)device, out) ||
        !matrix(a[2], (int)device, sc) || !values8(out) || !row_scales(sc, out) || x.rows != out.rows || x.cols != out.cols || float_code(x.type) < 0)
      return false;
    const QuantizeCall c = {x.data, x.ld, out.data, out.ld, sc.data, sc.ld, (int)x.rows, (int)x.cols, float_code(x.type), (void*)stream};
    return launch(g_quantize, c);
  });
}

// (x, weight, eps, out, scales, device, stream)
PyObject* rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return answer([&] {
    long long device, stream;
    Matrix x, out, sc;
    void* w = nullptr;
    if (n != 7 || !PyFloat_Check(a[2]) || !number(a[5], device) || !number(a[6], stream) || !matrix(a[0], (int)device, x) || !matrix(a[3], (int)device, out) ||
        !matrix(a[4], (int)device, sc) || !values8(out) || !row_scales(sc, out) || x.rows != out.rows || x.cols != out.cols || x.type != at::kFloat ||
        (x.rows > 1 && x.ld != x.cols) || !float_vector(a[1], (int)device, x.cols, &w))
      return false;
    const RmsNormCall c = {x.data, w, out.data, out.ld, sc.data, sc.ld, nullptr, (int)x.rows, (int)x.cols,
                           (float)PyFloat_AS_DOUBLE(a[2]), (void*)stream};
    return launch(g_rms_norm, c);
  });
}

// (w, out, scales, device, stream)
PyObject* quantize_weight(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return answer([&] {
    long long device, stream;
    Matrix w, out, sc;
    if (n != 5 || !number(a[3], device) || !number(a[4], stream) || !matrix(a[0], (int)device, w) || !matrix(a[1], (int)device, out) ||
        !matrix(a[2], (int)device, sc) || !values8(out) || !weight_scales(sc, out) || w.rows != out.rows || w.cols != out.cols || float_code(w.type) < 0)
      return false;
    const QuantizeWeightCall c = {w.data, w.ld, out.data, out.ld, sc.data, (int)w.rows, (int)w.cols, float_code(w.type), (void*)stream};
    return launch(g_quantize_weight, c);
  });
}

// what the products share: (a, a_scales, w, w_scales, out, ...)
bool operands(PyObject* const* a, int device, LinearFp8Call& c, Matrix& x, Matrix& w, Matrix& out) {
  Matrix xs, ws;
  if (!matrix(a[0], device, x) || !matrix(a[1], device, xs) || !matrix(a[2], device, w) || !matrix(a[3], device, ws) || !matrix(a[4], device, out) ||
      !values8(x) || !values8(w) || !row_scales(xs, x) || !weight_scales(ws, w) || x.cols != w.cols || out.rows != x.rows)
    return false;
  c.a = x.data; c.lda = x.ld; c.a_scales = xs.data; c.lda_s = xs.ld; c.w = w.data; c.ldw = w.ld; c.w_scales = ws.data;
  c.out = out.data; c.ldo = out.ld; c.m = (int)x.rows; c.n = (int)out.cols; c.k = (int)x.cols;
  return true;
}

// (a, a_scales, w, w_scales, out, accumulate, device, stream, status)
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return answer([&] {
    long long device, stream, status;
    LinearFp8Call c = {};
    Matrix x, w, out;
    if (n != 9 || !PyBool_Check(a[5]) || !number(a[6], device) || !number(a[7], stream) || !number(a[8], status) || !operands(a, (int)device, c, x, w, out) ||
        out.cols != w.rows)
      return false;
    const bool add = a[5] == Py_True;
    if (out.type == at::kFloat) c.mode = add ? OUT_ADD : OUT_F32;
    else if (out.type == at::kBFloat16 && !add) c.mode = OUT_BF16;
    else return false;
    c.status = (void*)status;
    c.stream = (void*)stream;
    return launch(g_linear, c);
  });
}

// (a, a_scales, w, w_scales, out, out_scales or None, act, limit, device, stream, status)
PyObject* gated(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return answer([&] {
    long long act, device, stream, status;
    LinearFp8Call c = {};
    Matrix x, w, out, os;
    if (n != 11 || !number(a[6], act) || !PyFloat_Check(a[7]) || !number(a[8], device) || !number(a[9], stream) || !number(a[10], status) ||
        !operands(a, (int)device, c, x, w, out) || w.rows != 256 * groups(out.cols))
      return false;
    if (a[5] == Py_None) {
      if (out.type != at::kBFloat16) return false;
      c.mode = OUT_BF16;
    } else {
      if (!matrix(a[5], (int)device, os) || !values8(out) || !row_scales(os, out)) return false;
      c.mode = OUT_FP8;
      c.out_scales = os.data;
      c.ldo_s = os.ld;
    }
    c.gated = 1;
    c.act = (int)act;
    c.limit = (float)PyFloat_AS_DOUBLE(a[7]);
    c.status = (void*)status;
    c.stream = (void*)stream;
    return launch(g_linear, c);
  });
}

// addresses of the C entry points: (quantize, rms_norm, quantize_weight, linear)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  long long at[4];
  for (int i = 0; i < 4; ++i)
    if (n != 4 || !number(a[i], at[i])) { PyErr_SetString(PyExc_TypeError, "bind takes four addresses"); return nullptr; }
  g_quantize = reinterpret_cast<decltype(g_quantize)>(at[0]);
  g_rms_norm = reinterpret_cast<decltype(g_rms_norm)>(at[1]);
  g_quantize_weight = reinterpret_cast<decltype(g_quantize_weight)>(at[2]);
  g_linear = reinterpret_cast<decltype(g_linear)>(at[3]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},
    {"quantize", (PyCFunction)(void (*)(void))quantize, METH_FASTCALL, nullptr},
    {"rms_norm", (PyCFunction)(void (*)(void))rms_norm, METH_FASTCALL, nullptr},
    {"quantize_weight", (PyCFunction)(void (*)(void))quantize_weight, METH_FASTCALL, nullptr},
    {"linear", (PyCFunction)(void (*)(void))linear, METH_FASTCALL, nullptr},
    {"gated", (PyCFunction)(void (*)(void))gated, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "fp8_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_fp8_calls(void) { return PyModule_Create(&module); }
