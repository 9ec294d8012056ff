// The usual calls of the torch front ends (norm, ptq.dequantize_rows, mxfp4,
// logprobs) without the interpreter: checks, outputs and launch in one C++ call
// (rms_norm_i8 of one row: 5 us of the host's time, 10 in Python, of which the
// launch takes 2.6).  A function here answers only calls that need no word of
// explanation; for every other one, and for those that the library refuses, it
// gives None, and the Python front end says what is wrong or does the rest.  A
// launch that fails raises as it would there, and is not tried again.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "taccel_b200.h"

namespace {

// The library's entries, whose addresses `bind` gets.
struct Entries {
  decltype(&tac_rms_norm) rms_norm;
  decltype(&tac_rms_norm_i8) rms_norm_i8;
  decltype(&tac_dequantize_rows_i8) dequantize;
  decltype(&tac_mxfp4_quantize) quantize;
  decltype(&tac_mxfp4_values) values;
  decltype(&tac_mxfp4_gemm) gemm;
  decltype(&tac_linear_mxfp4) linear;
  decltype(&tac_linear_mxfp4_workspace_bytes) linear_bytes;
  decltype(&tac_token_logprobs) logprobs;
} lib;

int type_of(at::ScalarType t) {
  return t == at::kFloat ? TAC_F32 : t == at::kHalf ? TAC_F16 : t == at::kBFloat16 ? TAC_BF16 : -1;
}

// The CUDA device of a tensor, if it is the current one; else -1.
int64_t device_of(PyObject* o) {
  if (!THPVariable_Check(o) || !THPVariable_Unpack(o).is_cuda()) return -1;
  const int64_t dev = THPVariable_Unpack(o).get_device();
  return dev == c10::cuda::current_device() ? dev : -1;
}
const at::Tensor* tensor(PyObject* o, int64_t dev) {
  if (dev < 0 || !THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.layout() == at::kStrided && t.get_device() == dev ? &t : nullptr;
}

// [M, K] of a floating-point type with contiguous rows that do not overlap.
struct Rows {
  const at::Tensor* t = nullptr;
  int type = -1, M = 0, K = 0;
  int64_t ld = 0;
  bool of(PyObject* o, int64_t dev) {
    t = tensor(o, dev);
    if (!t || t->dim() != 2) return false;
    type = type_of(t->scalar_type());
    const int64_t m = t->size(0), k = t->size(1);
    ld = t->stride(0);
    if (type < 0 || m <= 0 || k <= 0 || m > INT_MAX || k > INT_MAX || t->stride(1) != 1 || ld < k) return false;
    M = int(m), K = int(k);
    return true;
  }
};

// [n] contiguous, of any of the types; null stays null.
struct Vector {
  const void* p = nullptr;
  int type = 0;
  bool of(PyObject* o, int64_t n, int64_t dev) {
    if (o == Py_None) return true;
    const at::Tensor* t = tensor(o, dev);
    if (!t || t->dim() != 1 || t->size(0) != n || !t->is_contiguous() || (type = type_of(t->scalar_type())) < 0) return false;
    p = t->const_data_ptr();
    return true;
  }
};

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, int64_t dev) {
  return at::detail::empty_cuda(sizes, type, at::Device(at::kCUDA, c10::DeviceIndex(dev)), std::nullopt);
}
// A product's result: a new tensor where o is None, o itself where it is as that one would be.
bool result(PyObject* o, int64_t M, int64_t N, at::ScalarType type, int64_t dev, at::Tensor* y) {
  if (o == Py_None) {
    *y = empty({M, N}, type, dev);
    return true;
  }
  const at::Tensor* t = tensor(o, dev);
  if (!t || t->scalar_type() != type || t->dim() != 2 || t->size(0) != M || t->size(1) != N || !t->is_contiguous()) return false;
  *y = *t;
  return true;
}
void* stream(int64_t dev) { return c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(dev)).stream(); }

// The launch without the interpreter's lock, which an exception (a tensor without memory) takes back too.
struct Unlocked {
  PyThreadState* const state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};
template <typename F>
int launched(F f) {
  Unlocked u;
  return f();
}

PyObject* check = nullptr;             // raises the error of (status, name)

// What a call gives whose launch did not go well: None where the library refused its arguments, before any launch.
PyObject* failed(int status, const char* name) {
  if (status == TAC_E_ARGUMENT) Py_RETURN_NONE;
  Py_XDECREF(PyObject_CallFunction(check, "is", status, name));
  return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_RuntimeError, "%s failed (status %d)", name, status);
}

template <typename... T>
PyObject* tuple(const T&... t) {
  PyObject* r = PyTuple_New(sizeof...(t));
  Py_ssize_t i = 0;
  if (r) (PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(t)), ...);
  return r;
}

bool number(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &overflow);
  return !overflow;
}
// 4-bit rows on device `dev`, of four arguments: their codes and scales, rows, columns, device.  Codes and scales are two
// tensors, which have rows and device themselves (then None), or their addresses.
struct Rows4 {
  const uint8_t *codes = nullptr, *scales = nullptr;
  int64_t rows = 0, cols = 0;
  bool of(PyObject* const* a, int64_t dev) {
    if (dev < 0 || !PyTuple_CheckExact(a[0]) || PyTuple_GET_SIZE(a[0]) != 2 || !number(a[2], &cols) || cols <= 0 || cols > INT_MAX)
      return false;
    PyObject *c = PyTuple_GET_ITEM(a[0], 0), *s = PyTuple_GET_ITEM(a[0], 1);
    if (a[1] == Py_None && a[3] == Py_None) {
      const at::Tensor *ct = tensor(c, dev), *st = tensor(s, dev);
      if (!ct || !st || ct->scalar_type() != at::kByte || st->scalar_type() != at::kByte || ct->dim() != 2 ||
          !ct->is_contiguous() || !st->is_contiguous() || ct->size(1) != (cols + 31) / 32 * 16)
        return false;
      rows = ct->size(0);
      const int64_t shape[] = {(rows + 127) / 128, (cols + 255) / 256 * 2, 32, 4, 4};
      if (st->sizes() != at::IntArrayRef(shape)) return false;
      codes = static_cast<const uint8_t*>(ct->const_data_ptr());
      scales = static_cast<const uint8_t*>(st->const_data_ptr());
      if ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales)) & 15) return false;
    } else {
      int64_t at = -1;
      if (!PyLong_CheckExact(c) || !PyLong_CheckExact(s) || !number(a[1], &rows) || !number(a[3], &at) || at != dev) return false;
      codes = static_cast<const uint8_t*>(PyLong_AsVoidPtr(c));
      scales = static_cast<const uint8_t*>(PyLong_AsVoidPtr(s));
    }
    return codes && scales && rows > 0 && rows <= INT_MAX;
  }
  // device_of their tensors
  static int64_t device(PyObject* o) { return PyTuple_CheckExact(o) && PyTuple_GET_SIZE(o) == 2 ? device_of(PyTuple_GET_ITEM(o, 0)) : -1; }
};

struct NormCall {
  Rows x, r;
  Vector w;
  at::Tensor h;
  float eps = 0.f;
  int64_t dev = 0;
  bool of(PyObject* const* a) {        // x, weight, eps, residual
    dev = device_of(a[0]);
    if (!x.of(a[0], dev) || a[1] == Py_None || !w.of(a[1], x.K, dev) || !PyFloat_CheckExact(a[2])) return false;
    const double e = PyFloat_AS_DOUBLE(a[2]);
    if (!(e >= 0 && e <= 1e30)) return false;
    eps = float(e);
    if (a[3] == Py_None) return true;
    if (!r.of(a[3], dev) || r.type != x.type || r.M != x.M || r.K != x.K) return false;
    h = empty({x.M, x.K}, x.t->scalar_type(), dev);
    return true;
  }
  const void* residual() const { return r.t ? r.t->const_data_ptr() : nullptr; }
  void* sum() const { return r.t ? h.data_ptr() : nullptr; }
};

PyObject* rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  NormCall c;
  if (n != 4 || !c.of(a)) Py_RETURN_NONE;
  const at::Tensor y = empty({c.x.M, c.x.K}, c.x.t->scalar_type(), c.dev);
  const auto run = [&] {
    return lib.rms_norm(c.x.t->const_data_ptr(), c.x.type, c.x.ld, c.residual(), c.r.ld, c.sum(), c.x.K, c.w.p, c.w.type, c.eps,
                        y.data_ptr(), c.x.M, c.x.K, stream(c.dev));
  };
  if (const int status = launched(run)) return failed(status, "tac_rms_norm");
  return c.r.t ? tuple(y, c.h) : THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

PyObject* rms_norm_i8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  NormCall c;
  if (n != 4 || !c.of(a)) Py_RETURN_NONE;
  const at::Tensor q = empty({c.x.M, (int64_t(c.x.K) + 15) / 16 * 16}, at::kChar, c.dev), scale = empty({c.x.M}, at::kFloat, c.dev);
  const auto run = [&] {
    return lib.rms_norm_i8(c.x.t->const_data_ptr(), c.x.type, c.x.ld, c.residual(), c.r.ld, c.sum(), c.x.K, c.w.p, c.w.type, c.eps,
                           static_cast<int8_t*>(q.data_ptr()), static_cast<float*>(scale.data_ptr()), c.x.M, c.x.K, stream(c.dev));
  };
  if (const int status = launched(run)) return failed(status, "tac_rms_norm_i8");
  return c.r.t ? tuple(q, scale, c.h) : tuple(q, scale);
  END_HANDLE_TH_ERRORS
}

PyObject* dequantize_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {      // q, scale, K or None, dtype
  HANDLE_TH_ERRORS
  if (n != 4 || !THPDtype_Check(a[3])) Py_RETURN_NONE;
  const int64_t dev = device_of(a[0]);
  const at::ScalarType out = reinterpret_cast<THPDtype*>(a[3])->scalar_type;
  const at::Tensor *q = tensor(a[0], dev), *scale = tensor(a[1], dev);
  if (!q || !scale || type_of(out) < 0 || q->scalar_type() != at::kChar || scale->scalar_type() != at::kFloat || q->dim() != 2 ||
      scale->dim() != 1 || !q->is_contiguous() || !scale->is_contiguous())
    Py_RETURN_NONE;
  const int64_t M = q->size(0), most = q->size(1);
  int64_t K = most;
  if (a[2] != Py_None && !number(a[2], &K)) Py_RETURN_NONE;
  if (M <= 0 || M > INT_MAX || most <= 0 || most > INT_MAX || most % 16 || scale->size(0) != M || K <= most - 16 || K > most)
    Py_RETURN_NONE;
  const at::Tensor y = empty({M, K}, out, dev);
  const auto run = [&] {
    return lib.dequantize(static_cast<const int8_t*>(q->const_data_ptr()), static_cast<const float*>(scale->const_data_ptr()),
                          y.data_ptr(), type_of(out), int(M), int(K), stream(dev));
  };
  if (const int status = launched(run)) return failed(status, "tac_dequantize_rows_i8");
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {             // X; (codes, scales, K)
  HANDLE_TH_ERRORS
  Rows x;
  if (n != 1) Py_RETURN_NONE;
  const int64_t dev = device_of(a[0]);
  if (!x.of(a[0], dev)) Py_RETURN_NONE;
  const at::Tensor codes = empty({x.M, (int64_t(x.K) + 31) / 32 * 16}, at::kByte, dev);
  const at::Tensor scales = empty({(int64_t(x.M) + 127) / 128, (int64_t(x.K) + 255) / 256 * 2, 32, 4, 4}, at::kByte, dev);
  uint8_t *c = static_cast<uint8_t*>(codes.data_ptr()), *s = static_cast<uint8_t*>(scales.data_ptr());
  const auto run = [&] { return lib.quantize(x.t->const_data_ptr(), x.type, x.ld, c, s, x.M, x.K, stream(dev)); };
  if (const int status = launched(run)) return failed(status, "tac_mxfp4_quantize");
  return Py_BuildValue("(NNi)", THPVariable_Wrap(codes), THPVariable_Wrap(scales), x.K);
  END_HANDLE_TH_ERRORS
}

PyObject* values(PyObject*, PyObject* const* a, Py_ssize_t n) {               // 4-bit rows, dtype
  HANDLE_TH_ERRORS
  Rows4 x;
  if (n != 5) Py_RETURN_NONE;
  const int64_t dev = Rows4::device(a[0]);
  if (!x.of(a, dev) || !THPDtype_Check(a[4])) Py_RETURN_NONE;
  const at::ScalarType out = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
  if (type_of(out) < 0) Py_RETURN_NONE;
  const at::Tensor y = empty({x.rows, x.cols}, out, dev);
  const auto run = [&] { return lib.values(x.codes, x.scales, y.data_ptr(), type_of(out), int(x.rows), int(x.cols), stream(dev)); };
  if (const int status = launched(run)) return failed(status, "tac_mxfp4_values");
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

PyObject* gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {              // 4-bit rows twice, bias, dtype, out
  HANDLE_TH_ERRORS
  Rows4 a, b;
  Vector bias;
  if (n != 11) Py_RETURN_NONE;
  const int64_t dev = Rows4::device(args[0]);
  if (!a.of(args, dev) || !b.of(args + 4, dev) || a.cols != b.cols || !bias.of(args[8], b.rows, dev) || !THPDtype_Check(args[9]))
    Py_RETURN_NONE;
  const at::ScalarType out = reinterpret_cast<THPDtype*>(args[9])->scalar_type;
  at::Tensor y;
  if (type_of(out) < 0 || !result(args[10], a.rows, b.rows, out, dev, &y)) Py_RETURN_NONE;
  const auto run = [&] {
    return lib.gemm(a.codes, a.scales, b.codes, b.scales, bias.p, bias.type, y.data_ptr(), type_of(out), int(a.rows), int(b.rows),
                    int(a.cols), stream(dev));
  };
  if (const int status = launched(run)) return failed(status, "tac_mxfp4_gemm");
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {               // X; 4-bit rows; bias, and, or not, out and workspace
  HANDLE_TH_ERRORS
  Rows4 w;
  Rows x;
  Vector bias;
  if (n != 6 && n != 8) Py_RETURN_NONE;
  const int64_t dev = device_of(a[0]);
  if (!x.of(a[0], dev) || !w.of(a + 1, dev) || w.cols != x.K || !bias.of(a[5], w.rows, dev)) Py_RETURN_NONE;
  const int N = int(w.rows);
  at::Tensor y, ws;
  if (!result(n == 8 ? a[6] : Py_None, x.M, N, x.t->scalar_type(), dev, &y)) Py_RETURN_NONE;
  const char *xp = static_cast<const char*>(x.t->const_data_ptr()), *yp = static_cast<const char*>(y.const_data_ptr());
  if (xp < yp + y.nbytes() && yp < xp + ((x.M - 1) * x.ld + x.K) * int64_t(x.t->element_size())) Py_RETURN_NONE;
  void* p = nullptr;
  int64_t bytes = int64_t(lib.linear_bytes(x.M, N, x.K));
  if (n == 8 && a[7] != Py_None) {
    const at::Tensor* t = tensor(a[7], dev);
    if (!t || t->scalar_type() != at::kByte || !t->is_contiguous()) Py_RETURN_NONE;
    const uintptr_t from = reinterpret_cast<uintptr_t>(t->data_ptr()), at = (from + 255) & ~uintptr_t(255);
    p = reinterpret_cast<void*>(at);
    bytes = std::max<int64_t>(t->numel() - int64_t(at - from), 0);
  } else if (bytes) {
    ws = empty({bytes}, at::kByte, dev);
    p = ws.data_ptr();
  }
  const auto run = [&] {
    return lib.linear(x.t->const_data_ptr(), x.type, x.ld, w.codes, w.scales, bias.p, bias.type, y.data_ptr(), x.type, p, uint64_t(bytes),
                      x.M, N, x.K, stream(dev));
  };
  if (const int status = launched(run)) return failed(status, "tac_linear_mxfp4");
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {       // logits, tokens, top
  HANDLE_TH_ERRORS
  Rows x;
  int64_t top;
  if (n != 3) Py_RETURN_NONE;
  const int64_t dev = device_of(a[0]);
  if (!x.of(a[0], dev) || !number(a[2], &top) || top < 0 || top > 32 || top > x.K) Py_RETURN_NONE;
  const at::Tensor* tokens = tensor(a[1], dev);
  if (!tokens || tokens->dim() != 1 || tokens->size(0) != x.M || !tokens->is_contiguous()) Py_RETURN_NONE;
  const bool wide = tokens->scalar_type() == at::kLong;
  if (!wide && tokens->scalar_type() != at::kInt) Py_RETURN_NONE;
  const at::Tensor lp = empty({x.M}, at::kFloat, dev), entropy = empty({x.M}, at::kFloat, dev);
  at::Tensor top_lp, ids;
  if (top) top_lp = empty({x.M, top}, at::kFloat, dev), ids = empty({x.M, top}, at::kInt, dev);
  const auto run = [&] {
    return lib.logprobs(x.t->const_data_ptr(), x.type, x.ld, tokens->const_data_ptr(), wide, x.M, x.K, int(top),
                        static_cast<float*>(lp.data_ptr()), static_cast<float*>(entropy.data_ptr()),
                        top ? static_cast<float*>(top_lp.data_ptr()) : nullptr, top ? static_cast<int32_t*>(ids.data_ptr()) : nullptr,
                        stream(dev));
  };
  if (const int status = launched(run)) return failed(status, "tac_token_logprobs");
  return top ? tuple(lp, entropy, top_lp, ids) : tuple(lp, entropy);
  END_HANDLE_TH_ERRORS
}

PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {                 // addresses, in the order of Entries; check
  void* p[9];
  if (n != 10 || !PyCallable_Check(a[9])) return PyErr_Format(PyExc_TypeError, "bind() takes 9 addresses and a function");
  for (int i = 0; i < 9; ++i)
    if (!(p[i] = PyLong_AsVoidPtr(a[i]))) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "a null address");
  lib = {reinterpret_cast<decltype(lib.rms_norm)>(p[0]),     reinterpret_cast<decltype(lib.rms_norm_i8)>(p[1]),
         reinterpret_cast<decltype(lib.dequantize)>(p[2]),   reinterpret_cast<decltype(lib.quantize)>(p[3]),
         reinterpret_cast<decltype(lib.values)>(p[4]),       reinterpret_cast<decltype(lib.gemm)>(p[5]),
         reinterpret_cast<decltype(lib.linear)>(p[6]),       reinterpret_cast<decltype(lib.linear_bytes)>(p[7]),
         reinterpret_cast<decltype(lib.logprobs)>(p[8])};
  Py_INCREF(a[9]);
  Py_XDECREF(check);
  check = a[9];
  Py_RETURN_NONE;
}

#define TAC_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {TAC_METHOD(bind),   TAC_METHOD(rms_norm), TAC_METHOD(rms_norm_i8), TAC_METHOD(dequantize_rows),
                         TAC_METHOD(quantize), TAC_METHOD(values), TAC_METHOD(gemm),        TAC_METHOD(linear),
                         TAC_METHOD(token_logprobs), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_front", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__front() { return PyModule_Create(&module); }
