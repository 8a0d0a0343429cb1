// The usual calls of layer.py without its Python: on small operators the argument checks and the conversions of ctypes take longer
// than the launch (8 rows of layer norm: 7.8 us a call through them, 3.7 us from here; the product of one token 8.9 and 3.2, a norm's gradients 14.7
// and 7.4).
//
// Every function takes the operator's arguments by position, looks whether they are the usual ones (contiguous CUDA tensors
// of the right sizes and types on the current device; codes may have a pitch), and if so calls the C ABI and returns True.  Otherwise,
// and when the library refuses the arguments (which it does before it touches the device), it returns False and has done nothing:
// layer.py then checks one by one and says what is wrong.  Any other status comes back as a number: work may have been enqueued by
// then, and an operator that writes over its input must not be called a second time.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/b2blas.h"

namespace {

struct Library {
  decltype(&b2_layernorm) layernorm;
  decltype(&b2_layernorm_backward_workspace_bytes) layernorm_backward_workspace_bytes;
  decltype(&b2_layernorm_backward) layernorm_backward;
  decltype(&b2_w4_quantize) w4_quantize;
  decltype(&b2_w4_dequantize) w4_dequantize;
  decltype(&b2_w4_matvec_workspace_bytes) w4_matvec_workspace_bytes;
  decltype(&b2_w4_matvec) w4_matvec;
} lib;
PyObject *handles;      // blas.py's default handles, by device

struct Unusual {};      // thrown where layer.py's own path has to decide

int type_code(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return B2_F32;
    case at::kBFloat16: return B2_BF16;
    case at::kHalf: return B2_F16;
    default: throw Unusual();
  }
}

struct Call {
  PyObject *const *args;
  int next = 0;
  int device = -1;
  b2_handle handle = nullptr;
  void *stream = nullptr;
  explicit Call(PyObject *const *args) : args(args) {}

  PyObject *object() { return args[next++]; }
  int64_t integer() {
    PyObject *o = object();
    if (!PyLong_CheckExact(o)) throw Unusual();
    int overflow = 0;
    const long long v = PyLong_AsLongLongAndOverflow(o, &overflow);
    if (overflow) throw Unusual();
    return v;
  }
  float real() {
    PyObject *o = object();
    if (PyFloat_CheckExact(o)) return (float)PyFloat_AS_DOUBLE(o);
    --next;
    return (float)integer();
  }
  const at::Tensor &strided() {
    PyObject *o = object();
    if (!THPVariable_CheckExact(o)) throw Unusual();
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.layout() != at::kStrided) throw Unusual();
    if (device < 0) device = c10::cuda::current_device();
    if (t.get_device() != device) throw Unusual();
    return t;
  }
  const at::Tensor &tensor() {
    const at::Tensor &t = strided();
    if (!t.is_contiguous()) throw Unusual();
    return t;
  }
  // rows x cols, the rows counted over all leading dimensions.
  const at::Tensor &matrix(int64_t rows, int64_t cols) {
    const at::Tensor &t = tensor();
    if (t.dim() < 2 || t.size(-1) != cols || cols <= 0 || t.numel() / cols < rows) throw Unusual();
    return t;
  }
  // A contiguous vector of n elements at least, or nullptr for None.
  const at::Tensor *vector(int64_t n) {
    if (args[next] == Py_None) {
      ++next;
      return nullptr;
    }
    const at::Tensor &t = tensor();
    if (t.numel() < n) throw Unusual();
    return &t;
  }
  void *typed(int64_t n, at::ScalarType type) {
    const at::Tensor *t = vector(n);
    if (t && t->scalar_type() != type) throw Unusual();
    return t ? t->data_ptr() : nullptr;
  }
  // A parameter of the layer norm: FP32 or x's type, all that are given alike (`code`: -1 before the first).
  void *param(int64_t n, const at::Tensor &x, int &code) {
    const at::Tensor *t = vector(n);
    if (!t) return nullptr;
    const int c = type_code(*t);
    if ((c != B2_F32 && t->scalar_type() != x.scalar_type()) || (code >= 0 && code != c)) throw Unusual();
    code = c;
    return t->data_ptr();
  }
  // The caller's handle, or the device's default one (which blas.py makes), and the current stream; the first argument.
  void place(PyObject *h) {
    if (h == Py_None) {
      PyObject *key = PyLong_FromLong(device);
      h = key ? PyDict_GetItemWithError(handles, key) : nullptr;
      Py_XDECREF(key);
      if (!h) throw Unusual();
    }
    PyObject *raw = PyObject_GetAttrString(h, "_h"), *value = raw ? PyObject_GetAttrString(raw, "value") : nullptr;
    Py_XDECREF(raw);
    if (value && PyLong_CheckExact(value)) handle = (b2_handle)PyLong_AsVoidPtr(value);
    Py_XDECREF(value);
    if (!handle) throw Unusual();
    stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
  }
};

template <class F>
PyObject *guarded(Py_ssize_t given, Py_ssize_t wanted, F &&f) {
  int st = B2_ERR_INVALID_ARG;
  if (given == wanted && lib.layernorm) {
    try {
      st = f();
    } catch (...) {      // before the library's call, which throws nothing: layer.py meets the same and reports it
      st = B2_ERR_INVALID_ARG;
    }
  }
  PyErr_Clear();
  if (st == B2_OK) Py_RETURN_TRUE;
  if (st == B2_ERR_INVALID_ARG || st == B2_ERR_UNSUPPORTED || st == B2_ERR_WORKSPACE) Py_RETURN_FALSE;
  return PyLong_FromLong(st);
}
struct WithoutGil {
  PyThreadState *state = PyEval_SaveThread();
  ~WithoutGil() { PyEval_RestoreThread(state); }
};
template <class F>
int without_gil(F &&f) {
  const WithoutGil released;
  return f();
}
at::Tensor scratch(const at::Tensor &like, size_t bytes) { return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte).requires_grad(false)); }

// handle, rows, cols, eps, x, gamma, beta, y, mean, rstd
PyObject *layernorm(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded(n, 10, [&] {
    Call c(args);
    PyObject *h = c.object();
    const int64_t rows = c.integer(), cols = c.integer();
    const float eps = c.real();
    const at::Tensor &x = c.matrix(rows, cols);
    int code = -1;
    const int type = type_code(x);
    void *gamma = c.param(cols, x, code), *beta = c.param(cols, x, code);
    const at::Tensor &y = c.matrix(rows, cols);
    if (y.scalar_type() != x.scalar_type()) throw Unusual();
    float *mean = (float *)c.typed(rows, at::kFloat), *rstd = (float *)c.typed(rows, at::kFloat);
    c.place(h);
    return without_gil([&] {
      return lib.layernorm(c.handle, rows, cols, eps, type, x.data_ptr(), cols, code < 0 ? type : code, gamma, beta, y.data_ptr(), cols, mean,
                           rstd, c.stream);
    });
  });
}

// handle, rows, cols, dy, x, gamma, mean, rstd, dx, dgamma, dbeta, workspace
PyObject *layernorm_backward(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded(n, 12, [&] {
    Call c(args);
    PyObject *h = c.object();
    const int64_t rows = c.integer(), cols = c.integer();
    const at::Tensor &dy = c.matrix(rows, cols), &x = c.matrix(rows, cols);
    if (dy.scalar_type() != x.scalar_type()) throw Unusual();
    int code = -1;
    const int type = type_code(x);
    void *gamma = c.param(cols, x, code);
    const float *mean = (const float *)c.typed(rows, at::kFloat), *rstd = (const float *)c.typed(rows, at::kFloat);
    void *dx = nullptr;
    if (args[c.next] == Py_None) ++c.next;
    else {
      const at::Tensor &t = c.matrix(rows, cols);
      if (t.scalar_type() != x.scalar_type()) throw Unusual();
      dx = t.data_ptr();
    }
    void *dgamma = c.param(cols, x, code), *dbeta = c.param(cols, x, code);
    const at::Tensor *ws = c.vector(0);
    c.place(h);
    at::Tensor own;
    if (!ws && (dgamma || dbeta)) {
      own = scratch(x, lib.layernorm_backward_workspace_bytes(rows, cols));
      ws = &own;
    }
    return without_gil([&] {
      return lib.layernorm_backward(c.handle, rows, cols, type, dy.data_ptr(), cols, x.data_ptr(), cols, code < 0 ? type : code, gamma, mean,
                                    rstd, dx, cols, dgamma, dbeta, ws ? ws->data_ptr() : nullptr, ws ? ws->nbytes() : 0, c.stream);
    });
  });
}

// The arguments that the calls on 4-bit weights share: codes, scales, zeros.
struct Weights {
  uint8_t *codes, *zeros;
  void *scales;
  int64_t ldq;
  int scale_type;
  Weights(Call &c, int64_t N, int64_t K, int64_t group) {
    if (N <= 0 || K <= 0 || (group != 32 && group != 64 && group != 128 && group != 256)) throw Unusual();
    const int64_t count = N * ((K + group - 1) / group);
    const at::Tensor &q = c.strided();
    if (q.dim() != 2 || q.size(0) != N || q.size(1) != (K + 1) / 2 || (q.size(1) > 1 && q.stride(1) != 1)) throw Unusual();
    ldq = N > 1 ? q.stride(0) : q.size(1);
    const at::Tensor *s = c.vector(count);
    if (q.scalar_type() != at::kByte || !s) throw Unusual();
    codes = (uint8_t *)q.data_ptr();
    scales = s->data_ptr();
    scale_type = type_code(*s);
    zeros = (uint8_t *)c.typed(count, at::kByte);
  }
};

// handle, N, K, group, W, codes, scales, zeros
PyObject *w4_quantize(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded(n, 8, [&] {
    Call c(args);
    PyObject *h = c.object();
    const int64_t N = c.integer(), K = c.integer(), group = c.integer();
    const at::Tensor &w = c.matrix(N, K);
    const int type = type_code(w);
    const Weights q(c, N, K, group);
    c.place(h);
    return without_gil([&] {
      return lib.w4_quantize(c.handle, N, K, (int)group, type, w.data_ptr(), K, q.codes, q.ldq, q.scale_type, q.scales, q.zeros, c.stream);
    });
  });
}

// handle, N, K, group, codes, scales, zeros, transpose (0 or 1), W
PyObject *w4_dequantize(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded(n, 9, [&] {
    Call c(args);
    PyObject *h = c.object();
    const int64_t N = c.integer(), K = c.integer(), group = c.integer();
    const Weights q(c, N, K, group);
    const int64_t transpose = c.integer();
    const at::Tensor &w = c.matrix(transpose ? K : N, transpose ? N : K);
    const int type = type_code(w);
    c.place(h);
    return without_gil([&] {
      return lib.w4_dequantize(c.handle, N, K, (int)group, q.codes, q.ldq, q.scale_type, q.scales, q.zeros, type, w.data_ptr(),
                               transpose ? N : K, (int)transpose, c.stream);
    });
  });
}

// handle, M, N, K, group, alpha, x, codes, scales, zeros, beta, y, workspace
PyObject *w4_matvec(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded(n, 13, [&] {
    Call c(args);
    PyObject *h = c.object();
    const int64_t M = c.integer(), N = c.integer(), K = c.integer(), group = c.integer();
    const float alpha = c.real();
    const at::Tensor &x = c.matrix(M, K);
    const int type = type_code(x);
    const Weights q(c, N, K, group);
    const float beta = c.real();
    const at::Tensor &y = c.matrix(M, N);
    if (y.scalar_type() != x.scalar_type()) throw Unusual();
    const at::Tensor *ws = c.vector(0);
    c.place(h);
    at::Tensor own;
    if (!ws) {
      const size_t bytes = lib.w4_matvec_workspace_bytes(M, N, K, type);
      if (bytes) {
        own = scratch(x, bytes);
        ws = &own;
      }
    }
    return without_gil([&] {
      return lib.w4_matvec(c.handle, M, N, K, (int)group, alpha, type, x.data_ptr(), K, q.codes, q.ldq, q.scale_type, q.scales, q.zeros, beta,
                           y.data_ptr(), N, ws ? ws->data_ptr() : nullptr, ws ? ws->nbytes() : 0, c.stream);
    });
  });
}

// bind(handles, addresses of the library's functions in the order of Library)
PyObject *bind(PyObject *, PyObject *const *args, Py_ssize_t n) {
  void *at[7];
  if (n != 8 || !PyDict_Check(args[0])) {
    PyErr_SetString(PyExc_TypeError, "bind: a dict and 7 addresses");
    return nullptr;
  }
  for (int i = 0; i < 7; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i + 1]);
    if (PyErr_Occurred()) return nullptr;
  }
  Py_INCREF(args[0]);
  Py_XDECREF(handles);
  handles = args[0];
  lib.layernorm_backward_workspace_bytes = (decltype(lib.layernorm_backward_workspace_bytes))at[1];
  lib.layernorm_backward = (decltype(lib.layernorm_backward))at[2];
  lib.w4_quantize = (decltype(lib.w4_quantize))at[3];
  lib.w4_dequantize = (decltype(lib.w4_dequantize))at[4];
  lib.w4_matvec_workspace_bytes = (decltype(lib.w4_matvec_workspace_bytes))at[5];
  lib.w4_matvec = (decltype(lib.w4_matvec))at[6];
  lib.layernorm = (decltype(lib.layernorm))at[0];
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"bind", (PyCFunction)(void *)bind, METH_FASTCALL, nullptr},
                         {"layernorm", (PyCFunction)(void *)layernorm, METH_FASTCALL, nullptr},
                         {"layernorm_backward", (PyCFunction)(void *)layernorm_backward, METH_FASTCALL, nullptr},
                         {"w4_quantize", (PyCFunction)(void *)w4_quantize, METH_FASTCALL, nullptr},
                         {"w4_dequantize", (PyCFunction)(void *)w4_dequantize, METH_FASTCALL, nullptr},
                         {"w4_matvec", (PyCFunction)(void *)w4_matvec, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() {
  PyObject *m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", B2_BUILT_FOR_TORCH) < 0) Py_CLEAR(m);      // layer.py binds it to no other
  return m;
}
