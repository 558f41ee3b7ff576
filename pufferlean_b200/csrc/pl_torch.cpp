// The Python module behind pufferlean_b200/tokens.py: takes torch tensors, checks them, allocates the results and the
// workspace from torch's allocator and calls the C entries of include/pufferlean_b200.h on torch's current stream.
// A call through ctypes cost 12 us (layer norm) to 20 us (a head with gradients) on the host beside its launches;
// small calls are bound by that.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdarg.h>

#include <string>

#include "../../include/pufferlean_b200.h"

namespace {

PyObject* puffer_error = nullptr;

struct Refused {
  std::string msg;
};
[[noreturn]] void refuse(const char* what, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  throw Refused{std::string(what) + ": " + buf};
}
void check(int rc, const char* what) {
  if (rc != PL_OK) throw Refused{std::string(what) + " failed (status " + std::to_string(rc) + "): " + pl_last_error()};
}

const at::Tensor& tensor(PyObject* o, const char* what, const char* name) {
  if (!THPVariable_Check(o)) refuse(what, "%s must be a tensor", name);
  return THPVariable_Unpack(o);
}

// A 2-D CUDA tensor whose rows are contiguous and do not overlap; *ld is its row stride in elements.
const at::Tensor& matrix(PyObject* o, const char* what, const char* name, const at::Device* dev, int64_t* ld) {
  const at::Tensor& t = tensor(o, what, name);
  if (!t.is_cuda()) refuse(what, "%s must be a CUDA tensor", name);
  if (t.dim() != 2) refuse(what, "%s must have two dimensions, has %d", name, (int)t.dim());
  if (dev && t.device() != *dev) refuse(what, "%s is on %s, not on %s", name, t.device().str().c_str(), dev->str().c_str());
  const int64_t rows = t.size(0), cols = t.size(1), st = t.stride(0), sc = t.stride(1);
  if (sc == 1 && st >= cols)
    *ld = st;
  else if (cols <= 1 && rows <= 1)
    *ld = 1;
  else if (cols == 1 && st >= 1)  // a stride over one value says nothing
    *ld = st;
  else if (rows <= 1 && sc == 1)
    *ld = cols;
  else
    refuse(what, "%s must have contiguous rows that do not overlap (strides %lld, %lld)", name, (long long)st, (long long)sc);
  return t;
}
void of_type(const at::Tensor& t, const char* what, const char* name, at::ScalarType type) {
  if (t.scalar_type() != type) refuse(what, "%s has type %s, not %s", name, at::toString(t.scalar_type()), at::toString(type));
}
// The address of a contiguous tensor of this type and shape (n, or n x k where k >= 0); NULL for None where that may be.
void* vector(PyObject* o, const char* what, const char* name, at::ScalarType type, int64_t n, int64_t k,
             const at::Device& dev, bool optional) {
  if (o == Py_None) {
    if (!optional) refuse(what, "%s is needed", name);
    return nullptr;
  }
  const at::Tensor& t = tensor(o, what, name);
  if (t.device() != dev) refuse(what, "%s is on %s, not on %s", name, t.device().str().c_str(), dev.str().c_str());
  of_type(t, what, name, type);
  if (k < 0 ? (t.dim() != 1 || t.size(0) != n) : (t.dim() != 2 || t.size(0) != n || t.size(1) != k))
    refuse(what, "%s has the wrong shape (%lld%s%s wanted)", name, (long long)n, k < 0 ? "" : " x ",
           k < 0 ? "" : std::to_string(k).c_str());
  if (!t.is_contiguous()) refuse(what, "%s must be contiguous", name);
  return t.data_ptr();
}

at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type, const at::Device& dev) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(dev));
}
PyObject* wrap(const at::Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}
template <size_t N>
PyObject* tuple_of(const at::Tensor (&ts)[N], size_t n) {
  PyObject* r = PyTuple_New((Py_ssize_t)n);
  if (!r) return nullptr;
  for (size_t i = 0; i < n; i++) {
    PyObject* o = wrap(ts[i]);
    if (!o) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, (Py_ssize_t)i, o);
  }
  return r;
}

int library_device() {
  int d;
  check(pl_get_device(&d), "pl_get_device");
  return d;
}
// The tensors' device for torch and for the library while a call runs, and torch's stream there. Both get back the
// device that each had: a caller may have given the library another one than torch's.
struct On {
  int was, now;
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit On(const at::Device& d) : was(library_device()), now(d.index()), guard(d) {
    check(pl_set_device(now), "pl_set_device");
    stream = c10::cuda::getCurrentCUDAStream(d.index()).stream();
  }
  ~On() {
    if (was != now) pl_set_device(was);
  }
};

// layer_norm(x, weight, bias, eps)
PyObject* layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = "layer_norm";
  try {
    if (n != 4) refuse(what, "four arguments wanted, got %d", (int)n);
    int64_t ldx;
    const at::Tensor& x = matrix(a[0], what, "x", nullptr, &ldx);
    const at::ScalarType type = x.scalar_type();
    if (type != at::kFloat && type != at::kBFloat16) refuse(what, "x has type %s", at::toString(type));
    const at::Device dev = x.device();
    const int64_t rows = x.size(0), cols = x.size(1);
    const void* w = vector(a[1], what, "weight", at::kFloat, cols, -1, dev, true);
    const void* b = vector(a[2], what, "bias", at::kFloat, cols, -1, dev, true);
    const double eps = PyFloat_AsDouble(a[3]);
    if (PyErr_Occurred()) return nullptr;
    const On on(dev);
    const at::Tensor out[3] = {fresh({rows, cols}, type, dev), fresh({rows}, at::kFloat, dev), fresh({rows}, at::kFloat, dev)};
    check(pl_layernorm_dev(x.data_ptr(), ldx, (const float*)w, (const float*)b, rows, cols, eps, type == at::kBFloat16,
                           out[0].data_ptr(), cols, out[1].data_ptr<float>(), out[2].data_ptr<float>(), on.stream),
          what);
    return tuple_of(out, 3);
  } catch (const Refused& r) {
    PyErr_SetString(puffer_error, r.msg.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// layer_norm_grad(dy, x, weight, mean, rstd, params)
PyObject* layer_norm_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = "layer_norm_grad";
  try {
    if (n != 6) refuse(what, "six arguments wanted, got %d", (int)n);
    int64_t ldx, lddy;
    const at::Tensor& x = matrix(a[1], what, "x", nullptr, &ldx);
    const at::ScalarType type = x.scalar_type();
    if (type != at::kFloat && type != at::kBFloat16) refuse(what, "x has type %s", at::toString(type));
    const at::Device dev = x.device();
    const int64_t rows = x.size(0), cols = x.size(1);
    const at::Tensor& dy = matrix(a[0], what, "dy", &dev, &lddy);
    of_type(dy, what, "dy", type);
    if (dy.size(0) != rows || dy.size(1) != cols) refuse(what, "dy and x differ in shape");
    const void* w = vector(a[2], what, "weight", at::kFloat, cols, -1, dev, true);
    const void* mean = vector(a[3], what, "mean", at::kFloat, rows, -1, dev, false);
    const void* rstd = vector(a[4], what, "rstd", at::kFloat, rows, -1, dev, false);
    const int params = PyObject_IsTrue(a[5]);
    if (params < 0) return nullptr;
    const On on(dev);
    at::Tensor out[3] = {fresh({rows, cols}, type, dev), at::Tensor(), at::Tensor()};
    at::Tensor ws;
    size_t size = 0;
    if (params) {
      out[1] = fresh({cols}, at::kFloat, dev);
      out[2] = fresh({cols}, at::kFloat, dev);
      size = pl_layernorm_grad_ws(rows, cols);
      ws = fresh({(int64_t)size}, at::kByte, dev);
    }
    check(pl_layernorm_grad_dev(dy.data_ptr(), lddy, x.data_ptr(), ldx, (const float*)w, (const float*)mean,
                                (const float*)rstd, rows, cols, type == at::kBFloat16, out[0].data_ptr(), cols,
                                params ? out[1].data_ptr<float>() : nullptr, params ? out[2].data_ptr<float>() : nullptr,
                                params ? ws.data_ptr() : nullptr, size, on.stream),
          what);
    return tuple_of(out, 3);
  } catch (const Refused& r) {
    PyErr_SetString(puffer_error, r.msg.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// vocab(what, x, w, ids, teacher or None, bias, temperature, row_scale, grad, dw_f32, piece_bytes)
PyObject* vocab(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = "vocab";
  try {
    if (n != 11) refuse(what, "eleven arguments wanted, got %d", (int)n);
    what = PyUnicode_AsUTF8(a[0]);
    if (!what) return nullptr;
    int64_t ldx, ldw;
    const at::Tensor& x = matrix(a[1], what, "x", nullptr, &ldx);
    of_type(x, what, "x", at::kBFloat16);
    const at::Device dev = x.device();
    const at::Tensor& w = matrix(a[2], what, "w", &dev, &ldw);
    of_type(w, what, "w", at::kBFloat16);
    const int64_t N = x.size(0), D = x.size(1), V = w.size(0);
    if (w.size(1) != D) refuse(what, "w has %lld columns, x has %lld", (long long)w.size(1), (long long)D);
    if (V == 0 || D == 0) refuse(what, "w has shape %lld x %lld", (long long)V, (long long)D);
    const bool distill = a[4] != Py_None;
    int64_t K = 0;
    const void *ids, *teacher = nullptr;
    double temperature = 1.0;
    if (distill) {
      const at::Tensor& i = tensor(a[3], what, "ids");
      if (i.dim() != 2 || i.size(1) == 0) refuse(what, "ids must have shape %lld x K with K > 0", (long long)N);
      K = i.size(1);
      ids = vector(a[3], what, "ids", at::kInt, N, K, dev, false);
      teacher = vector(a[4], what, "teacher", at::kFloat, N, K, dev, false);
      temperature = PyFloat_AsDouble(a[6]);
      if (PyErr_Occurred()) return nullptr;
    } else {
      ids = vector(a[3], what, "target", at::kInt, N, -1, dev, false);
    }
    const void* bias = vector(a[5], what, "bias", at::kBFloat16, V, -1, dev, true);
    const void* scale = vector(a[7], what, "row_scale", at::kFloat, N, -1, dev, true);
    const int grad = PyObject_IsTrue(a[8]), f32 = PyObject_IsTrue(a[9]);
    const size_t piece = PyLong_AsSize_t(a[10]);
    if (PyErr_Occurred()) return nullptr;
    const On on(dev);
    const bool aligned = D % 8 == 0 && ldx % 8 == 0 && ldw % 64 == 0 && (uintptr_t)x.data_ptr() % 16 == 0 &&
                         (uintptr_t)w.data_ptr() % 128 == 0;
    at::Tensor out[5] = {fresh({N}, at::kFloat, dev), fresh({N}, at::kFloat, dev), at::Tensor(), at::Tensor(), at::Tensor()};
    if (grad) {
      const at::ScalarType type = f32 ? at::kFloat : at::kBFloat16;
      out[2] = fresh({N, D}, at::kBFloat16, dev);
      out[3] = fresh({V, D}, type, dev);
      if (bias) out[4] = fresh({V}, type, dev);
    }
    const size_t size = pl_vocab_ws(N, V, D, K, bias != nullptr, grad, aligned, piece);
    const at::Tensor ws = fresh({(int64_t)size}, at::kByte, dev);
    float *loss = out[0].data_ptr<float>(), *lse = out[1].data_ptr<float>();
    int rc;
    if (grad) {
      void *dx = out[2].data_ptr(), *dw = out[3].data_ptr(), *db = bias ? out[4].data_ptr() : nullptr;
      rc = distill ? pl_vocab_distill_grad_dev(x.data_ptr(), ldx, w.data_ptr(), ldw, bias, (const int32_t*)ids,
                                               (const float*)teacher, K, temperature, (const float*)scale, N, V, D, loss,
                                               lse, dx, D, dw, D, db, (uint8_t)f32, piece, ws.data_ptr(), size, on.stream)
                   : pl_vocab_ce_grad_dev(x.data_ptr(), ldx, w.data_ptr(), ldw, bias, (const int32_t*)ids,
                                          (const float*)scale, N, V, D, loss, lse, dx, D, dw, D, db, (uint8_t)f32, piece,
                                          ws.data_ptr(), size, on.stream);
    } else {
      rc = distill ? pl_vocab_distill_dev(x.data_ptr(), ldx, w.data_ptr(), ldw, bias, (const int32_t*)ids,
                                          (const float*)teacher, K, temperature, N, V, D, loss, lse, ws.data_ptr(), size,
                                          on.stream)
                   : pl_vocab_ce_dev(x.data_ptr(), ldx, w.data_ptr(), ldw, bias, (const int32_t*)ids, N, V, D, loss, lse,
                                     ws.data_ptr(), size, on.stream);
    }
    check(rc, what);
    return tuple_of(out, grad ? 5 : 2);
  } catch (const Refused& r) {
    PyErr_SetString(puffer_error, r.msg.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// check(device index): waits for the device and raises if a wait inside one of the library's kernels ran out
PyObject* check_device(PyObject*, PyObject* o) {
  HANDLE_TH_ERRORS
  const char* what = "check";
  try {
    const long index = PyLong_AsLong(o);
    if (PyErr_Occurred()) return nullptr;
    if (index < 0 || index >= pl_device_count()) refuse(what, "no CUDA device %ld", index);
    const On on(at::Device(at::kCUDA, (c10::DeviceIndex)index));
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = pl_device_check();
    Py_END_ALLOW_THREADS
    check(rc, what);
    Py_RETURN_NONE;
  } catch (const Refused& r) {
    PyErr_SetString(puffer_error, r.msg.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// set_error(PufferError): the exception that refusals and failed calls raise
PyObject* set_error(PyObject*, PyObject* e) {
  Py_XINCREF(e);
  Py_XSETREF(puffer_error, e);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"layer_norm", (PyCFunction)(void (*)(void))layer_norm, METH_FASTCALL, nullptr},
    {"layer_norm_grad", (PyCFunction)(void (*)(void))layer_norm_grad, METH_FASTCALL, nullptr},
    {"vocab", (PyCFunction)(void (*)(void))vocab, METH_FASTCALL, nullptr},
    {"check", check_device, METH_O, nullptr},
    {"set_error", set_error, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "pl_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_pl_torch(void) {
  puffer_error = PyExc_RuntimeError;
  Py_INCREF(puffer_error);
  return PyModule_Create(&module);
}
