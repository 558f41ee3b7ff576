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

#include <math.h>
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

// One option of every row: None or a number (for all rows, into *all), or a tensor of `type` [n].
const void* option(PyObject* o, const char* what, const char* name, at::ScalarType type, int64_t n, const at::Device& dev,
                   double* all) {
  if (THPVariable_Check(o)) return vector(o, what, name, type, n, -1, dev, false);
  *all = PyFloat_AsDouble(o);
  if (*all == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(what, "%s must be a number or a tensor", name);
  }
  return nullptr;
}

// sample(logits, u, temperature, top_k, top_p, min_p)
PyObject* sample(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = "sample";
  try {
    if (n != 6) refuse(what, "six arguments wanted, got %d", (int)n);
    int64_t ld;
    const at::Tensor& x = matrix(a[0], what, "logits", nullptr, &ld);
    const at::ScalarType type = x.scalar_type();
    if (type != at::kFloat && type != at::kBFloat16) refuse(what, "logits has type %s", at::toString(type));
    const at::Device dev = x.device();
    const int64_t rows = x.size(0), V = x.size(1);
    const void* u = vector(a[1], what, "u", at::kFloat, rows, -1, dev, false);
    double temp = 1.0, k = 0.0, p = 1.0, min_p = 0.0;
    const void* temps = option(a[2], what, "temperature", at::kFloat, rows, dev, &temp);
    const void* ks = option(a[3], what, "top_k", at::kInt, rows, dev, &k);
    const void* ps = option(a[4], what, "top_p", at::kFloat, rows, dev, &p);
    const void* mps = option(a[5], what, "min_p", at::kFloat, rows, dev, &min_p);
    if (!(k >= 0.0) || k != floor(k)) refuse(what, "top_k = %g", k);
    const On on(dev);
    const at::Tensor out[2] = {fresh({rows}, at::kInt, dev), fresh({rows}, at::kFloat, dev)};
    check(pl_sample_dev(x.data_ptr(), (size_t)(ld < V ? V : ld), rows, V, type == at::kBFloat16, (const float*)u,
                        (const float*)temps, temp, (const int32_t*)ks, k >= 1e9 ? 0 : (size_t)k, (const float*)ps, p,
                        (const float*)mps, min_p, out[0].data_ptr<int32_t>(), out[1].data_ptr<float>(), on.stream),
          what);
    return tuple_of(out, 2);
  } catch (const Refused& r) {
    PyErr_SetString(puffer_error, r.msg.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// The rows of an optional matrix of x's type and shape.
const void* like(PyObject* o, const char* what, const char* name, const at::Tensor& x, int64_t* ld) {
  const at::Device dev = x.device();
  const at::Tensor& t = matrix(o, what, name, &dev, ld);
  of_type(t, what, name, x.scalar_type());
  if (t.size(0) != x.size(0) || t.size(1) != x.size(1)) refuse(what, "%s has another shape", name);
  return t.data_ptr();
}

// block_norm(x, branch, gate, branch_weight, weight, scale, eps, post)
PyObject* block_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = "block_norm";
  try {
    if (n != 8) refuse(what, "eight arguments wanted, got %d", (int)n);
    int64_t ldx, ldb, ldg = 0;
    const at::Tensor& x = matrix(a[0], what, "x", nullptr, &ldx);
    const at::ScalarType type = x.scalar_type();
    if (type != at::kFloat && type != at::kBFloat16) refuse(what, "x has type %s", at::toString(type));
    const at::Device dev = x.device();
    const int64_t rows = x.size(0), cols = x.size(1);
    const void* branch = like(a[1], what, "branch", x, &ldb);
    const void* gate = a[2] == Py_None ? nullptr : like(a[2], what, "gate", x, &ldg);
    const void* w1 = vector(a[3], what, "branch_weight", at::kFloat, cols, -1, dev, true);
    const void* w2 = vector(a[4], what, "weight", at::kFloat, cols, -1, dev, true);
    const double scale = PyFloat_AsDouble(a[5]), eps = PyFloat_AsDouble(a[6]);
    const int post = PyObject_IsTrue(a[7]);
    if (PyErr_Occurred()) return nullptr;
    const On on(dev);
    at::Tensor out[4] = {fresh({rows, cols}, type, dev), fresh({rows, cols}, type, dev), at::Tensor(),
                         fresh({rows}, at::kFloat, dev)};
    if (post) out[2] = fresh({rows}, at::kFloat, dev);
    check(pl_block_norm_dev(x.data_ptr(), ldx, branch, ldb, gate, ldg, (const float*)w1, (const float*)w2, scale, eps,
                            (uint8_t)post, rows, cols, type == at::kBFloat16, out[0].data_ptr(), cols, out[1].data_ptr(),
                            cols, post ? out[2].data_ptr<float>() : nullptr, out[3].data_ptr<float>(), on.stream),
          what);
    return tuple_of(out, 4);
  } catch (const Refused& r) {
    PyErr_SetString(puffer_error, r.msg.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// block_norm_grad(dr, dy, branch, gate, r, rstd_branch, rstd, branch_weight, weight, scale, params)
PyObject* block_norm_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = "block_norm_grad";
  try {
    if (n != 11) refuse(what, "eleven arguments wanted, got %d", (int)n);
    int64_t lddr = 0, lddy, ldb, ldg = 0, ldr;
    const at::Tensor& r = matrix(a[4], what, "r", nullptr, &ldr);
    const at::ScalarType type = r.scalar_type();
    if (type != at::kFloat && type != at::kBFloat16) refuse(what, "r has type %s", at::toString(type));
    const at::Device dev = r.device();
    const int64_t rows = r.size(0), cols = r.size(1);
    const void* dr = a[0] == Py_None ? nullptr : like(a[0], what, "dr", r, &lddr);
    const void* dy = like(a[1], what, "dy", r, &lddy);
    const void* branch = like(a[2], what, "branch", r, &ldb);
    const void* gate = a[3] == Py_None ? nullptr : like(a[3], what, "gate", r, &ldg);
    const void* rstd_b = vector(a[5], what, "rstd_branch", at::kFloat, rows, -1, dev, true);
    const void* rstd = vector(a[6], what, "rstd", at::kFloat, rows, -1, dev, false);
    const void* w1 = vector(a[7], what, "branch_weight", at::kFloat, cols, -1, dev, true);
    const void* w2 = vector(a[8], what, "weight", at::kFloat, cols, -1, dev, true);
    const double scale = PyFloat_AsDouble(a[9]);
    const int params = PyObject_IsTrue(a[10]);
    if (PyErr_Occurred()) return nullptr;
    const On on(dev);
    at::Tensor out[5] = {fresh({rows, cols}, type, dev), fresh({rows, cols}, type, dev), at::Tensor(), at::Tensor(),
                         at::Tensor()};
    if (gate) out[2] = fresh({rows, cols}, type, dev);
    at::Tensor ws;
    size_t size = 0;
    if (params) {
      out[3] = fresh({cols}, at::kFloat, dev);
      out[4] = fresh({cols}, at::kFloat, dev);
      size = pl_block_norm_grad_ws(rows, cols);
      ws = fresh({(int64_t)size}, at::kByte, dev);
    }
    // a statistics tensor of no rows has no address, and there is nothing for the first norm to do then
    check(pl_block_norm_grad_dev(dr, lddr, dy, lddy, branch, ldb, gate, ldg, r.data_ptr(), ldr, (const float*)rstd_b,
                                 (const float*)rstd, (const float*)w1, (const float*)w2, scale, rows, cols,
                                 type == at::kBFloat16, out[0].data_ptr(), cols, out[1].data_ptr(), cols,
                                 gate ? out[2].data_ptr() : nullptr, cols, params ? out[3].data_ptr<float>() : nullptr,
                                 params ? out[4].data_ptr<float>() : nullptr, params ? ws.data_ptr() : nullptr, size,
                                 on.stream),
          what);
    return tuple_of(out, 5);
  } catch (const Refused& r) {
    PyErr_SetString(puffer_error, r.msg.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// A bf16 tensor [n][h][d] whose last dimension is contiguous, and its strides (h, d < 0: any).
const at::Tensor& heads(PyObject* o, const char* what, const char* name, const at::Device* dev, int64_t n, int64_t h,
                        int64_t d, size_t* token, size_t* head) {
  const at::Tensor& t = tensor(o, what, name);
  if (!t.is_cuda()) refuse(what, "%s must be a CUDA tensor", name);
  if (t.dim() != 3) refuse(what, "%s must have three dimensions, has %d", name, (int)t.dim());
  if (dev && t.device() != *dev) refuse(what, "%s is on %s, not on %s", name, t.device().str().c_str(), dev->str().c_str());
  of_type(t, what, name, at::kBFloat16);
  if ((n >= 0 && t.size(0) != n) || (h >= 0 && t.size(1) != h) || (d >= 0 && t.size(2) != d))
    refuse(what, "%s has shape %lld x %lld x %lld, %lld x %lld x %lld wanted", name, (long long)t.size(0),
           (long long)t.size(1), (long long)t.size(2), (long long)(n < 0 ? t.size(0) : n),
           (long long)(h < 0 ? t.size(1) : h), (long long)(d < 0 ? t.size(2) : d));
  if (t.size(2) > 1 && t.stride(2) != 1) refuse(what, "%s must be contiguous in its last dimension", name);
  *token = t.size(0) > 1 ? (size_t)t.stride(0) : 0;  // a stride over one value says nothing
  *head = t.size(1) > 1 ? (size_t)t.stride(1) : 0;
  return t;
}
// A contiguous f32 tensor [n][h][dk][dv] of states; NULL for None where that may be.
const float* states(PyObject* o, const char* what, const char* name, const pl_delta_shape& s, int64_t n,
                    const at::Device& dev, bool optional) {
  if (o == Py_None) {
    if (!optional) refuse(what, "%s is needed", name);
    return nullptr;
  }
  const at::Tensor& t = tensor(o, what, name);
  if (t.device() != dev) refuse(what, "%s is on %s, not on %s", name, t.device().str().c_str(), dev.str().c_str());
  of_type(t, what, name, at::kFloat);
  if (t.dim() != 4 || t.size(0) != n || t.size(1) != (int64_t)s.heads_v || t.size(2) != (int64_t)s.dk ||
      t.size(3) != (int64_t)s.dv)
    refuse(what, "%s has the wrong shape (%lld x %zu x %zu x %zu wanted)", name, (long long)n, s.heads_v, s.dk, s.dv);
  if (!t.is_contiguous()) refuse(what, "%s must be contiguous", name);
  return t.data_ptr<float>();
}
struct Delta {
  pl_delta_shape s = {};
  const at::Tensor *q, *k, *v;
  const float *g, *beta;
  at::Device dev = at::Device(at::kCPU);
  // q, k, v, g, beta from a[0], scale
  Delta(PyObject* const* a, const char* what, double scale) {
    q = &heads(a[0], what, "q", nullptr, -1, -1, -1, &s.q_token, &s.q_head);
    dev = q->device();
    const int64_t n = q->size(0), hk = q->size(1), dk = q->size(2);
    k = &heads(a[1], what, "k", &dev, n, hk, dk, &s.k_token, &s.k_head);
    v = &heads(a[2], what, "v", &dev, n, -1, -1, &s.v_token, &s.v_head);
    const int64_t hv = v->size(1);
    s.tokens = n;
    s.heads_k = hk;
    s.heads_v = hv;
    s.dk = dk;
    s.dv = v->size(2);
    s.scale = scale;
    if (hk < 1 || hv < 1 || hv % hk) refuse(what, "v has %lld heads, a multiple of q's %lld wanted", (long long)hv, (long long)hk);
    g = (const float*)vector(a[3], what, "g", at::kFloat, n, hv, dev, false);
    beta = (const float*)vector(a[4], what, "beta", at::kFloat, n, hv, dev, false);
  }
};
at::Tensor bytes(size_t n, const at::Device& dev) { return fresh({(int64_t)(n ? n : 1)}, at::kByte, dev); }

// delta_rule(q, k, v, g, beta, offsets or None, sequences, state or None, scale, save)
PyObject* delta_rule(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = "delta_rule";
  try {
    if (n != 10) refuse(what, "ten arguments wanted, got %d", (int)n);
    const double scale = PyFloat_AsDouble(a[8]);
    const int64_t seqs = PyLong_AsLongLong(a[6]);
    const int save = PyObject_IsTrue(a[9]);
    if (PyErr_Occurred()) return nullptr;
    Delta d(a, what, scale);
    if (seqs < 0) refuse(what, "%lld sequences", (long long)seqs);
    d.s.sequences = seqs;
    const void* offsets = vector(a[5], what, "offsets", at::kInt, seqs + 1, -1, d.dev, true);
    const float* state = states(a[7], what, "state", d.s, seqs, d.dev, true);
    const int64_t N = d.s.tokens, hv = d.s.heads_v, dk = d.s.dk, dv = d.s.dv;
    const On on(d.dev);
    at::Tensor out[3] = {fresh({N, hv, dv}, at::kBFloat16, d.dev), fresh({seqs, hv, dk, dv}, at::kFloat, d.dev), at::Tensor()};
    const size_t size = save ? 0 : pl_delta_ws(&d.s, 0), kept = pl_delta_saved(&d.s);
    const at::Tensor ws = bytes(size, d.dev);
    if (save) out[2] = bytes(kept, d.dev);
    check(pl_delta_dev(&d.s, d.q->data_ptr(), d.k->data_ptr(), d.v->data_ptr(), d.g, d.beta, (const int32_t*)offsets, state,
                       out[0].data_ptr(), out[1].data_ptr<float>(), save ? out[2].data_ptr() : nullptr, save ? kept : 0,
                       ws.data_ptr(), size, on.stream),
          what);
    return tuple_of(out, 3);
  } catch (const Refused& r) {
    PyErr_SetString(puffer_error, r.msg.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// delta_rule_grad(q, k, v, g, beta, offsets or None, sequences, do, dstate or None, scale, saved)
PyObject* delta_rule_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = "delta_rule_grad";
  try {
    if (n != 11) refuse(what, "eleven arguments wanted, got %d", (int)n);
    const double scale = PyFloat_AsDouble(a[9]);
    const int64_t seqs = PyLong_AsLongLong(a[6]);
    if (PyErr_Occurred()) return nullptr;
    Delta d(a, what, scale);
    if (seqs < 0) refuse(what, "%lld sequences", (long long)seqs);
    d.s.sequences = seqs;
    const void* offsets = vector(a[5], what, "offsets", at::kInt, seqs + 1, -1, d.dev, true);
    const int64_t N = d.s.tokens, hk = d.s.heads_k, hv = d.s.heads_v, dk = d.s.dk, dv = d.s.dv;
    size_t token, head;
    const at::Tensor& dout = heads(a[7], what, "do", &d.dev, N, hv, dv, &token, &head);
    const float* dfinal = states(a[8], what, "dstate", d.s, seqs, d.dev, true);
    const size_t size = pl_delta_ws(&d.s, 1), kept = pl_delta_saved(&d.s);
    const void* saved = vector(a[10], what, "saved", at::kByte, (int64_t)(kept ? kept : 1), -1, d.dev, false);
    const On on(d.dev);
    const at::Tensor out[6] = {fresh({N, hk, dk}, at::kBFloat16, d.dev), fresh({N, hk, dk}, at::kBFloat16, d.dev),
                               fresh({N, hv, dv}, at::kBFloat16, d.dev), fresh({N, hv}, at::kFloat, d.dev),
                               fresh({N, hv}, at::kFloat, d.dev),        fresh({seqs, hv, dk, dv}, at::kFloat, d.dev)};
    const at::Tensor ws = bytes(size, d.dev);
    check(pl_delta_grad_dev(&d.s, dout.data_ptr(), token, head, dfinal, d.q->data_ptr(), d.k->data_ptr(), d.v->data_ptr(),
                            d.g, d.beta, (const int32_t*)offsets, saved, kept, out[0].data_ptr(), out[1].data_ptr(),
                            out[2].data_ptr(), out[3].data_ptr<float>(), out[4].data_ptr<float>(), out[5].data_ptr<float>(),
                            ws.data_ptr(), size, on.stream),
          what);
    return tuple_of(out, 6);
  } catch (const Refused& r) {
    PyErr_SetString(puffer_error, r.msg.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// delta_rule_step(q, k, v, g, beta, state, scale, out or None)
PyObject* delta_rule_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = "delta_rule_step";
  try {
    if (n != 8) refuse(what, "eight arguments wanted, got %d", (int)n);
    const double scale = PyFloat_AsDouble(a[6]);
    if (PyErr_Occurred()) return nullptr;
    const Delta d(a, what, scale);
    const int64_t N = d.s.tokens, hv = d.s.heads_v, dk = d.s.dk, dv = d.s.dv;
    const float* state = states(a[5], what, "state", d.s, N, d.dev, false);
    const bool given = a[7] != Py_None;
    if (given) states(a[7], what, "out", d.s, N, d.dev, false);
    const On on(d.dev);
    const at::Tensor out[2] = {fresh({N, hv, dv}, at::kBFloat16, d.dev),
                               given ? tensor(a[7], what, "out") : fresh({N, hv, dk, dv}, at::kFloat, d.dev)};
    float* to = out[1].data_ptr<float>();
    const size_t all = (size_t)N * hv * dk * dv;
    if (to != state && to < state + all && state < to + all) refuse(what, "out overlaps state");
    check(pl_delta_step_dev(&d.s, d.q->data_ptr(), d.k->data_ptr(), d.v->data_ptr(), d.g, d.beta, state, to,
                            out[0].data_ptr(), on.stream),
          what);
    return tuple_of(out, 2);
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
    {"sample", (PyCFunction)(void (*)(void))sample, METH_FASTCALL, nullptr},
    {"block_norm", (PyCFunction)(void (*)(void))block_norm, METH_FASTCALL, nullptr},
    {"block_norm_grad", (PyCFunction)(void (*)(void))block_norm_grad, METH_FASTCALL, nullptr},
    {"delta_rule", (PyCFunction)(void (*)(void))delta_rule, METH_FASTCALL, nullptr},
    {"delta_rule_grad", (PyCFunction)(void (*)(void))delta_rule_grad, METH_FASTCALL, nullptr},
    {"delta_rule_step", (PyCFunction)(void (*)(void))delta_rule_step, METH_FASTCALL, nullptr},
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
