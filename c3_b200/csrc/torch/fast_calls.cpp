// The calls of the 8-bit path (c3_b200/quant.py, norm.py, linear.py) for the usual case: operands
// well formed, outputs to be allocated. A single token's kernel takes a few microseconds, and checking
// a dozen attributes and allocating four tensors from Python takes longer than that; here both take
// about one. Each function answers None for anything unusual (an operand it would have to refuse, a
// tensor subclass, another device than the current one), and the Python wrapper then goes its own way,
// which also says what is wrong. A nonzero status of the C ABI is returned as a number.
//
// The entry points are those of libc3cu.so, handed over by address at import (`bind`).
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "c3cu.h"

namespace {

struct Entry {
  decltype(&c3cu_quantize_rows) quantize_rows;
  decltype(&c3cu_rms_norm_int8) rms_norm_int8;
  decltype(&c3cu_rms_norm_bwd_workspace) rms_norm_bwd_workspace;
  decltype(&c3cu_rms_norm_bwd) rms_norm_bwd;
  decltype(&c3cu_linear_int8_fwd) linear_int8_fwd;
  decltype(&c3cu_gemm_dw_int8_workspace) gemm_dw_int8_workspace;
  decltype(&c3cu_gemm_dw_int8) gemm_dw_int8;
} g_entry{};
bool g_bound = false;

// A plain tensor (or parameter) on the current device, else null.
const at::Tensor* tensor(PyObject* o, int dev) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.get_device() != dev || t.layout() != at::kStrided || t.is_conj() || t.is_neg()) return nullptr;
  return &t;
}

int64_t rounded16(int64_t k) { return (k + 15) / 16 * 16; }

// A [rows][cols] operand with unit column stride: its row stride, else -1.
int64_t rows_of(const at::Tensor* t, at::ScalarType type, int64_t rows, int64_t cols) {
  if (!t || t->scalar_type() != type || t->dim() != 2 || t->size(0) != rows || t->size(1) != cols) return -1;
  if (t->stride(1) != 1) return -1;
  if (rows <= 1) return rounded16(cols);
  return t->stride(0) >= cols ? t->stride(0) : -1;
}

bool vector_of(const at::Tensor* t, int64_t n) {
  return t && t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == n && t->is_contiguous();
}

at::Tensor empty(at::IntArrayRef size, at::ScalarType type, int dev) {
  return at::detail::empty_cuda(size, type, c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(dev)), c10::nullopt);
}

// int8 rows starting on 16 bytes (quant.empty_rows).
at::Tensor empty_rows(int64_t m, int64_t k, int dev) {
  at::Tensor q = empty({m, rounded16(k)}, at::kChar, dev);
  return k % 16 == 0 ? q : q.narrow(1, 0, k);
}

int dtype_code(const at::Tensor& t) {
  return t.scalar_type() == at::kFloat ? C3CU_DTYPE_F32 : t.scalar_type() == at::kBFloat16 ? C3CU_DTYPE_BF16 : -1;
}

c3cu_stream_t stream(int dev) {
  return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream();
}

float* f32(const at::Tensor& t) { return static_cast<float*>(t.data_ptr()); }

PyObject* wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }

PyObject* none() { Py_RETURN_NONE; }

// Runs `f` with the current device's index; C++ exceptions (an allocation that failed) become Python's.
template <class F>
PyObject* guarded(F f) {
  HANDLE_TH_ERRORS
  if (!g_bound) return none();
  return f(static_cast<int>(c10::cuda::current_device()));
  END_HANDLE_TH_ERRORS
}

PyObject* quantize_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 1) return none();
  return guarded([&](int dev) -> PyObject* {
    const at::Tensor* x = tensor(a[0], dev);
    if (!x || x->dim() != 2 || dtype_code(*x) < 0) return none();
    const int64_t M = x->size(0), K = x->size(1);
    const int64_t ldx = rows_of(x, x->scalar_type(), M, K);
    if (ldx < 0 || K < 1) return none();
    at::Tensor q = empty_rows(M, K, dev), scale = empty({M}, at::kFloat, dev);
    const int rc = g_entry.quantize_rows(x->data_ptr(), ldx, dtype_code(*x), static_cast<int8_t*>(q.data_ptr()),
                                         rounded16(K), f32(scale), M, K, stream(dev));
    if (rc != C3CU_OK) return PyLong_FromLong(rc);
    return Py_BuildValue("(NN)", wrap(std::move(q)), wrap(std::move(scale)));
  });
}

// (x, weight, eps, residual or None)
PyObject* rms_norm_int8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4 || !PyFloat_CheckExact(a[2])) return none();
  return guarded([&](int dev) -> PyObject* {
    const at::Tensor *x = tensor(a[0], dev), *w = tensor(a[1], dev);
    const double eps = PyFloat_AS_DOUBLE(a[2]);
    const bool has = a[3] != Py_None;
    const at::Tensor* res = has ? tensor(a[3], dev) : nullptr;
    if (!x || x->dim() != 2 || dtype_code(*x) < 0 || !(eps >= 0. && eps < 1e30)) return none();
    const int64_t M = x->size(0), K = x->size(1);
    const int64_t ldx = rows_of(x, x->scalar_type(), M, K);
    const int64_t ldr = has ? rows_of(res, x->scalar_type(), M, K) : 0;
    if (ldx < 0 || ldr < 0 || K < 1 || !vector_of(w, K)) return none();
    at::Tensor q = empty_rows(M, K, dev), scale = empty({M}, at::kFloat, dev), rstd = empty({M}, at::kFloat, dev);
    at::Tensor h;
    if (has) h = empty({M, K}, x->scalar_type(), dev);
    const int rc = g_entry.rms_norm_int8(x->data_ptr(), ldx, has ? res->data_ptr() : nullptr, ldr, dtype_code(*x),
                                         f32(*w), static_cast<float>(eps), has ? h.data_ptr() : nullptr, K,
                                         static_cast<int8_t*>(q.data_ptr()), rounded16(K), f32(scale), f32(rstd), M, K,
                                         stream(dev));
    if (rc != C3CU_OK) return PyLong_FromLong(rc);
    PyObject* ho;
    if (has) {
      ho = wrap(std::move(h));
    } else {
      ho = a[0];
      Py_INCREF(ho);
    }
    return Py_BuildValue("(NNNN)", wrap(std::move(q)), wrap(std::move(scale)), ho, wrap(std::move(rstd)));
  });
}

// (dy, h, weight, rstd, dh or None)
PyObject* rms_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5) return none();
  return guarded([&](int dev) -> PyObject* {
    const at::Tensor *dy = tensor(a[0], dev), *h = tensor(a[1], dev), *w = tensor(a[2], dev), *r = tensor(a[3], dev);
    const bool has = a[4] != Py_None;
    const at::Tensor* dh = has ? tensor(a[4], dev) : nullptr;
    if (!h || h->dim() != 2 || dtype_code(*h) < 0) return none();
    const int64_t M = h->size(0), K = h->size(1);
    const int64_t ldh = rows_of(h, h->scalar_type(), M, K), ldy = rows_of(dy, h->scalar_type(), M, K);
    const int64_t lddh = has ? rows_of(dh, h->scalar_type(), M, K) : 0;
    if (ldh < 0 || ldy < 0 || lddh < 0 || K < 1 || !vector_of(w, K) || !vector_of(r, M)) return none();
    at::Tensor dx = empty({M, K}, h->scalar_type(), dev), dw = empty({K}, at::kFloat, dev), ws;
    const size_t bytes = g_entry.rms_norm_bwd_workspace(M, K);
    if (bytes > 0) ws = empty({static_cast<int64_t>(bytes)}, at::kByte, dev);
    const int rc = g_entry.rms_norm_bwd(dy->data_ptr(), ldy, h->data_ptr(), ldh, has ? dh->data_ptr() : nullptr, lddh,
                                        dtype_code(*h), f32(*w), f32(*r), dx.data_ptr(), K, f32(dw), M, K,
                                        bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream(dev));
    if (rc != C3CU_OK) return PyLong_FromLong(rc);
    return Py_BuildValue("(NN)", wrap(std::move(dx)), wrap(std::move(dw)));
  });
}

// (Xq, x_scale, Wq, w_scale, b or None, relu, fp32 output, mask wanted)
PyObject* forward_int8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8) return none();
  return guarded([&](int dev) -> PyObject* {
    const at::Tensor *x = tensor(a[0], dev), *xs = tensor(a[1], dev), *w = tensor(a[2], dev), *ws = tensor(a[3], dev);
    const bool has = a[4] != Py_None, relu = a[5] == Py_True, wide = a[6] == Py_True, want = relu && a[7] == Py_True;
    const at::Tensor* b = has ? tensor(a[4], dev) : nullptr;
    if (!x || !w || x->dim() != 2 || w->dim() != 2) return none();
    const int64_t M = x->size(0), K = x->size(1), N = w->size(0);
    const int64_t ldx = rows_of(x, at::kChar, M, K), ldw = rows_of(w, at::kChar, N, K);
    if (ldx < 0 || ldw < 0 || K < 1 || K > C3CU_INT8_MAX_K || !vector_of(xs, M) || !vector_of(ws, N) ||
        (has && !vector_of(b, N)))
      return none();
    const int64_t words = (N + 31) / 32;
    at::Tensor y = empty({M, N}, wide ? at::kFloat : at::kBFloat16, dev), mask;
    if (want) mask = empty({M, words}, at::kInt, dev);
    const int rc = g_entry.linear_int8_fwd(
        static_cast<const int8_t*>(x->data_ptr()), ldx, f32(*xs), static_cast<const int8_t*>(w->data_ptr()), ldw,
        f32(*ws), has ? f32(*b) : nullptr, y.data_ptr(), N, wide ? C3CU_DTYPE_F32 : C3CU_DTYPE_BF16, relu ? 1 : 0,
        want ? static_cast<uint32_t*>(mask.data_ptr()) : nullptr, words, M, N, K, stream(dev));
    if (rc != C3CU_OK) return PyLong_FromLong(rc);
    PyObject* mo;
    if (want) {
      mo = wrap(std::move(mask));
    } else {
      mo = Py_None;
      Py_INCREF(mo);
    }
    return Py_BuildValue("(NN)", wrap(std::move(y)), mo);
  });
}

// (dZ, Xq, x_scale)
PyObject* grad_weight_int8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3) return none();
  return guarded([&](int dev) -> PyObject* {
    const at::Tensor *dz = tensor(a[0], dev), *x = tensor(a[1], dev), *xs = tensor(a[2], dev);
    if (!dz || !x || dz->dim() != 2 || x->dim() != 2) return none();
    const int64_t M = dz->size(0), N = dz->size(1), K = x->size(1);
    const int64_t lddz = rows_of(dz, at::kBFloat16, M, N), ldx = rows_of(x, at::kChar, M, K);
    if (lddz < 0 || ldx < 0 || !vector_of(xs, M)) return none();
    at::Tensor dw = empty({N, K}, at::kBFloat16, dev), ws;
    const size_t bytes = g_entry.gemm_dw_int8_workspace(M, N, K);
    if (bytes > 0) ws = empty({static_cast<int64_t>(bytes)}, at::kByte, dev);
    const int rc = g_entry.gemm_dw_int8(dz->data_ptr(), lddz, static_cast<const int8_t*>(x->data_ptr()), ldx, f32(*xs),
                                        dw.data_ptr(), K, M, N, K, bytes > 0 ? ws.data_ptr() : nullptr, bytes,
                                        stream(dev));
    if (rc != C3CU_OK) return PyLong_FromLong(rc);
    return wrap(std::move(dw));
  });
}

// The addresses of Entry's functions, in its order.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* p[7];
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "bind takes seven addresses");
    return nullptr;
  }
  for (int i = 0; i < 7; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  g_entry.quantize_rows = reinterpret_cast<decltype(g_entry.quantize_rows)>(p[0]);
  g_entry.rms_norm_int8 = reinterpret_cast<decltype(g_entry.rms_norm_int8)>(p[1]);
  g_entry.rms_norm_bwd_workspace = reinterpret_cast<decltype(g_entry.rms_norm_bwd_workspace)>(p[2]);
  g_entry.rms_norm_bwd = reinterpret_cast<decltype(g_entry.rms_norm_bwd)>(p[3]);
  g_entry.linear_int8_fwd = reinterpret_cast<decltype(g_entry.linear_int8_fwd)>(p[4]);
  g_entry.gemm_dw_int8_workspace = reinterpret_cast<decltype(g_entry.gemm_dw_int8_workspace)>(p[5]);
  g_entry.gemm_dw_int8 = reinterpret_cast<decltype(g_entry.gemm_dw_int8)>(p[6]);
  g_bound = true;
  Py_RETURN_NONE;
}

#define C3_FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {C3_FAST(bind),
                           C3_FAST(quantize_rows),
                           C3_FAST(rms_norm_int8),
                           C3_FAST(rms_norm_backward),
                           C3_FAST(forward_int8),
                           C3_FAST(grad_weight_int8),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_fast_calls", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fast_calls() { return PyModule_Create(&g_module); }
