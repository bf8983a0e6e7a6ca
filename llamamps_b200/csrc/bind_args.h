// Argument reading of the Python extensions (bind_q4.cpp, bind_q8.cpp): tensors
// are checked without going through Python attributes, and a call that is in
// any way out of the ordinary is left to kernels.py.
#pragma once

#define PY_SSIZE_T_CLEAN
#include <torch/csrc/autograd/python_variable.h>

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/llamamps_b200.h"

namespace {

constexpr auto kHalf = at::kHalf, kFloat = at::kFloat, kInt = at::kInt, kByte = at::kByte, kChar = at::kChar;

// The arguments of one call; ok turns false at the first that does not fit.
struct Args {
  PyObject* const* a;
  bool ok;
  int dev = -1;

  Args(PyObject* const* args, Py_ssize_t n, Py_ssize_t want) : a(args), ok(n == want) {}

  const at::Tensor* tensor(int i) {
    if (!ok || !THPVariable_Check(a[i])) {
      ok = false;
      return nullptr;
    }
    return &THPVariable_Unpack(a[i]);
  }
  // Address of argument i: this type, on the call's device (the first one sets it: the current one),
  // contiguous, exactly n elements (at least -n for n < 0).
  void* data(int i, at::ScalarType type, int64_t n) {
    const at::Tensor* t = tensor(i);
    if (!t) return nullptr;
    const int64_t m = t->numel();
    ok = t->scalar_type() == type && t->is_cuda() && t->is_contiguous() && (n >= 0 ? m == n : m >= -n);
    if (!ok) return nullptr;
    if (dev < 0) dev = t->get_device();
    ok = t->get_device() == dev;
    return ok ? t->data_ptr() : nullptr;
  }
  void* optional(int i, at::ScalarType type, int64_t n) { return ok && a[i] == Py_None ? nullptr : data(i, type, n); }
  int number(int i) {
    if (!ok) return 0;
    int overflow = 0;
    const long long v = PyLong_Check(a[i]) ? PyLong_AsLongLongAndOverflow(a[i], &overflow) : (ok = false, 0);
    if (overflow || v != static_cast<int>(v)) ok = false;
    return static_cast<int>(v);
  }
  int64_t rows(int i) {
    const at::Tensor* t = tensor(i);
    if (!t || t->dim() < 1 || t->size(0) > 0x7FFFFFFF) {
      ok = false;
      return 0;
    }
    return t->size(0);
  }
  // Address and row stride of argument i as rows of k elements: [rows, k], or [k] for one row; elements of a row
  // side by side, rows not overlapping.
  void* matrix(int i, at::ScalarType type, int64_t rows, int64_t k, int& ld) {
    const at::Tensor* t = tensor(i);
    if (!t) return nullptr;
    const int64_t d = t->dim();
    ok = t->scalar_type() == type && t->is_cuda() && (d == 2 ? t->size(0) == rows : d == 1 && rows == 1) &&
         t->size(-1) == k && (k == 1 || t->stride(-1) == 1);
    if (!ok) return nullptr;
    const int64_t apart = rows > 1 ? t->stride(0) : (k + 15) / 16 * 16;
    if (dev < 0) dev = t->get_device();
    ok = t->get_device() == dev && apart >= k && apart <= 0x7FFFFFFF;
    ld = static_cast<int>(apart);
    return ok ? t->data_ptr() : nullptr;
  }
  void* optional_matrix(int i, at::ScalarType type, int64_t rows, int64_t k, int& ld) {
    ld = 0;
    return ok && a[i] == Py_None ? nullptr : matrix(i, type, rows, k, ld);
  }
  // Rows and columns of the matrix at argument i.
  void shape(int i, int64_t& rows, int64_t& k) {
    const at::Tensor* t = tensor(i);
    if (!t || t->dim() < 1 || t->dim() > 2) {
      ok = false;
      return;
    }
    rows = t->dim() == 2 ? t->size(0) : 1;
    k = t->size(-1);
    ok = rows >= 1 && rows <= 0x7FFFFFFF && k >= 1 && k <= 0x7FFFFFFF;
  }
  // Element counts stay in 64 bits with these (others are refused by the entry points, through ctypes).
  void heads(int n_q, int n_kv, int head_dim) {
    ok = ok && n_q >= 1 && n_q <= 65535 && n_kv >= 1 && n_kv <= 65535 && head_dim == 128;
  }
};

uint16_t* half(void* p) { return static_cast<uint16_t*>(p); }

// Calls on the current stream where the tensors are on the current device.
template <class Call>
PyObject* run(Args& A, Call call) {
  if (!A.ok || A.dev != c10::cuda::current_device()) Py_RETURN_NONE;
  void* stream = c10::cuda::getCurrentCUDAStream(A.dev).stream();
  int status;
  Py_BEGIN_ALLOW_THREADS;
  status = call(stream);
  Py_END_ALLOW_THREADS;
  return PyLong_FromLong(status);
}

template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n) {
  try {
    return F(args, n);
  } catch (...) {  // (a tensor without storage, and the like)
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<F>)), METH_FASTCALL, nullptr};
}

}  // namespace
