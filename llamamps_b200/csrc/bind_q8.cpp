// The eager calls of the 8-bit linear layers' entry points, for Python (see
// bind_q4.cpp: the entry point's status comes back, or None for anything that
// kernels.py has to diagnose).
//
// bind(addresses) takes the entry points' addresses in the order of Entry.
#include "bind_args.h"

namespace {

struct Entry {
  decltype(&lmps_quantise_rows_q8) quantise;
  decltype(&lmps_rms_norm_q8) norm;
  decltype(&lmps_w8a8_gemm) gemm;
} entry;

// x, codes, scales, values
PyObject* quantise(PyObject* const* args, Py_ssize_t n) {
  Args A(args, n, 4);
  int64_t rows = 0, k = 0;
  A.shape(0, rows, k);
  int ldx = 0, ldc = 0, ldv = 0;
  auto* x = half(A.matrix(0, kHalf, rows, k, ldx));
  auto* codes = static_cast<int8_t*>(A.matrix(1, kChar, rows, k, ldc));
  auto* scales = static_cast<float*>(A.data(2, kFloat, rows));
  auto* values = half(A.optional_matrix(3, kHalf, rows, k, ldv));
  return run(A, [&](void* s) {
    return entry.quantise(x, ldx, codes, ldc, scales, values, ldv, static_cast<int>(rows), static_cast<int>(k), s);
  });
}

// x, gamma, eps, residual, sum_out, codes, scales, values
PyObject* norm(PyObject* const* args, Py_ssize_t n) {
  Args A(args, n, 8);
  int64_t rows = 0, k = 0;
  A.shape(0, rows, k);
  int ldx = 0, ldr = 0, lds = 0, ldc = 0, ldv = 0;
  auto* x = half(A.matrix(0, kHalf, rows, k, ldx));
  auto* gamma = half(A.data(1, kHalf, k));
  const double eps = A.ok && PyFloat_Check(args[2]) ? PyFloat_AS_DOUBLE(args[2]) : (A.ok = false, 0.0);
  auto* residual = half(A.optional_matrix(3, kHalf, rows, k, ldr));
  auto* sum = half(A.optional_matrix(4, kHalf, rows, k, lds));
  auto* codes = static_cast<int8_t*>(A.matrix(5, kChar, rows, k, ldc));
  auto* scales = static_cast<float*>(A.data(6, kFloat, rows));
  auto* values = half(A.optional_matrix(7, kHalf, rows, k, ldv));
  return run(A, [&](void* s) {
    return entry.norm(x, ldx, residual, ldr, sum, lds, gamma, static_cast<float>(eps), codes, ldc, scales, values, ldv,
                      static_cast<int>(rows), static_cast<int>(k), s);
  });
}

// codes, scales, w_codes, w_scales, bias, residual, swiglu (0 or 1), out, error
PyObject* gemm(PyObject* const* args, Py_ssize_t n) {
  Args A(args, n, 9);
  int64_t m = 0, k = 0, w_rows = 0, w_k = 0;
  A.shape(0, m, k);
  A.shape(2, w_rows, w_k);
  const int gated = A.number(6);
  A.ok = A.ok && w_k == k && (gated == 0 || (gated == 1 && w_rows % 2 == 0 && args[4] == Py_None && args[5] == Py_None));
  const int64_t cols = gated ? w_rows / 2 : w_rows;
  int ldx = 0, ldw = 0, ldr = 0, ldy = 0;
  auto* x = static_cast<int8_t*>(A.matrix(0, kChar, m, k, ldx));
  auto* xs = static_cast<float*>(A.data(1, kFloat, m));
  auto* w = static_cast<int8_t*>(A.matrix(2, kChar, w_rows, k, ldw));
  auto* ws = static_cast<float*>(A.data(3, kFloat, w_rows));
  auto* bias = half(A.optional(4, kHalf, cols));
  auto* residual = half(A.optional_matrix(5, kHalf, m, cols, ldr));
  auto* y = half(A.matrix(7, kHalf, m, cols, ldy));
  auto* err = static_cast<int32_t*>(A.data(8, kInt, -1));
  A.ok = A.ok && ldx % 16 == 0 && ldw % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(w) % 16 == 0;
  return run(A, [&](void* s) {
    return entry.gemm(x, ldx, xs, w, ldw, ws, bias, residual, ldr, y, ldy, static_cast<int>(m), static_cast<int>(cols),
                      static_cast<int>(k), gated, err, s);
  });
}

PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long a, b, c;
  if (!PyArg_ParseTuple(args, "KKK", &a, &b, &c)) return nullptr;
  entry.quantise = reinterpret_cast<decltype(entry.quantise)>(a);
  entry.norm = reinterpret_cast<decltype(entry.norm)>(b);
  entry.gemm = reinterpret_cast<decltype(entry.gemm)>(c);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {method<quantise>("quantise"),
                         method<norm>("norm"),
                         method<gemm>("gemm"),
                         {"bind", bind, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "bind_q8", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// torch_version: the torch it was built against, whose tensors alone it can read.
PyMODINIT_FUNC PyInit_bind_q8() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", LMPS_TORCH_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
