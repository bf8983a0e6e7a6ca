// The eager calls of the 4-bit KV cache's entry points, for Python.
//
// A ctypes call of these functions spends some 7 us on the host: five attribute
// reads for each of ten tensors and the conversion of twenty arguments, more
// than the small kernels take.  Here the same checks read the tensors
// directly.  A function returns the entry point's status, or None for
// anything out of the ordinary -- a wrong type, size, device or layout, an
// argument that is not a tensor -- which kernels.py then diagnoses.
//
// bind(addresses) takes the entry points' addresses in the order of Entry.
#define PY_SSIZE_T_CLEAN
#include <torch/csrc/autograd/python_variable.h>

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/llamamps_b200.h"

namespace {

struct Entry {
  decltype(&lmps_rope_kv_append_q4) append;
  decltype(&lmps_gqa_decode_attention_q4) decode;
  decltype(&lmps_gqa_decode_attention_rope_q4) step;
  decltype(&lmps_prefill_attention_q4) prefill;
} entry;

constexpr auto kHalf = at::kHalf, kFloat = at::kFloat, kInt = at::kInt, kByte = at::kByte;

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
  // Element counts stay in 64 bits with these (others are refused by the entry points, through ctypes).
  void heads(int n_q, int n_kv, int head_dim) {
    ok = ok && n_q >= 1 && n_q <= 65535 && n_kv >= 1 && n_kv <= 65535 && head_dim == 128;
  }
};

// One layer's pools at arguments i, i + 1 and the block table at i + 2.
struct Pools {
  uint8_t *k = nullptr, *v = nullptr;
  int32_t* table = nullptr;
  int n_pages = 0, max_pages = 0;

  Pools(Args& A, int i, int page_size, int n_kv, int64_t rows) {
    const at::Tensor *kt = A.tensor(i), *vt = A.tensor(i + 1), *bt = A.tensor(i + 2);
    if (!A.ok) return;
    A.ok = kt->dim() == 3 && kt->size(1) == n_kv && kt->size(2) == static_cast<int64_t>(page_size) * 72 &&
           vt->sizes() == kt->sizes() && bt->dim() == 2 && bt->size(0) >= rows && kt->size(0) <= 0x7FFFFFFF &&
           bt->size(1) <= 0x7FFFFFFF;
    if (!A.ok) return;
    k = static_cast<uint8_t*>(A.data(i, kByte, kt->numel()));
    v = static_cast<uint8_t*>(A.data(i + 1, kByte, kt->numel()));
    table = static_cast<int32_t*>(A.data(i + 2, kInt, bt->numel()));
    n_pages = static_cast<int>(kt->size(0));
    max_pages = static_cast<int>(bt->size(1));
  }
};

struct Workspace {
  void* p = nullptr;
  size_t n = 0;
  Workspace(Args& A, int i) {
    if (!A.ok || A.a[i] == Py_None) return;
    const at::Tensor* t = A.tensor(i);
    if (!t || t->numel() == 0) return;
    p = A.data(i, kByte, -1);
    n = static_cast<size_t>(t->numel());
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

// qkv, pos, inv_freq, q_out, k_pool, v_pool, block_table, page_size, n_q, n_kv, head_dim, style, k_out, v_out, error
PyObject* append(PyObject* const* args, Py_ssize_t n) {
  Args A(args, n, 15);
  const int page = A.ok ? A.number(7) : 0, n_q = A.number(8), n_kv = A.number(9), hd = A.number(10), style = A.number(11);
  A.heads(n_q, n_kv, hd);
  const int64_t rows = A.rows(0), q_n = rows * n_q * hd, kv_n = rows * n_kv * hd;
  auto* qkv = half(A.data(0, kHalf, q_n + 2 * kv_n));
  auto* pos = static_cast<int32_t*>(A.data(1, kInt, -rows));
  auto* inv = static_cast<float*>(A.data(2, kFloat, hd / 2));
  auto* q = half(A.data(3, kHalf, q_n));
  const Pools P(A, 4, page, n_kv, rows);
  auto* k_out = half(A.optional(12, kHalf, kv_n));
  auto* v_out = half(A.optional(13, kHalf, kv_n));
  auto* err = static_cast<int32_t*>(A.optional(14, kInt, -1));
  return run(A, [&](void* s) {
    return entry.append(qkv, pos, inv, q, k_out, v_out, P.k, P.v, P.n_pages, P.table, P.max_pages, page, n_q, n_kv, hd,
                        static_cast<int>(rows), style, err, s);
  });
}

// q, k_pool, v_pool, block_table, seq_lens, out, workspace, page_size, n_q, n_kv, head_dim, max_seq_len, n_splits, error
PyObject* decode(PyObject* const* args, Py_ssize_t n) {
  Args A(args, n, 14);
  const int page = A.ok ? A.number(7) : 0, n_q = A.number(8), n_kv = A.number(9), hd = A.number(10);
  const int max_len = A.number(11), splits = A.number(12);
  A.heads(n_q, n_kv, hd);
  const int64_t rows = A.rows(0), q_n = rows * n_q * hd;
  auto* q = half(A.data(0, kHalf, q_n));
  const Pools P(A, 1, page, n_kv, rows);
  auto* lens = static_cast<int32_t*>(A.data(4, kInt, -rows));
  auto* out = half(A.data(5, kHalf, q_n));
  const Workspace W(A, 6);
  auto* err = static_cast<int32_t*>(A.optional(13, kInt, -1));
  return run(A, [&](void* s) {
    return entry.decode(q, P.k, P.v, P.n_pages, P.table, lens, out, W.p, W.n, P.max_pages, page, n_q, n_kv, hd,
                        static_cast<int>(rows), max_len, splits, err, s);
  });
}

// qkv, pos, inv_freq, k_pool, v_pool, block_table, seq_lens, out, workspace, page_size, n_q, n_kv, head_dim,
// max_seq_len, n_splits, style, error
PyObject* step(PyObject* const* args, Py_ssize_t n) {
  Args A(args, n, 17);
  const int page = A.ok ? A.number(9) : 0, n_q = A.number(10), n_kv = A.number(11), hd = A.number(12);
  const int max_len = A.number(13), splits = A.number(14), style = A.number(15);
  A.heads(n_q, n_kv, hd);
  const int64_t rows = A.rows(0), q_n = rows * n_q * hd;
  auto* qkv = half(A.data(0, kHalf, q_n + 2 * rows * n_kv * hd));
  auto* pos = static_cast<int32_t*>(A.data(1, kInt, -rows));
  auto* inv = static_cast<float*>(A.data(2, kFloat, hd / 2));
  const Pools P(A, 3, page, n_kv, rows);
  auto* lens = static_cast<int32_t*>(A.data(6, kInt, -rows));
  auto* out = half(A.data(7, kHalf, q_n));
  const Workspace W(A, 8);
  auto* err = static_cast<int32_t*>(A.optional(16, kInt, -1));
  return run(A, [&](void* s) {
    return entry.step(qkv, pos, inv, style, P.k, P.v, P.n_pages, P.table, lens, out, W.p, W.n, P.max_pages, page, n_q,
                      n_kv, hd, static_cast<int>(rows), max_len, splits, err, s);
  });
}

// q, k_pool, v_pool, block_table, out, batch, seq_len, page_size, n_q, n_kv, head_dim, max_seq_len, starts, q_lens,
// workspace, n_splits, error
PyObject* prefill(PyObject* const* args, Py_ssize_t n) {
  Args A(args, n, 17);
  const int batch = A.ok ? A.number(5) : 0, seq = A.number(6), page = A.number(7), n_q = A.number(8);
  const int n_kv = A.number(9), hd = A.number(10), max_len = A.number(11), splits = A.number(15);
  A.heads(n_q, n_kv, hd);
  const int64_t rows = static_cast<int64_t>(batch) * seq, q_n = rows * n_q * hd;
  A.ok = A.ok && batch >= 1 && seq >= 1 && rows <= 0x7FFFFFFF;
  auto* q = half(A.data(0, kHalf, q_n));
  const Pools P(A, 1, page, n_kv, batch);
  auto* out = half(A.data(4, kHalf, q_n));
  auto* starts = static_cast<int32_t*>(A.optional(12, kInt, -static_cast<int64_t>(batch)));
  auto* lens = static_cast<int32_t*>(A.optional(13, kInt, -static_cast<int64_t>(batch)));
  const Workspace W(A, 14);
  auto* err = static_cast<int32_t*>(A.data(16, kInt, -1));
  return run(A, [&](void* s) {
    return entry.prefill(q, P.k, P.v, P.n_pages, P.table, starts, lens, out, W.p, W.n, P.max_pages, page, n_q, n_kv, hd,
                         batch, seq, max_len, splits, err, s);
  });
}

PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long a, b, c, d;
  if (!PyArg_ParseTuple(args, "KKKK", &a, &b, &c, &d)) return nullptr;
  entry.append = reinterpret_cast<decltype(entry.append)>(a);
  entry.decode = reinterpret_cast<decltype(entry.decode)>(b);
  entry.step = reinterpret_cast<decltype(entry.step)>(c);
  entry.prefill = reinterpret_cast<decltype(entry.prefill)>(d);
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<F>)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<append>("append"),   method<decode>("decode"), method<step>("step"),
                         method<prefill>("prefill"), {"bind", bind, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "bind_q4", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// torch_version: the torch it was built against, whose tensors alone it can read.
PyMODINIT_FUNC PyInit_bind_q4() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", LMPS_TORCH_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
