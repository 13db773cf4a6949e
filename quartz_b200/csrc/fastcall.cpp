// fastcall.cpp -- the paged-cache calls of quartz_b200.device without their Python
// argument handling.
//
// A decode step's calls take 2 to 10 us on the GPU; checking their tensors in
// Python and passing two dozen arguments through ctypes takes longer than that
// (12 to 14 us a call). The functions here look at the same tensors directly and
// call the same C entry points. They take only what is right: on anything else
// (a wrong type or shape, another current device, stream capture without a
// workspace, arguments that the library refuses) they return None, having queued
// nothing, and the Python function goes through its checks and says what is wrong. A
// failure of CUDA is raised here: one of a call's launches may be queued by then.
#include <torch/csrc/autograd/python_variable.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <ATen/ATen.h>

#include <map>
#include <utility>

#include "quartz_b200.h"

namespace {

struct Entry {
  decltype(&qz_kv4_plan) plan;
  decltype(&qz_kv4_append) append;
  decltype(&qz_kv4_gather) gather;
  decltype(&qz_kv4_attention) attention;
  decltype(&qz_kv4_attention_workspace_bytes) attention_ws;
  decltype(&qz_last_error) last_error;
} entry{};
PyObject* quartz_error = nullptr;   // the exception class of a CUDA failure

uint64_t ready = 0;   // devices that ensure_device has seen
std::map<std::pair<int, cudaStream_t>, std::pair<void*, size_t>> workspaces;

PyObject* decline() { Py_RETURN_NONE; }

// The result of a call that the library did not take.
PyObject* failed(int rc) {
  if (rc != QZ_ERR_CUDA) return decline();
  char msg[512];
  entry.last_error(msg, sizeof msg);
  PyErr_SetString(quartz_error, msg);
  return nullptr;
}

// The tensor behind an argument, or null.
const at::Tensor* tensor(PyObject* o) {
  return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
}

bool is(const at::Tensor* t, at::ScalarType type, int64_t ndim, int idx) {
  return t && t->scalar_type() == type && t->dim() == ndim && t->is_cuda() &&
         t->get_device() == idx && t->is_contiguous();
}

int dtype_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return QZ_F32;
    case at::kBFloat16: return QZ_BF16;
    case at::kHalf: return QZ_F16;
    default: return -1;
  }
}

// Rows [n, heads, hd] on GPU idx, hd contiguous.
bool rows(const at::Tensor* t, int idx) {
  return t && t->dim() == 3 && t->is_cuda() && t->get_device() == idx && dtype_of(*t) >= 0 &&
         t->stride(2) == 1;
}

// Page size of a pool's blocks, or 0.
int64_t page_size(const at::Tensor& pool, int64_t hd) {
  if (hd != 64 && hd != 128) return 0;
  const int64_t bytes = pool.size(2);
  for (int64_t ps = 16; ps <= 256; ps *= 2)
    if (ps * (hd + 8) == bytes) return ps;
  return 0;
}

// Whether GPU idx is initialised and current.
bool here(int idx) {
  return idx >= 0 && idx < 64 && (ready >> idx & 1) && c10::cuda::current_device() == idx;
}

// A pool, its device, or -1.
int home(const at::Tensor* pool) {
  if (!pool || !pool->is_cuda()) return -1;
  const int idx = pool->get_device();
  return here(idx) && is(pool, at::kByte, 3, idx) ? idx : -1;
}

bool integer(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  *v = PyLong_AsLongLong(o);
  if (*v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

// `n` int64 elements of buf from `at` on, as a tensor of their own.
at::Tensor part(const at::Tensor& buf, int64_t at, int64_t n) {
  at::Tensor v = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buf.storage()), buf.key_set(),
                                                          buf.dtype());
  v.unsafeGetTensorImpl()->set_storage_offset(at);
  v.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return v;
}

// (lens, new_rows, block_table, free_pages, used, page_size, rows, lens_out, used_out)
// -> (cu_rows, lens, used, slots, positions)
PyObject* plan(PyObject*, PyObject* const* a, Py_ssize_t na) try {
  if (na != 9) return decline();
  const at::Tensor *lens = tensor(a[0]), *joins = tensor(a[1]), *table = tensor(a[2]),
                   *free_pages = tensor(a[3]), *used = tensor(a[4]);
  int64_t ps, n;
  if (!lens || !lens->is_cuda() || !integer(a[5], &ps) || !integer(a[6], &n) || n < 0) return decline();
  const int idx = lens->get_device();
  if (!here(idx) || !is(lens, at::kLong, 1, idx) || !is(joins, at::kLong, 1, idx) ||
      !is(table, at::kInt, 2, idx) || !is(free_pages, at::kInt, 1, idx) || !is(used, at::kLong, 1, idx))
    return decline();
  const int64_t B = table->size(0);
  if (lens->numel() != B || joins->numel() != B || used->numel() != 1) return decline();
  const bool own_lens = a[7] == Py_None, own_used = a[8] == Py_None;
  const at::Tensor *lo = own_lens ? nullptr : tensor(a[7]), *uo = own_used ? nullptr : tensor(a[8]);
  if (!own_lens && !(is(lo, at::kLong, 1, idx) && lo->numel() == B)) return decline();
  if (!own_used && !(is(uo, at::kLong, 1, idx) && uo->numel() == 1)) return decline();
  const at::Tensor buf = at::empty({2 * B + 2 + 2 * n}, lens->options());
  int64_t* p = buf.data_ptr<int64_t>();
  const int64_t at_len = B + 1, at_used = 2 * B + 1, at_slots = 2 * B + 2, at_pos = at_slots + n;
  if (const int rc = entry.plan(lens->data_ptr<int64_t>(), joins->data_ptr<int64_t>(), B, table->data_ptr<int32_t>(),
                 table->size(1), free_pages->data_ptr<int32_t>(), free_pages->numel(),
                 used->data_ptr<int64_t>(), ps, n, p, own_lens ? p + at_len : lo->data_ptr<int64_t>(),
                 own_used ? p + at_used : uo->data_ptr<int64_t>(), p + at_slots, p + at_pos,
                 c10::cuda::getCurrentCUDAStream(idx).stream()))
    return failed(rc);
  PyObject* out = PyTuple_New(5);
  if (!out) return nullptr;
  auto put = [&](int i, PyObject* o) { PyTuple_SET_ITEM(out, i, o); };
  put(0, THPVariable_Wrap(part(buf, 0, B + 1)));
  put(1, own_lens ? THPVariable_Wrap(part(buf, at_len, B)) : Py_NewRef(a[7]));
  put(2, own_used ? THPVariable_Wrap(part(buf, at_used, 1)) : Py_NewRef(a[8]));
  put(3, THPVariable_Wrap(part(buf, at_slots, n)));
  put(4, THPVariable_Wrap(part(buf, at_pos, n)));
  return out;
} catch (...) {
  return decline();
}

// (k, v, pool, slots) -> True
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t na) try {
  if (na != 4) return decline();
  const at::Tensor *k = tensor(a[0]), *v = tensor(a[1]), *pool = tensor(a[2]), *slots = tensor(a[3]);
  const int idx = home(pool);
  if (idx < 0 || !rows(k, idx) || !rows(v, idx) || k->scalar_type() != v->scalar_type() ||
      k->sizes() != v->sizes() || !is(slots, at::kLong, 1, idx))
    return decline();
  const int64_t n = k->size(0), nkv = k->size(1), hd = k->size(2), ps = page_size(*pool, hd);
  if (!ps || pool->size(1) != nkv || slots->numel() != n) return decline();
  if (const int rc = entry.append(k->data_ptr(), v->data_ptr(), dtype_of(*k), k->stride(0), k->stride(1), v->stride(0),
                   v->stride(1), n, static_cast<int>(nkv), static_cast<int>(hd), pool->data_ptr<uint8_t>(),
                   pool->size(0), ps, slots->data_ptr<int64_t>(),
                   c10::cuda::getCurrentCUDAStream(idx).stream()))
    return failed(rc);
  Py_RETURN_TRUE;
} catch (...) {
  return decline();
}

// (pool, slots, head_dim) -> (k, v)
PyObject* gather(PyObject*, PyObject* const* a, Py_ssize_t na) try {
  if (na != 3) return decline();
  const at::Tensor *pool = tensor(a[0]), *slots = tensor(a[1]);
  int64_t hd;
  const int idx = home(pool);
  if (idx < 0 || !is(slots, at::kLong, 1, idx) || !integer(a[2], &hd)) return decline();
  const int64_t ps = page_size(*pool, hd), n = slots->numel(), nkv = pool->size(1);
  if (!ps) return decline();
  const auto opts = pool->options().dtype(at::kFloat);
  const at::Tensor k = at::empty({n, nkv, hd}, opts), v = at::empty({n, nkv, hd}, opts);
  if (const int rc = entry.gather(pool->data_ptr<uint8_t>(), pool->size(0), ps, static_cast<int>(nkv),
                   static_cast<int>(hd), slots->data_ptr<int64_t>(), n, k.data_ptr<float>(),
                   v.data_ptr<float>(), c10::cuda::getCurrentCUDAStream(idx).stream()))
    return failed(rc);
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(k));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(v));
  return out;
} catch (...) {
  return decline();
}

// (q, pool, block_table, lens, cu_rows, max_rows, scale, out, workspace) -> out
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t na) try {
  if (na != 9) return decline();
  const at::Tensor *q = tensor(a[0]), *pool = tensor(a[1]), *table = tensor(a[2]), *lens = tensor(a[3]);
  const bool no_cu = a[4] == Py_None, no_out = a[7] == Py_None, no_ws = a[8] == Py_None;
  int64_t max_rows;
  const int idx = home(pool);
  if (idx < 0 || !rows(q, idx) || !is(table, at::kInt, 2, idx) || !is(lens, at::kLong, 1, idx))
    return decline();
  if (a[5] == Py_None)
    max_rows = no_cu || q->size(0) < 1 ? 1 : q->size(0);
  else if (!integer(a[5], &max_rows))
    return decline();
  const int64_t n = q->size(0), nq = q->size(1), hd = q->size(2), ps = page_size(*pool, hd);
  const int64_t nkv = pool->size(1), B = table->size(0);
  if (!ps || nkv < 1 || nq % nkv || lens->numel() != B) return decline();
  const at::Tensor* cu = no_cu ? nullptr : tensor(a[4]);
  if (!no_cu && !(is(cu, at::kLong, 1, idx) && cu->numel() == B + 1)) return decline();
  double scale;
  if (a[6] == Py_None) {
    scale = 1.0 / std::sqrt(static_cast<double>(hd));
  } else if (PyFloat_CheckExact(a[6])) {
    scale = PyFloat_AS_DOUBLE(a[6]);
  } else {
    return decline();
  }
  at::Tensor made;
  const at::Tensor* out = no_out ? nullptr : tensor(a[7]);
  if (no_out) {
    // rows that no request has, or that are not computed, are zeros
    made = no_cu && n <= B ? at::empty({n, nq, hd}, q->options()) : at::zeros({n, nq, hd}, q->options());
    out = &made;
  } else {
    if (!rows(out, idx) || out->scalar_type() != q->scalar_type() || out->sizes() != q->sizes())
      return decline();
    const int64_t s0 = out->stride(0), s1 = out->stride(1);   // rows and heads must not overlap
    if (!(((nq == 1 || s1 >= hd) && (n == 1 || s0 >= (nq - 1) * s1 + hd)) ||
          ((n == 1 || s0 >= hd) && (nq == 1 || s1 >= (n - 1) * s0 + hd))))
      return decline();
  }
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream(idx).stream();
  void* ws = nullptr;
  size_t ws_bytes = 0;
  if (no_ws) {
    cudaStreamCaptureStatus status;
    if (cudaStreamIsCapturing(st, &status) != cudaSuccess || status != cudaStreamCaptureStatusNone)
      return decline();
    const auto it = workspaces.find({idx, st});
    if (it == workspaces.end()) return decline();
    ws = it->second.first;
    ws_bytes = it->second.second;
    int64_t need;
    if (entry.attention_ws(static_cast<int>(nq), static_cast<int>(nkv), static_cast<int>(hd), max_rows,
                           &need) != QZ_OK || static_cast<size_t>(need) > ws_bytes)
      return decline();
  } else {
    const at::Tensor* w = tensor(a[8]);
    if (!is(w, at::kByte, 1, idx)) return decline();
    ws = w->data_ptr();
    ws_bytes = static_cast<size_t>(w->numel());
  }
  const auto s = q->strides(), os = out->strides();
  if (const int rc = entry.attention(q->data_ptr(), dtype_of(*q), s[0], s[1], out->data_ptr(), os[0], os[1],
                      pool->data_ptr<uint8_t>(), pool->size(0), ps, table->data_ptr<int32_t>(),
                      table->size(1), lens->data_ptr<int64_t>(), no_cu ? nullptr : cu->data_ptr<int64_t>(),
                      B, n, max_rows, static_cast<int>(nq), static_cast<int>(nkv), static_cast<int>(hd),
                      static_cast<float>(scale), ws, ws_bytes, st))
    return failed(rc);
  return no_out ? THPVariable_Wrap(made) : Py_NewRef(a[7]);
} catch (...) {
  return decline();
}

// bind(error class, plan, append, gather, attention, attention_workspace_bytes, last_error): the
// entry points' addresses
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t na) {
  if (na != 7 || !PyExceptionClass_Check(a[0])) {
    PyErr_SetString(PyExc_TypeError, "bind takes an exception class and six addresses");
    return nullptr;
  }
  Py_INCREF(a[0]);
  Py_XSETREF(quartz_error, a[0]);
  ++a;
  void* p[6];
  for (int i = 0; i < 6; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) return PyErr_Occurred() ? nullptr : decline();
  }
  entry = Entry{reinterpret_cast<decltype(&qz_kv4_plan)>(p[0]),
                reinterpret_cast<decltype(&qz_kv4_append)>(p[1]),
                reinterpret_cast<decltype(&qz_kv4_gather)>(p[2]),
                reinterpret_cast<decltype(&qz_kv4_attention)>(p[3]),
                reinterpret_cast<decltype(&qz_kv4_attention_workspace_bytes)>(p[4]),
                reinterpret_cast<decltype(&qz_last_error)>(p[5])};
  Py_RETURN_NONE;
}

// device_ready(idx)
PyObject* device_ready(PyObject*, PyObject* arg) {
  const long idx = PyLong_AsLong(arg);
  if (idx == -1 && PyErr_Occurred()) return nullptr;
  if (entry.plan && idx >= 0 && idx < 64) ready |= uint64_t(1) << idx;
  Py_RETURN_NONE;
}

// workspace(idx, stream, address, bytes): the workspace of calls on a stream that
// bring none; the caller keeps the memory
PyObject* workspace(PyObject*, PyObject* const* a, Py_ssize_t na) {
  int64_t idx, st, p, n;
  if (na != 4 || !integer(a[0], &idx) || !integer(a[1], &st) || !integer(a[2], &p) || !integer(a[3], &n)) {
    PyErr_SetString(PyExc_TypeError, "workspace takes four integers");
    return nullptr;
  }
  workspaces[{static_cast<int>(idx), reinterpret_cast<cudaStream_t>(st)}] = {
      reinterpret_cast<void*>(p), static_cast<size_t>(n)};
  Py_RETURN_NONE;
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(plan), FAST(append), FAST(gather), FAST(attention), FAST(bind),
                         FAST(workspace), {"device_ready", device_ready, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastcall", "Paged-cache calls without Python argument handling.",
                      -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// The torch and the Python whose headers this was built with (quartz_b200/build.py).
extern "C" __attribute__((visibility("default"))) const char qz_fastcall_stamp[] = QZ_FASTCALL_STAMP;

PyMODINIT_FUNC PyInit__fastcall() { return PyModule_Create(&module); }
