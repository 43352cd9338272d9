// Short way from Python to the paged-cache operators of libbi.so.
//
// A decode step's plan and rotary write take the GPU 3 to 5 us; checking the arguments and
// calling the C ABI through ctypes took 24 us of the host's time, so that the host set the
// step's pace.  Each function here checks that its arguments are the plain case (exact tensor
// type, CUDA, the dtypes, shapes and strides that the kernels take as they are), allocates the
// outputs and calls the C ABI: 6 to 9 us.  Whatever is not the plain case returns None, and the
// Python function goes its full way, with its checks and messages; a status that is not 0 comes
// back as a number for it to raise.  No C++ exception leaves a function here: what torch throws
// becomes the Python exception that torch makes of it (running out of memory among them).
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <exception>
#include <optional>

#include "bi.h"

namespace {

decltype(&bi_paged_plan) g_plan = nullptr;
decltype(&bi_rope_kv_paged) g_rope = nullptr;
decltype(&bi_paged_sdpa) g_sdpa = nullptr;
decltype(&bi_paged_sdpa_workspace) g_workspace = nullptr;

using at::ScalarType;
using at::Tensor;

// All that a plain CUDA tensor's keys may be.  Tensors under vmap, jvp, grad or functionalize,
// nested ones and ones that only stand for zeros are of the exact tensor type too; they have a
// key more, and no storage or not their values in it.
constexpr c10::DispatchKeySet kPlainKeys =
    c10::DispatchKeySet({c10::DispatchKey::CUDA, c10::DispatchKey::AutogradCUDA,
                         c10::DispatchKey::AutocastCUDA, c10::DispatchKey::ADInplaceOrView});

// The tensor of a plain CUDA tensor argument, else null.
const Tensor* cuda_tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.is_cuda() && (t.key_set() | kPlainKeys) == kPlainKeys && t.has_storage()
             ? &t : nullptr;
}

// What F answers, or the Python exception of what it throws.
template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    return F(a, n);
  } catch (...) {
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
}

bool is_vector(const Tensor* t, ScalarType type, int64_t n, c10::Device dev) {
  return t != nullptr && t->dim() == 1 && t->scalar_type() == type && t->size(0) == n &&
         (n <= 1 || t->stride(0) == 1) && t->device() == dev;
}

bool is_table(const Tensor* t, int64_t rows, c10::Device dev) {
  return t != nullptr && t->dim() == 2 && t->scalar_type() == at::kInt && t->size(0) == rows &&
         (t->size(1) <= 1 || t->stride(1) == 1) && (rows <= 1 || t->stride(0) >= t->size(1)) &&
         t->device() == dev;
}

int dtype_code(ScalarType t) {
  return t == at::kFloat ? BI_F32 : t == at::kHalf ? BI_F16 : t == at::kBFloat16 ? BI_BF16 : -1;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A cache (pages, kv heads, page, D): its strides of page, head and token, where they are what
// the kernels take.
bool cache_strides(const Tensor* t, ScalarType type, c10::Device dev, int64_t (&s)[3]) {
  if (t == nullptr || t->dim() != 4 || t->scalar_type() != type || t->device() != dev ||
      t->numel() == 0 || t->stride(3) != 1 || !aligned16(t->data_ptr())) {
    return false;
  }
  const int64_t vec = 16 / static_cast<int64_t>(t->element_size());
  for (int i = 0; i < 3; ++i) {
    s[i] = t->size(i) > 1 ? t->stride(i) : t->size(3);
    if (s[i] <= 0 || s[i] % vec != 0) return false;
  }
  return true;
}

Tensor empty(at::IntArrayRef size, ScalarType type, c10::Device dev) {
  return at::detail::empty_cuda(size, type, dev, std::nullopt);
}

// A contiguous tensor over part of `store` (a byte tensor) from byte `at` on, which moves
// behind it: several small outputs from one allocation.
Tensor carve(const Tensor& store, int64_t& at, int64_t n, ScalarType type) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(
      c10::Storage(store.storage()), store.key_set(), c10::scalarTypeToTypeMeta(type));
  const int64_t size = static_cast<int64_t>(c10::elementSize(type));
  t.unsafeGetTensorImpl()->set_storage_offset(at / size);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  at += (n * size + 15) / 16 * 16;
  return t;
}

void* stream_of(c10::Device dev) {
  return static_cast<void*>(c10::cuda::getCurrentCUDAStream(dev.index()).stream());
}

// (query_lens, context_lens, block_table, page_size, num_tokens, free_pages, free_head)
PyObject* plan(PyObject* const* a, Py_ssize_t n) {
  if (n != 7 || g_plan == nullptr || !PyLong_CheckExact(a[3]) || !PyLong_CheckExact(a[4])) {
    Py_RETURN_NONE;
  }
  const Tensor *q = cuda_tensor(a[0]), *c = cuda_tensor(a[1]), *table = cuda_tensor(a[2]);
  const int64_t page = PyLong_AsLongLong(a[3]), tokens = PyLong_AsLongLong(a[4]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  if (q == nullptr || q->dim() != 1 || page < 1 || tokens < 0) Py_RETURN_NONE;
  const c10::Device dev = q->device();
  const int64_t R = q->size(0);
  if (!is_vector(q, at::kInt, R, dev) || !is_vector(c, at::kInt, R, dev) ||
      !is_table(table, R, dev)) {
    Py_RETURN_NONE;
  }
  const bool alloc = a[5] != Py_None;
  const Tensor *free = nullptr, *head = nullptr;
  if (alloc != (a[6] != Py_None)) Py_RETURN_NONE;
  if (alloc) {
    free = cuda_tensor(a[5]);
    head = cuda_tensor(a[6]);
    if (free == nullptr || free->dim() != 1 || free->numel() == 0 ||
        !is_vector(free, at::kInt, free->size(0), dev) || !is_vector(head, at::kInt, 1, dev)) {
      Py_RETURN_NONE;
    }
  }
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor store = empty({16 * (tokens + 2) + 8 * R + 64}, at::kByte, dev);
  int64_t at = 0;
  Tensor pos = carve(store, at, tokens, at::kLong), slots = carve(store, at, tokens, at::kLong),
         start = carve(store, at, R + 1, at::kInt), seq = carve(store, at, R, at::kInt), next;
  if (alloc) next = carve(store, at, 1, at::kInt);
  const int st = g_plan(
      q->const_data_ptr<int>(), c->const_data_ptr<int>(), R, tokens,
      table->mutable_data_ptr<int>(), table->stride(0), table->size(1), page,
      alloc ? free->const_data_ptr<int>() : nullptr, alloc ? free->size(0) : 0,
      alloc ? head->const_data_ptr<int>() : nullptr, start.mutable_data_ptr<int>(),
      seq.mutable_data_ptr<int>(), pos.mutable_data_ptr<int64_t>(),
      slots.mutable_data_ptr<int64_t>(), alloc ? next.mutable_data_ptr<int>() : nullptr,
      stream_of(dev));
  if (st != BI_OK) return PyLong_FromLong(st);
  PyObject* out = PyTuple_New(5);
  if (out == nullptr) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(start)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(seq)));
  PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(std::move(pos)));
  PyTuple_SET_ITEM(out, 3, THPVariable_Wrap(std::move(slots)));
  PyTuple_SET_ITEM(out, 4, alloc ? THPVariable_Wrap(std::move(next)) : Py_NewRef(Py_None));
  return out;
}

// (qkv, cos, sin, positions, slots, k_cache, v_cache, out)
PyObject* rope(PyObject* const* a, Py_ssize_t n) {
  if (n != 8 || g_rope == nullptr) Py_RETURN_NONE;
  const Tensor *qkv = cuda_tensor(a[0]), *cs = cuda_tensor(a[1]), *sn = cuda_tensor(a[2]),
               *pos = cuda_tensor(a[3]), *slots = cuda_tensor(a[4]), *k = cuda_tensor(a[5]),
               *v = cuda_tensor(a[6]);
  if (qkv == nullptr || qkv->dim() != 2 || k == nullptr || v == nullptr) Py_RETURN_NONE;
  const c10::Device dev = qkv->device();
  const ScalarType type = qkv->scalar_type();
  const int code = dtype_code(type);
  int64_t ks[3], vs[3];
  if (code < 0 || !cache_strides(k, type, dev, ks) || !cache_strides(v, type, dev, vs) ||
      k->sizes() != v->sizes()) {
    Py_RETURN_NONE;
  }
  const int64_t T = qkv->size(0), width = qkv->size(1), hk = k->size(1), hd = k->size(3);
  const int64_t hq = width / hd - 2 * hk;
  if (hd % 2 != 0 || width % hd != 0 || hq < 0 || (width > 1 && qkv->stride(1) != 1) ||
      (T > 1 && qkv->stride(0) < width)) {
    Py_RETURN_NONE;
  }
  if (cs == nullptr || sn == nullptr || cs->dim() != 2 || cs->sizes() != sn->sizes() ||
      cs->scalar_type() != at::kFloat || sn->scalar_type() != at::kFloat ||
      !cs->is_contiguous() || !sn->is_contiguous() || cs->device() != dev ||
      sn->device() != dev || 2 * cs->size(1) > hd || !is_vector(pos, at::kLong, T, dev) ||
      !is_vector(slots, at::kLong, T, dev)) {
    Py_RETURN_NONE;
  }
  const Tensor* given = nullptr;
  if (a[7] != Py_None) {
    given = cuda_tensor(a[7]);
    if (given == nullptr || given->scalar_type() != type || given->device() != dev ||
        given->sizes() != at::IntArrayRef({T, hq, hd}) || !given->is_contiguous()) {
      Py_RETURN_NONE;
    }
  }
  const c10::cuda::CUDAGuard guard(dev);
  Tensor out = given != nullptr ? *given : empty({T, hq, hd}, type, dev);
  const int st = g_rope(
      qkv->const_data_ptr(), T > 1 ? qkv->stride(0) : width, T, hq, hk, hd, 2 * cs->size(1),
      cs->const_data_ptr<float>(), sn->const_data_ptr<float>(), cs->size(0),
      pos->const_data_ptr<int64_t>(), slots->const_data_ptr<int64_t>(), out.mutable_data_ptr(),
      k->mutable_data_ptr(), ks, v->mutable_data_ptr(), vs, k->size(0), k->size(2), code,
      stream_of(dev));
  if (st != BI_OK) return PyLong_FromLong(st);
  return given != nullptr ? Py_NewRef(a[7]) : THPVariable_Wrap(std::move(out));
}

// (q, k_cache, v_cache, block_table, query_start, seq_lens, scale, window, first_tokens, sinks,
//  out)
PyObject* attention(PyObject* const* a, Py_ssize_t n) {
  if (n != 11 || g_sdpa == nullptr || !PyLong_CheckExact(a[8])) Py_RETURN_NONE;
  const Tensor *q = cuda_tensor(a[0]), *k = cuda_tensor(a[1]), *v = cuda_tensor(a[2]),
               *table = cuda_tensor(a[3]), *start = cuda_tensor(a[4]), *seq = cuda_tensor(a[5]);
  if (q == nullptr || q->dim() != 3 || k == nullptr || v == nullptr || seq == nullptr ||
      seq->dim() != 1 || q->numel() == 0) {
    Py_RETURN_NONE;
  }
  const c10::Device dev = q->device();
  const ScalarType type = q->scalar_type();
  const int code = dtype_code(type);
  int64_t ks[3], vs[3];
  if (code < 0 || !cache_strides(k, type, dev, ks) || !cache_strides(v, type, dev, vs) ||
      k->sizes() != v->sizes()) {
    Py_RETURN_NONE;
  }
  const int64_t T = q->size(0), H = q->size(1), D = q->size(2), R = seq->size(0);
  const int64_t Hkv = k->size(1), vec = 16 / static_cast<int64_t>(q->element_size());
  const int64_t qs[2] = {T > 1 ? q->stride(0) : H * D, H > 1 ? q->stride(1) : D};
  if (R == 0 || k->size(3) != D || H % Hkv != 0 || D % 32 != 0 || D > 256 || q->stride(2) != 1 ||
      qs[0] <= 0 || qs[1] <= 0 || qs[0] % vec != 0 || qs[1] % vec != 0 ||
      !aligned16(q->const_data_ptr()) || !is_vector(seq, at::kInt, R, dev) ||
      !is_vector(start, at::kInt, R + 1, dev) || !is_table(table, R, dev) ||
      table->size(1) == 0) {
    Py_RETURN_NONE;
  }
  double scale;
  if (a[6] == Py_None) {
    scale = 1.0 / std::sqrt(static_cast<double>(D));
  } else if (PyFloat_CheckExact(a[6])) {
    scale = PyFloat_AS_DOUBLE(a[6]);
    if (!(scale >= 0.0 && scale < 3.0e38)) Py_RETURN_NONE;
  } else {
    Py_RETURN_NONE;
  }
  int64_t window = 0;
  if (a[7] != Py_None) {
    if (!PyLong_CheckExact(a[7])) Py_RETURN_NONE;
    window = PyLong_AsLongLong(a[7]);
  }
  const int64_t first = PyLong_AsLongLong(a[8]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  if (window < 0 || first < 0 || (first > 0 && window == 0)) Py_RETURN_NONE;
  const Tensor* sinks = nullptr;
  if (a[9] != Py_None) {
    sinks = cuda_tensor(a[9]);
    if (!is_vector(sinks, type, H, dev)) Py_RETURN_NONE;
  }
  const Tensor* given = nullptr;
  if (a[10] != Py_None) {
    given = cuda_tensor(a[10]);
    if (given == nullptr || given->scalar_type() != type || given->device() != dev ||
        given->sizes() != q->sizes() || given->stride(2) != 1 ||
        given->stride(0) % vec != 0 || given->stride(1) % vec != 0 ||
        (T > 1 && given->stride(0) == 0) || (H > 1 && given->stride(1) == 0) ||
        !aligned16(given->const_data_ptr())) {
      Py_RETURN_NONE;
    }
  }
  const c10::cuda::CUDAGuard guard(dev);
  Tensor out = given != nullptr ? *given : empty({T, H, D}, type, dev);
  const int64_t os[2] = {out.stride(0), out.stride(1)};
  const int64_t bytes = g_workspace(T, R, H, D, table->size(1), k->size(2));
  const Tensor ws = empty({bytes}, at::kByte, dev);
  const int st = g_sdpa(
      q->const_data_ptr(), qs, k->const_data_ptr(), ks, v->const_data_ptr(), vs, k->size(0),
      k->size(2), table->const_data_ptr<int>(), table->stride(0), table->size(1),
      start->const_data_ptr<int>(), seq->const_data_ptr<int>(),
      sinks != nullptr ? sinks->const_data_ptr() : nullptr, static_cast<float>(scale), window,
      first, T, R, H, Hkv, D, code, out.mutable_data_ptr(), os, ws.mutable_data_ptr(), bytes,
      stream_of(dev));
  if (st != BI_OK) return PyLong_FromLong(st);
  return given != nullptr ? Py_NewRef(a[10]) : THPVariable_Wrap(std::move(out));
}

// Addresses of libbi.so's functions, in the order of the pointers above.
PyObject* init(PyObject* const* a, Py_ssize_t n) {
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "init takes the four entry points' addresses");
    return nullptr;
  }
  void* p[4];
  for (int i = 0; i < 4; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (p[i] == nullptr) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "null");
  }
  g_plan = reinterpret_cast<decltype(g_plan)>(p[0]);
  g_rope = reinterpret_cast<decltype(g_rope)>(p[1]);
  g_sdpa = reinterpret_cast<decltype(g_sdpa)>(p[2]);
  g_workspace = reinterpret_cast<decltype(g_workspace)>(p[3]);
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(&guarded<f>)), \
                METH_FASTCALL
PyMethodDef g_methods[] = {{"init", FAST(init), nullptr},
                           {"plan", FAST(plan), nullptr},
                           {"rope", FAST(rope), nullptr},
                           {"attention", FAST(attention), nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_bind",
                        "Short way to libbi.so's paged-cache operators", -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__bind(void) {
  PyObject* m = PyModule_Create(&g_module);
  // the torch whose headers this was compiled with; with another one it is not used
  if (m != nullptr && PyModule_AddStringConstant(m, "torch_version", BI_TORCH_VERSION) != 0) {
    Py_CLEAR(m);
  }
  return m;
}
