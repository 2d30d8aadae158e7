// torch_ops.cpp — the operators of ops.py that a program calls once per layer and token, from Python to the C ABI without Python in between.
//
// What the path costs: checks, an empty result, the stream and a ctypes call with a dozen converted arguments took 4.7 of the 8.8 µs of a
// small Linear.  Host µs a call, from Python / from here: a Linear of one row 8.8 / 4.9, an attention row over 20 keys 8.2 / 4.3, a fused GEMV
// 8.6 / 5.1, a norm or a sum 6.2 / 3.9; what is left is the result's allocation and the launch.
//
// A function takes what its ops.py namesake was given.  It answers None for everything but the plain case — a tensor that is no ordinary strided
// CUDA tensor of the type the operator takes, or not contiguous; a shape that ops.py refuses; an active torch-function mode — and
// ops.py then goes its own way, which copies, converts or raises; a status other than 0 comes back as a number.  Everything else is the same
// call of the C ABI: the result comes from torch's caching allocator (captured graphs, dispatch modes and the deterministic fill see
// it), the launch goes to the current stream of the current device, and the GIL is free meanwhile.
#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/TensorSubclassLikeUtils.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <dlfcn.h>

#include "b200_decode.h"

namespace {

// The C ABI of the library that _lib.py has loaded, whatever its file is called: this module is linked to none.
#define B200_FUNCTIONS(F) \
  F(gemv_bf16) F(gemm_bf16) F(rmsnorm_bf16) F(silu_mul_bf16) F(add_bf16) F(attn_bf16) F(gemv_fused_bf16) F(attn_decode_workspace_bytes) F(attn_decode_bf16) F(w4_workspace_bytes) F(w4_linear_bf16) \
  F(kv4_store) F(kv4_load) F(kv4_attention_workspace_bytes) F(kv4_attention) F(kv4_extend) F(kv4_fork) F(kv4_free) F(kv4_compact) F(kv4_workspace_bytes)
struct {
#define B200_FIELD(f) decltype(&b200_##f) f;
  B200_FUNCTIONS(B200_FIELD)
} abi;

PyObject* bind(PyObject*, PyObject* handle) {   // what dlopen gave; before any other function here
  void* const lib = PyLong_AsVoidPtr(handle);
  if (lib == nullptr) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "no library");
#define B200_BIND(f)                                                             \
  abi.f = reinterpret_cast<decltype(abi.f)>(dlsym(lib, "b200_" #f));             \
  if (abi.f == nullptr) return PyErr_Format(PyExc_AttributeError, "the library does not export b200_" #f);
  B200_FUNCTIONS(B200_BIND)
  Py_RETURN_NONE;
}

// an ordinary contiguous CUDA tensor of this type, or null
const at::Tensor* plain(PyObject* o, at::ScalarType type = at::kBFloat16, bool contiguous = true) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || t.layout() != at::kStrided || !t.is_cuda() || t.scalar_type() != type || !t.unsafeGetTensorImpl()->has_storage() ||
      at::isTensorSubclassLike(t) || t.key_set().has(c10::DispatchKey::Functionalize) || t._is_zerotensor() || (contiguous && !t.is_contiguous()) || t.is_neg() ||
      t.is_conj())
    return nullptr;
  return &t;
}
// the same, or None
bool plain_or_none(PyObject* o, const at::Tensor*& t, at::ScalarType type = at::kBFloat16) {
  t = nullptr;
  return o == Py_None || (t = plain(o, type)) != nullptr;
}
bool modes() { return at::impl::torch_function_mode_enabled(); }
void* ptr(const at::Tensor* t) { return t == nullptr ? nullptr : t->data_ptr(); }

// A result of shape `sizes` on x's device, handed to `call` with the current stream: the tensor, or the status that is not 0.
template <typename F>
PyObject* run(const at::Tensor& x, at::IntArrayRef sizes, F call) {
  at::Tensor y;
  int rc;
  {
    pybind11::gil_scoped_release free;
    y = at::empty(sizes, at::TensorOptions().dtype(at::kBFloat16).device(x.device()));
    rc = call(y.data_ptr(), (void*)c10::cuda::getCurrentCUDAStream().stream());
  }
  return rc == 0 ? THPVariable_Wrap(y) : PyLong_FromLong(rc);
}

// Device memory of torch's caching allocator for a call, on the current stream of the current device; a tensor around it would cost 0.7 µs more
at::DataPtr scratch(int64_t bytes) { return c10::cuda::CUDACachingAllocator::get()->allocate((size_t)bytes); }
// whether a tensor lies on the current device: what runs there runs on its current stream
bool here(const at::Tensor& t) { return t.device().index() == c10::cuda::current_device(); }
// whether a weight's parts have the sizes of its layout
bool w4_fits(const at::Tensor& q, const at::Tensor& scale, const at::Tensor* zero, int64_t n, int64_t k, int64_t group) {
  const int64_t tiles = (n + 15) / 16, small = tiles * 16 * ((k + group - 1) / group);
  return q.numel() == tiles * ((k + 63) / 64) * 512 && scale.numel() == small && (zero == nullptr || zero->numel() == small);
}

// x's sizes with another last one
c10::SmallVector<int64_t, 6> with_last(const at::Tensor& x, int64_t n) {
  c10::SmallVector<int64_t, 6> s(x.sizes().begin(), x.sizes().end());
  s.back() = n;
  return s;
}

PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n_args) {   // x, weight, bias or None
  HANDLE_TH_ERRORS
  const at::Tensor *x, *w, *b;
  if (n_args != 3 || modes() || !(x = plain(a[0])) || !(w = plain(a[1])) || !plain_or_none(a[2], b) || w->dim() != 2 || x->dim() < 1) Py_RETURN_NONE;
  const int64_t n = w->size(0), k = w->size(1);
  if (k < 1 || x->size(-1) != k || x->numel() < 1) Py_RETURN_NONE;
  const int64_t m = x->numel() / k;
  return run(*x, with_last(*x, n), [&](void* y, void* st) { return abi.gemv_bf16(y, x->data_ptr(), w->data_ptr(), ptr(b), m, n, k, st); });
  END_HANDLE_TH_ERRORS
}

PyObject* gemm(PyObject*, PyObject* const* a, Py_ssize_t n_args) {   // a, weight
  HANDLE_TH_ERRORS
  const at::Tensor *x, *w;
  if (n_args != 2 || modes() || !(x = plain(a[0])) || !(w = plain(a[1])) || w->dim() != 2 || x->dim() < 1) Py_RETURN_NONE;
  const int64_t n = w->size(0), k = w->size(1);
  if (k < 1 || x->size(-1) != k || x->numel() < 1) Py_RETURN_NONE;
  const int64_t m = x->numel() / k;
  return run(*x, with_last(*x, n), [&](void* y, void* st) { return abi.gemm_bf16(y, x->data_ptr(), w->data_ptr(), m, n, k, st); });
  END_HANDLE_TH_ERRORS
}

PyObject* rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n_args) {   // x, weight or None, eps
  HANDLE_TH_ERRORS
  const at::Tensor *x, *w;
  if (n_args != 3 || modes() || !(x = plain(a[0])) || !plain_or_none(a[1], w) || !PyFloat_Check(a[2]) || x->dim() < 1 || x->numel() < 1) Py_RETURN_NONE;
  const int64_t dim = x->size(-1);
  const float eps = (float)PyFloat_AS_DOUBLE(a[2]);
  return run(*x, x->sizes(), [&](void* y, void* st) { return abi.rmsnorm_bf16(y, x->data_ptr(), ptr(w), x->numel() / dim, dim, eps, st); });
  END_HANDLE_TH_ERRORS
}

PyObject* silu_mul(PyObject*, PyObject* const* a, Py_ssize_t n_args) {   // x
  HANDLE_TH_ERRORS
  const at::Tensor* x;
  if (n_args != 1 || modes() || !(x = plain(a[0])) || x->dim() < 1 || x->numel() < 1 || x->size(-1) % 2 != 0) Py_RETURN_NONE;
  const int64_t n = x->size(-1) / 2;
  return run(*x, with_last(*x, n), [&](void* y, void* st) { return abi.silu_mul_bf16(y, x->data_ptr(), x->numel() / (2 * n), n, st); });
  END_HANDLE_TH_ERRORS
}

PyObject* add(PyObject*, PyObject* const* a, Py_ssize_t n_args) {   // a, b of one shape
  HANDLE_TH_ERRORS
  const at::Tensor *x, *z;
  if (n_args != 2 || modes() || !(x = plain(a[0])) || !(z = plain(a[1])) || x->sizes() != z->sizes()) Py_RETURN_NONE;
  return run(*x, x->sizes(), [&](void* y, void* st) { return abi.add_bf16(y, x->data_ptr(), z->data_ptr(), x->numel(), st); });
  END_HANDLE_TH_ERRORS
}

PyObject* flash_attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {   // q, k, v, causal
  HANDLE_TH_ERRORS
  const at::Tensor *q, *k, *v;
  if (n_args != 4 || modes() || !(q = plain(a[0])) || !(k = plain(a[1])) || !(v = plain(a[2])) || !PyBool_Check(a[3]) || q->dim() != 4 || k->dim() < 3)
    Py_RETURN_NONE;
  const int64_t B = q->size(0), Sq = q->size(1), Hq = q->size(2), D = q->size(3), Skv = k->size(1), Hkv = k->size(2);
  const int causal = a[3] == Py_True;
  return run(*q, q->sizes(), [&](void* y, void* st) {
    return abi.attn_bf16(y, q->data_ptr(), k->data_ptr(), v->data_ptr(), B, Sq, Skv, Hq, Hkv, D, causal, st);
  });
  END_HANDLE_TH_ERRORS
}

PyObject* gemv_fused(PyObject*, PyObject* const* a, Py_ssize_t n_args) {   // x, weight, norm or None, eps, bias or None, residual or None, silu
  HANDLE_TH_ERRORS
  const at::Tensor *x, *w, *norm, *b, *r;
  if (n_args != 7 || modes() || !(x = plain(a[0])) || !(w = plain(a[1])) || !plain_or_none(a[2], norm) || !PyFloat_Check(a[3]) ||
      !plain_or_none(a[4], b) || !plain_or_none(a[5], r) || !PyBool_Check(a[6]) || w->dim() != 2)
    Py_RETURN_NONE;
  const int silu = a[6] == Py_True, nseg = silu ? 2 : 1;
  const int64_t n = w->size(0) / nseg, k = w->size(1);
  const float eps = (float)PyFloat_AS_DOUBLE(a[3]);
  return run(*x, {n}, [&](void* y, void* st) {
    return abi.gemv_fused_bf16(y, x->data_ptr(), w->data_ptr(), n, k, nseg, ptr(norm), eps, ptr(b), ptr(r), silu, st);
  });
  END_HANDLE_TH_ERRORS
}

// qkv, kcache, vcache, q_heads, kv_heads, head_dim, pos or None, fixed_len, rope table or None, q_norm or None, k_norm or None, eps
PyObject* attn_decode(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  const at::Tensor *qkv, *kc, *vc, *pos, *rope, *qn, *kn;
  if (n_args != 12 || modes() || !(qkv = plain(a[0])) || !(kc = plain(a[1])) || !(vc = plain(a[2])) || !PyLong_Check(a[3]) || !PyLong_Check(a[4]) ||
      !PyLong_Check(a[5]) || !plain_or_none(a[6], pos, at::kInt) || !PyLong_Check(a[7]) || !plain_or_none(a[8], rope, at::kFloat) ||
      !plain_or_none(a[9], qn) || !plain_or_none(a[10], kn) || !PyFloat_Check(a[11]) || kc->dim() < 1)
    Py_RETURN_NONE;
  const int64_t Hq = PyLong_AsLongLong(a[3]), Hkv = PyLong_AsLongLong(a[4]), hd = PyLong_AsLongLong(a[5]), len = PyLong_AsLongLong(a[7]);
  if (PyErr_Occurred()) {   // a number that no int64 holds
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  const int64_t ctx = kc->size(0);
  if (Hq < 1 || Hq > (1 << 20) || hd < 1 || hd > 1024) Py_RETURN_NONE;
  if (abi.attn_decode_workspace_bytes(Hq, Hkv, hd, ctx) < 0) Py_RETURN_NONE;
  const float eps = (float)PyFloat_AS_DOUBLE(a[11]);
  return run(*qkv, {Hq * hd}, [&](void* y, void* st) {
    // no workspace is taken: any address will do
    return abi.attn_decode_bf16(y, qkv->data_ptr(), ptr(qn), ptr(kn), eps, (const float*)ptr(rope), (const int32_t*)ptr(pos), len, kc->data_ptr(),
                                vc->data_ptr(), Hq, Hkv, hd, ctx, y, st);
  });
  END_HANDLE_TH_ERRORS
}

int64_t whole_number(PyObject* o) {   // −1, which nothing here takes, for one that no int64 holds
  const int64_t v = PyLong_AsLongLong(o);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return -1;
  }
  return v;
}

PyObject* linear_w4(PyObject*, PyObject* const* a, Py_ssize_t n_args) {   // x, q, scale, zero or None, n, k, group, bias or None
  HANDLE_TH_ERRORS
  const at::Tensor *x, *q, *scale, *zero, *b;
  if (n_args != 8 || modes() || !(x = plain(a[0])) || !(q = plain(a[1], at::kByte)) || !(scale = plain(a[2])) || !plain_or_none(a[3], zero) ||
      !PyLong_Check(a[4]) || !PyLong_Check(a[5]) || !PyLong_Check(a[6]) || !plain_or_none(a[7], b) || x->dim() < 1)
    Py_RETURN_NONE;
  const int64_t n = whole_number(a[4]), k = whole_number(a[5]), group = whole_number(a[6]);
  if (n < 1 || k < 1 || (group != 32 && group != 64 && group != 128) || n > 16 * 65535 || k > 1 << 24 || x->size(-1) != k || x->numel() < 1 || !w4_fits(*q, *scale, zero, n, k, group) ||
      (b != nullptr && b->numel() != n))
    Py_RETURN_NONE;
  if (!here(*x) || q->device() != x->device() || scale->device() != x->device() || (zero && zero->device() != x->device()) || (b && b->device() != x->device()))
    Py_RETURN_NONE;
  const b200_w4_weight w{q->data_ptr(), scale->data_ptr(), ptr(zero), (int32_t)n, (int32_t)k, (int32_t)group};
  const int64_t m = x->numel() / k, bytes = abi.w4_workspace_bytes(m, n, k);
  return run(*x, with_last(*x, n), [&](void* y, void* st) {
    at::DataPtr ws;
    if (bytes > 0) ws = scratch(bytes);
    return abi.w4_linear_bf16(y, x->data_ptr(), &w, ptr(b), m, ws.get(), st);
  });
  END_HANDLE_TH_ERRORS
}

// ---- the paged cache of 4 bits.  A call starts with the cache's descriptor (its address, as KV4Cache keeps it) and its device.
struct Kv4 {
  const b200_kv4_cache* c;
  int64_t device;
  bool take(PyObject* const* a) {
    if (modes() || !PyLong_Check(a[0]) || !PyLong_Check(a[1])) return false;
    c = static_cast<const b200_kv4_cache*>(PyLong_AsVoidPtr(a[0]));
    device = PyLong_AsLongLong(a[1]);
    return c != nullptr && device == c10::cuda::current_device();
  }
  bool with(const at::Tensor& t) const { return t.device().index() == device; }
  at::TensorOptions options(at::ScalarType type) const { return at::TensorOptions().dtype(type).device(at::kCUDA, (int8_t)device); }
};
// n whole numbers beside the cache
const at::Tensor* numbers(const Kv4& kv, PyObject* o, int64_t n = -1) {
  const at::Tensor* t = plain(o, at::kInt);
  return t != nullptr && t->dim() == 1 && kv.with(*t) && (n < 0 || t->size(0) == n) ? t : nullptr;
}
// rows [any number, heads, dim] whose heads lie side by side
const at::Tensor* head_rows(const Kv4& kv, PyObject* o) {
  const at::Tensor* t = plain(o, at::kBFloat16, false);
  return t != nullptr && t->dim() == 3 && kv.with(*t) && t->size(0) > 0 && t->size(2) == kv.c->dim && t->stride(2) == 1 && t->stride(1) == t->size(2) &&
                 (t->size(0) == 1 || (t->stride(0) >= t->size(1) * t->size(2) && t->stride(0) % 8 == 0)) &&
                 reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0
             ? t : nullptr;
}
int64_t row_stride(const at::Tensor& t) { return t.size(0) == 1 ? t.size(1) * t.size(2) : t.stride(0); }
struct Kv4Where {
  const at::Tensor *seqs, *starts, *pos;
  int64_t n;
  bool take(const Kv4& kv, PyObject* const* a) {
    if (!(seqs = numbers(kv, a[0]))) return false;
    n = seqs->size(0);   // (a call without sequences launches nothing: ops.py's)
    return n > 0 && (starts = numbers(kv, a[1], n + 1)) && (pos = numbers(kv, a[2], n));
  }
  static const int32_t* at(const at::Tensor* t) { return static_cast<const int32_t*>(t->data_ptr()); }
};
template <typename F>
PyObject* status(F call) {   // of a call without a result: None was not for it, so True or the status
  int rc;
  {
    pybind11::gil_scoped_release free;
    rc = call((void*)c10::cuda::getCurrentCUDAStream().stream());
  }
  if (rc == 0) Py_RETURN_TRUE;
  return PyLong_FromLong(rc);
}

PyObject* kv4_store(PyObject*, PyObject* const* a, Py_ssize_t n_args) {   // cache, device, layer, k, v, seqs, starts, pos
  HANDLE_TH_ERRORS
  Kv4 kv;
  Kv4Where w;
  const at::Tensor *k, *v;
  if (n_args != 8 || !kv.take(a) || !PyLong_Check(a[2]) || !(k = head_rows(kv, a[3])) || !(v = head_rows(kv, a[4])) || !w.take(kv, a + 5) ||
      k->sizes() != v->sizes() || k->size(1) != kv.c->kv_heads)
    Py_RETURN_NONE;
  const int64_t layer = whole_number(a[2]);
  return status([&](void* st) {
    return abi.kv4_store(kv.c, layer, k->data_ptr(), row_stride(*k), v->data_ptr(), row_stride(*v), w.at(w.seqs), w.at(w.starts), w.at(w.pos), w.n, k->size(0), st);
  });
  END_HANDLE_TH_ERRORS
}

PyObject* kv4_load(PyObject*, PyObject* const* a, Py_ssize_t n_args) {   // cache, device, layer, seqs, starts, pos, rows
  HANDLE_TH_ERRORS
  Kv4 kv;
  Kv4Where w;
  if (n_args != 7 || !kv.take(a) || !PyLong_Check(a[2]) || !w.take(kv, a + 3) || !PyLong_Check(a[6])) Py_RETURN_NONE;
  const int64_t layer = whole_number(a[2]), rows = whole_number(a[6]);
  if (rows < 1 || rows > 1 << 24) Py_RETURN_NONE;
  at::Tensor k, v;
  int rc;
  {
    pybind11::gil_scoped_release free;
    k = at::empty({rows, kv.c->kv_heads, kv.c->dim}, kv.options(at::kFloat));
    v = at::empty_like(k);
    rc = abi.kv4_load(static_cast<float*>(k.data_ptr()), static_cast<float*>(v.data_ptr()), kv.c, layer, w.at(w.seqs), w.at(w.starts), w.at(w.pos), w.n, rows,
                      (void*)c10::cuda::getCurrentCUDAStream().stream());
  }
  if (rc != 0) return PyLong_FromLong(rc);
  PyObject *pk = THPVariable_Wrap(k), *pv = THPVariable_Wrap(v);
  PyObject* both = pk && pv ? PyTuple_Pack(2, pk, pv) : nullptr;
  Py_XDECREF(pk);
  Py_XDECREF(pv);
  return both;
  END_HANDLE_TH_ERRORS
}

PyObject* kv4_attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {   // cache, device, layer, q, seqs, starts, pos, scale, window
  HANDLE_TH_ERRORS
  Kv4 kv;
  Kv4Where w;
  const at::Tensor* q;
  if (n_args != 9 || !kv.take(a) || !PyLong_Check(a[2]) || !(q = head_rows(kv, a[3])) || !w.take(kv, a + 4) || !PyFloat_Check(a[7]) || !PyLong_Check(a[8]))
    Py_RETURN_NONE;
  const int64_t layer = whole_number(a[2]), window = whole_number(a[8]), heads = q->size(1), rows = q->size(0);
  const float scale = (float)PyFloat_AS_DOUBLE(a[7]);
  const int64_t bytes = abi.kv4_attention_workspace_bytes(kv.c, heads, w.n, rows);
  if (bytes < 0) Py_RETURN_NONE;
  return run(*q, q->sizes(), [&](void* y, void* st) {
    const at::DataPtr ws = scratch(bytes);
    return abi.kv4_attention(y, q->data_ptr(), row_stride(*q), kv.c, layer, heads, w.at(w.seqs), w.at(w.starts), w.at(w.pos), w.n, rows, scale, window, ws.get(),
                             st);
  });
  END_HANDLE_TH_ERRORS
}

// Bookkeeping: `first` and `second` lists of n numbers → n numbers
template <typename F>
PyObject* kv4_lists(PyObject* const* a, Py_ssize_t n_args, F call) {   // cache, device, first, second
  Kv4 kv;
  const at::Tensor *x, *y;
  if (n_args != 4 || !kv.take(a) || !(x = numbers(kv, a[2])) || !(y = numbers(kv, a[3], x->size(0))) || x->size(0) < 1) Py_RETURN_NONE;
  at::Tensor out;
  int rc;
  {
    pybind11::gil_scoped_release free;
    out = at::empty({x->size(0)}, kv.options(at::kInt));
    const at::DataPtr ws = scratch(abi.kv4_workspace_bytes(kv.c));
    rc = call(kv.c, Kv4Where::at(x), Kv4Where::at(y), static_cast<int32_t*>(out.data_ptr()), x->size(0), ws.get(),
              (void*)c10::cuda::getCurrentCUDAStream().stream());
  }
  return rc == 0 ? THPVariable_Wrap(out) : PyLong_FromLong(rc);
}
PyObject* kv4_extend(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  return kv4_lists(a, n_args, abi.kv4_extend);
  END_HANDLE_TH_ERRORS
}
PyObject* kv4_fork(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  return kv4_lists(a, n_args, abi.kv4_fork);
  END_HANDLE_TH_ERRORS
}
PyObject* kv4_free(PyObject*, PyObject* const* a, Py_ssize_t n_args) {   // cache, device, seqs
  HANDLE_TH_ERRORS
  Kv4 kv;
  const at::Tensor* s;
  if (n_args != 3 || !kv.take(a) || !(s = numbers(kv, a[2])) || s->size(0) < 1) Py_RETURN_NONE;
  return status([&](void* st) { return abi.kv4_free(kv.c, Kv4Where::at(s), s->size(0), st); });
  END_HANDLE_TH_ERRORS
}
PyObject* kv4_compact(PyObject*, PyObject* const* a, Py_ssize_t n_args) {   // cache, device
  HANDLE_TH_ERRORS
  Kv4 kv;
  if (n_args != 2 || !kv.take(a)) Py_RETURN_NONE;
  at::Tensor out;
  int rc;
  {
    pybind11::gil_scoped_release free;
    out = at::empty({1}, kv.options(at::kInt));
    const at::DataPtr ws = scratch(abi.kv4_workspace_bytes(kv.c));
    rc = abi.kv4_compact(kv.c, static_cast<int32_t*>(out.data_ptr()), ws.get(), (void*)c10::cuda::getCurrentCUDAStream().stream());
  }
  return rc == 0 ? THPVariable_Wrap(out) : PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

#define B200_OP(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"_bind", bind, METH_O, nullptr}, B200_OP(linear),     B200_OP(gemm),        B200_OP(rms_norm),
                         B200_OP(silu_mul),                B200_OP(add),        B200_OP(flash_attention),
                         B200_OP(gemv_fused),              B200_OP(attn_decode), B200_OP(linear_w4),
                         B200_OP(kv4_store), B200_OP(kv4_load), B200_OP(kv4_attention), B200_OP(kv4_extend), B200_OP(kv4_fork), B200_OP(kv4_free),
                         B200_OP(kv4_compact), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "b200ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_b200ops() { return PyModule_Create(&module); }
