// binding.cpp -- the small calls' launch paths from torch tensors, for CPython.
//
// scatter(src, kv, slots, block_size, hnd, shift, k_scale, error_flags) is
// shift_kernels.scatter_shifted's usual call: it reads the tensors through torch's C++
// interface, checks what that function checks and calls mkv_scatter_shifted on the current
// stream.  Through Python methods and ctypes the same call spent 3.6 us of its 6.7 around
// the launch, longer than the kernel of a short span runs (2.4 us for 300 tokens), so a loop
// over layers was bound by it: 28 calls of 301 fp16 tokens 165 -> 79 to 108 us, a process
// settling at one figure or another between these (2.8 to 3.8 us a call).
//
// Returns the library's status, or None wherever the call is not the usual one (tensors
// that need a copy or a conversion, subclasses and wrapped tensors, another current device,
// anything the general path refuses): nothing has been launched then, and the caller takes
// the general path, which also raises the errors.
//
// slots, store and attend are scaled_cache.py's step_slots, store_scaled and attend_scaled in
// the same way: a decode step's kernels run 4 to 20 us, and through Python methods and ctypes
// the calls took 10 to 15 on the host.  They return their tensors (store: None on success
// becomes True), the library's status as an int, or None for the general path.  rotate, put and
// attend_shared are scaled_step.py's calls in the same way: 20 us on the host became 4 to 6 (into a
// caller's outputs, in place among them, 27 to 39).

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cmath>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "marathon_kvscaled.h"
#include "marathon_kvshift.h"
#include "marathon_kvstep.h"

namespace {

typedef decltype(&mkv_scatter_shifted) scatter_fn;
scatter_fn g_scatter = nullptr;

PyObject* s_delta;
PyObject* s_cos;
PyObject* s_sgn;
PyObject* s_emb_cos;
PyObject* s_rotary;

struct Ref {  // one owned reference
  PyObject* p;
  explicit Ref(PyObject* o) : p(o) {}
  ~Ref() { Py_XDECREF(p); }
  Ref(const Ref&) = delete;
  Ref& operator=(const Ref&) = delete;
};

// The plain tensor behind `o` (no subclass, nothing that wraps another tensor), or null.
const at::Tensor* plain(PyObject* o) {
  if (o == nullptr || !THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.layout() == at::kStrided && t.has_storage() ? &t : nullptr;
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16:
      return MKV_BF16;
    case at::kHalf:
      return MKV_F16;
    case at::kFloat:
      return MKV_F32;
    case at::kFloat8_e4m3fn:
      return MKV_FP8_E4M3;
    default:
      return -1;
  }
}

enum { kUsual, kOther, kError };

struct Shift {
  int64_t rotary = 0;
  const float* cos = nullptr;
  const float* sgn = nullptr;
};

// A RopeShift's tables; kOther unless they are plain tensors on `dev` that fit.
int read_shift(PyObject* shift, const at::Device& dev, int64_t head_size, Shift& out) {
  const Ref emb(PyObject_GetAttr(shift, s_emb_cos));
  const Ref delta(emb.p != nullptr ? PyObject_GetAttr(shift, s_delta) : nullptr);
  if (delta.p == nullptr) return kError;
  const at::Tensor* e = plain(emb.p);
  if (e == nullptr || !PyLong_CheckExact(delta.p)) return kOther;
  const Ref declared(PyObject_GetAttr(shift, s_rotary));
  if (declared.p == nullptr) {  // the reference's RopeShift has no such field
    if (!PyErr_ExceptionMatches(PyExc_AttributeError)) return kError;
    PyErr_Clear();
  } else if (declared.p != Py_None) {
    if (!PyLong_CheckExact(declared.p)) return kOther;
    int over = 0;
    if (PyLong_AsLongLongAndOverflow(declared.p, &over) != e->numel() || over != 0) return kOther;
  }
  const int moved = PyObject_IsTrue(delta.p);
  if (moved == 0 || e->numel() == 0) return kUsual;  // a plain scatter
  const Ref cos_o(PyObject_GetAttr(shift, s_cos));
  const Ref sgn_o(cos_o.p != nullptr ? PyObject_GetAttr(shift, s_sgn) : nullptr);
  if (sgn_o.p == nullptr) return kError;
  const at::Tensor* cos = plain(cos_o.p);
  const at::Tensor* sgn = plain(sgn_o.p);
  if (cos == nullptr || sgn == nullptr || cos->device() != dev || sgn->device() != dev ||
      cos->numel() != head_size || sgn->numel() != head_size || e->numel() > INT32_MAX)
    return kOther;
  out.rotary = e->numel();
  out.cos = static_cast<const float*>(cos->data_ptr());
  out.sgn = static_cast<const float*>(sgn->data_ptr());
  return kUsual;
}

PyObject* scatter(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 8 || g_scatter == nullptr) {
    PyErr_SetString(PyExc_TypeError, "scatter takes 8 arguments, after bind()");
    return nullptr;
  }
  try {
    if (at::impl::PythonTorchFunctionTLS::stack_len() != 0) Py_RETURN_NONE;
    const at::Tensor* src = plain(args[0]);
    const at::Tensor* kv = plain(args[1]);
    const at::Tensor* slots = plain(args[2]);
    if (src == nullptr || kv == nullptr || slots == nullptr || !kv->is_cuda() ||
        src->dim() != 3 || kv->dim() != 4)
      Py_RETURN_NONE;
    const at::Device dev = kv->device();
    const int64_t n = src->size(0), two_d = src->size(2);
    const int code = dtype_code(kv->scalar_type());
    if (n == 0 || two_d % 2 != 0 || kv->size(3) != two_d || code < 0 ||
        src->scalar_type() != kv->scalar_type() || src->device() != dev ||
        slots->device() != dev || src->stride(2) != 1 || kv->stride(3) != 1 ||
        slots->scalar_type() != at::kLong || !slots->is_contiguous() || slots->numel() != n ||
        src->size(1) > INT32_MAX || two_d > INT32_MAX)
      Py_RETURN_NONE;
    if (!PyLong_CheckExact(args[3])) Py_RETURN_NONE;
    int over = 0;
    const long long block_size = PyLong_AsLongLongAndOverflow(args[3], &over);
    if (over != 0 || block_size > INT32_MAX || block_size < INT32_MIN) Py_RETURN_NONE;
    const int hnd = PyObject_IsTrue(args[4]);
    if (hnd < 0) return nullptr;
    Shift sh;
    if (args[5] != Py_None) {
      const int got = read_shift(args[5], dev, two_d / 2, sh);
      if (got == kError) return nullptr;
      if (got == kOther) Py_RETURN_NONE;
    }
    const float* scale = nullptr;
    if (sh.rotary > 0 && code == MKV_FP8_E4M3) {
      const at::Tensor* k = plain(args[6]);
      if (k == nullptr || k->device() != dev || k->scalar_type() != at::kFloat || k->numel() < 1)
        Py_RETURN_NONE;
      scale = static_cast<const float*>(k->data_ptr());
    }
    int32_t* flags = nullptr;
    if (args[7] != Py_None) {
      const at::Tensor* f = plain(args[7]);
      if (f == nullptr) Py_RETURN_NONE;
      flags = static_cast<int32_t*>(f->data_ptr());
    }
    if (c10::hip::current_device() != dev.index()) Py_RETURN_NONE;
    void* stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
    const int head_dim = hnd ? 1 : 2, off_dim = hnd ? 2 : 1;
    const void* src_p = src->data_ptr();
    void* kv_p = kv->data_ptr();
    const int64_t* slots_p = static_cast<const int64_t*>(slots->data_ptr());
    const int64_t st = src->stride(0), sh_ = src->stride(1), kb = kv->stride(0),
                  kh = kv->stride(head_dim), ko = kv->stride(off_dim), blocks = kv->size(0);
    const int32_t heads = static_cast<int32_t>(src->size(1));
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_scatter(src_p, st, sh_, kv_p, kb, kh, ko, blocks, slots_p, n, heads,
                   static_cast<int32_t>(two_d / 2), static_cast<int32_t>(block_size), code,
                   sh.cos, sh.sgn, static_cast<int32_t>(sh.rotary), scale, flags, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// ------------------------------------------------------- the block-scaled cache's calls

typedef decltype(&mkv_step_slots) slots_fn;
typedef decltype(&mkv_store_scaled) store_fn;
typedef decltype(&mkv_attend_scaled) attend_fn;
typedef decltype(&mkv_attend_workspace_size) attend_size_fn;
slots_fn g_slots = nullptr;
store_fn g_store = nullptr;
attend_fn g_attend = nullptr;
attend_size_fn g_attend_size = nullptr;

// A contiguous int32 vector on `dev` (of n entries, unless n < 0), or null.
const int32_t* vector_of(PyObject* o, const at::Device& dev, int64_t n) {
  const at::Tensor* t = plain(o);
  if (t == nullptr || t->device() != dev || t->scalar_type() != at::kInt || t->dim() != 1 ||
      !t->is_contiguous() || (n >= 0 && t->size(0) != n))
    return nullptr;
  // (an empty vector has no address; any other will do)
  return t->numel() > 0 ? static_cast<const int32_t*>(t->data_ptr()) : reinterpret_cast<int32_t*>(64);
}

struct Table {
  int32_t* at = nullptr;
  int64_t stride = 0, n = 0, width = 0;
};

bool table_of(PyObject* o, const at::Device* dev, Table& out) {
  const at::Tensor* t = plain(o);
  if (t == nullptr || !t->is_cuda() || (dev != nullptr && t->device() != *dev) ||
      t->scalar_type() != at::kInt || t->dim() != 2 || (t->size(1) > 1 && t->stride(1) != 1) ||
      t->size(0) > MKV_MAX_REQUESTS || t->size(1) > INT32_MAX)
    return false;
  out.at = static_cast<int32_t*>(t->data_ptr());
  out.n = t->size(0);
  out.width = t->size(1);
  out.stride = out.n > 1 ? t->stride(0) : out.width;
  return true;
}

// error_flags: kUsual with null for None; kOther for anything but an int32 tensor on `dev`.
int flags_of(PyObject* o, const at::Device& dev, int32_t*& out) {
  out = nullptr;
  if (o == Py_None) return kUsual;
  const at::Tensor* t = plain(o);
  if (t == nullptr || t->device() != dev || t->scalar_type() != at::kInt || t->numel() < 1)
    return kOther;
  out = static_cast<int32_t*>(t->data_ptr());
  return kUsual;
}

bool whole(PyObject* o, int64_t lo, int64_t hi, int64_t& out) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  out = PyLong_AsLongLongAndOverflow(o, &over);
  return over == 0 && out >= lo && out <= hi;
}

// A contiguous tensor over a part of `base`'s storage (one allocation serves a call's outputs).
at::Tensor part_of(const at::Tensor& base, at::ScalarType type, int64_t byte, int64_t n) {
  const caffe2::TypeMeta meta = c10::scalarTypeToTypeMeta(type);
  auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(base.storage()), base.key_set(), meta);
  impl->set_storage_offset(byte / static_cast<int64_t>(meta.itemsize()));
  impl->set_sizes_contiguous({n});
  return at::Tensor(std::move(impl));
}

// Whether a call on `t` would lose a gradient, backward or forward (the general path refuses).
bool needs_grad(const at::Tensor& t) {
  return (t.requires_grad() && c10::GradMode::is_enabled()) || t._fw_grad(0).defined();
}

// The addresses of a [tokens, heads, D] tensor's rows, from its first byte to behind its last.
struct Range {
  uintptr_t from, to;
  bool meets(uintptr_t a, uintptr_t b) const { return from < b && a < to; }
};

Range range_of(const at::Tensor& t) {
  const uintptr_t from = reinterpret_cast<uintptr_t>(t.data_ptr());
  if (t.numel() == 0) return {from, from};
  const int64_t last = (t.size(0) - 1) * t.stride(0) + (t.size(1) - 1) * t.stride(1) + t.size(2);
  return {from, from + static_cast<uintptr_t>(last) * t.element_size()};
}

// Whether two [tokens, heads, D] tensors' rows share no memory, as far as their ranges say it, or
// that they are parts of one projection: the same step from token to token, and within it the one's
// heads beside the other's.  (Others interleave in ways that the general path looks into.)
bool apart(const at::Tensor& a, const at::Tensor& b) {
  const Range x = range_of(a), y = range_of(b);
  if (a.numel() == 0 || b.numel() == 0 || !x.meets(y.from, y.to)) return true;
  const int64_t size = a.element_size(), step = a.stride(0) * size;
  if (a.size(0) < 2 || b.size(0) < 2 || a.stride(0) != b.stride(0) || step <= 0) return false;
  const auto span = [size](const at::Tensor& t) {
    return ((t.size(1) - 1) * t.stride(1) + t.size(2)) * size;
  };
  const int64_t off = static_cast<int64_t>(y.from - x.from) % step, from = off < 0 ? off + step : off;
  return from >= span(a) && from + span(b) <= step;
}

// Whether rows in `r` may lie in the cache.
bool meets_cache(const Range& r, const mkv_scaled_cache_t& c) {
  if (c.num_blocks <= 0) return false;
  const uintptr_t size = (c.num_blocks - 1) * c.block_stride + (c.heads - 1) * c.head_stride +
                         (c.block_size - 1) * c.token_stride + c.head_size;
  for (const void* p : {static_cast<const void*>(c.k_base), static_cast<const void*>(c.v_base)})
    if (r.meets(reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + size)) return true;
  const uintptr_t s = reinterpret_cast<uintptr_t>(c.scales);
  return r.meets(s, s + 2 * c.num_blocks * c.heads);
}

// slots(held, new, block_tables, free_blocks, free_at, block_size, max_tokens, error_flags)
PyObject* slots(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 8 || g_slots == nullptr) {
    PyErr_SetString(PyExc_TypeError, "slots takes 8 arguments, after bind_scaled()");
    return nullptr;
  }
  try {
    if (at::impl::PythonTorchFunctionTLS::stack_len() != 0) Py_RETURN_NONE;
    Table tab;
    if (!table_of(args[2], nullptr, tab) || (tab.n > 1 && tab.stride < tab.width)) Py_RETURN_NONE;
    const at::Device dev = THPVariable_Unpack(args[2]).device();
    const int32_t* held = vector_of(args[0], dev, tab.n);
    const int32_t* fresh = vector_of(args[1], dev, tab.n);
    const int32_t* free_blocks = vector_of(args[3], dev, -1);
    const int32_t* free_at = vector_of(args[4], dev, 1);
    int64_t bs, most;
    int32_t* flags;
    if (held == nullptr || fresh == nullptr || free_blocks == nullptr || free_at == nullptr ||
        !whole(args[5], 1, INT32_MAX, bs) || !whole(args[6], 0, INT32_MAX, most) ||
        flags_of(args[7], dev, flags) != kUsual || c10::hip::current_device() != dev.index())
      Py_RETURN_NONE;
    const int64_t free_len = THPVariable_Unpack(args[3]).numel(), n = tab.n;
    // slots, positions, starts, lens, free_at: each at a multiple of 16 bytes
    const auto up = [](int64_t x) { return (x + 15) / 16 * 16; };
    const int64_t at1 = up(8 * most), at2 = at1 + up(4 * most), at3 = at2 + up(4 * (n + 1)),
                  at4 = at3 + up(4 * n);
    const at::Tensor base = at::empty({(at4 + 16) / 8}, at::TensorOptions().dtype(at::kLong).device(dev));
    char* b = static_cast<char*>(base.data_ptr());
    void* stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_slots(held, fresh, static_cast<int32_t>(n), tab.at, tab.stride,
                 static_cast<int32_t>(tab.width), free_blocks, free_len, free_at,
                 static_cast<int32_t>(bs), reinterpret_cast<int32_t*>(b + at2),
                 reinterpret_cast<int32_t*>(b + at3), reinterpret_cast<int64_t*>(b),
                 reinterpret_cast<int32_t*>(b + at1), most, reinterpret_cast<int32_t*>(b + at4), flags,
                 stream);
    Py_END_ALLOW_THREADS
    if (rc != MKV_OK) return PyLong_FromLong(rc);
    const at::Tensor out[5] = {part_of(base, at::kInt, at2, n + 1), part_of(base, at::kInt, at3, n),
                               part_of(base, at::kLong, 0, most), part_of(base, at::kInt, at1, most),
                               part_of(base, at::kInt, at4, 1)};
    PyObject* made = PyTuple_New(5);
    if (made == nullptr) return nullptr;
    for (int i = 0; i < 5; ++i) {
      PyObject* o = THPVariable_Wrap(out[i]);
      if (o == nullptr) {
        Py_DECREF(made);
        return nullptr;
      }
      PyTuple_SET_ITEM(made, i, o);
    }
    return made;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// store(cache descriptor's address, device index, k, v, block_tables, starts, lens, error_flags)
PyObject* store(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 8 || g_store == nullptr) {
    PyErr_SetString(PyExc_TypeError, "store takes 8 arguments, after bind_scaled()");
    return nullptr;
  }
  try {
    if (at::impl::PythonTorchFunctionTLS::stack_len() != 0) Py_RETURN_NONE;
    const auto* cache = static_cast<const mkv_scaled_cache_t*>(PyLong_AsVoidPtr(args[0]));
    if (cache == nullptr) return nullptr;
    int64_t index;
    const at::Tensor* k = plain(args[2]);
    const at::Tensor* v = plain(args[3]);
    if (!whole(args[1], 0, 127, index) || k == nullptr || v == nullptr || !k->is_cuda()) Py_RETURN_NONE;
    const at::Device dev(at::kCUDA, static_cast<c10::DeviceIndex>(index));
    Table tab;
    int32_t* flags;
    const int code = dtype_code(k->scalar_type());
    if (k->dim() != 3 || k->device() != dev || v->device() != dev || k->sizes() != v->sizes() ||
        k->scalar_type() != v->scalar_type() || (code != MKV_BF16 && code != MKV_F16 && code != MKV_F32) ||
        k->size(1) != cache->heads || k->size(2) != cache->head_size || k->stride(2) != 1 ||
        v->stride(2) != 1 || needs_grad(*k) || needs_grad(*v) || !table_of(args[4], &dev, tab) ||
        flags_of(args[7], dev, flags) != kUsual ||
        c10::hip::current_device() != dev.index())
      Py_RETURN_NONE;
    const int32_t* starts = vector_of(args[5], dev, tab.n + 1);
    const int32_t* lens = vector_of(args[6], dev, tab.n);
    if (starts == nullptr || lens == nullptr) Py_RETURN_NONE;
    const int64_t n = k->size(0), many = n > 1, heads = k->size(1) > 1;
    void* stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
    const void* kp = k->data_ptr();
    const void* vp = v->data_ptr();
    const int64_t kt = many ? k->stride(0) : 0, kh = heads ? k->stride(1) : 0,
                  vt = many ? v->stride(0) : 0, vh = heads ? v->stride(1) : 0;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_store(cache, kp, kt, kh, vp, vt, vh, n, code, tab.at, tab.stride,
                 static_cast<int32_t>(tab.width), starts, lens, static_cast<int32_t>(tab.n), flags, stream);
    Py_END_ALLOW_THREADS
    if (rc != MKV_OK) return PyLong_FromLong(rc);
    Py_RETURN_TRUE;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// An attention call's arguments, but for its workspace: cache descriptor's address, device index,
// q, block_tables, starts, lens, scale, max_new, max_len, out, error_flags.
int read_attend(PyObject* cache_at, PyObject* device, PyObject* q_o, PyObject* tables, PyObject* starts_o,
                PyObject* lens_o, PyObject* scale, PyObject* max_new, PyObject* max_len, PyObject* out_o,
                PyObject* flags_o, mkv_attend_desc_t& d, at::Device& dev, at::Tensor& out) {
  if (at::impl::PythonTorchFunctionTLS::stack_len() != 0) return kOther;
  const auto* cache = static_cast<const mkv_scaled_cache_t*>(PyLong_AsVoidPtr(cache_at));
  if (cache == nullptr) return kError;
  int64_t index, most_new = 0, most_len = 0;
  const at::Tensor* q = plain(q_o);
  if (!whole(device, 0, 127, index) || q == nullptr || !q->is_cuda()) return kOther;
  dev = at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(index));
  Table tab;
  int32_t* flags;
  const int code = dtype_code(q->scalar_type());
  if (q->dim() != 3 || q->device() != dev || (code != MKV_BF16 && code != MKV_F16) ||
      cache->heads <= 0 || q->size(2) != cache->head_size || q->size(1) == 0 ||
      q->size(1) % cache->heads != 0 || q->size(1) > INT32_MAX || q->stride(2) != 1 ||
      needs_grad(*q) || !table_of(tables, &dev, tab) ||
      flags_of(flags_o, dev, flags) != kUsual || c10::hip::current_device() != dev.index())
    return kOther;
  const int32_t* starts = vector_of(starts_o, dev, tab.n + 1);
  const int32_t* lens = vector_of(lens_o, dev, tab.n);
  if (starts == nullptr || lens == nullptr ||
      (max_new != Py_None && !whole(max_new, 0, INT32_MAX, most_new)) ||
      (max_len != Py_None && !whole(max_len, 0, INT32_MAX, most_len)))
    return kOther;
  if (scale == Py_None) {
    d.softmax_scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(cache->head_size)));
  } else {
    if (!PyFloat_CheckExact(scale)) return kOther;
    d.softmax_scale = static_cast<float>(PyFloat_AS_DOUBLE(scale));
  }
  if (out_o == Py_None) {
    out = at::empty(q->sizes(), at::TensorOptions().dtype(q->dtype()).device(dev));
  } else {
    const at::Tensor* o = plain(out_o);
    if (o == nullptr || o->device() != dev || o->scalar_type() != q->scalar_type() ||
        o->sizes() != q->sizes() || o->stride(2) != 1 || needs_grad(*o))
      return kOther;
    // the general path tells rows that interleave from rows that share memory
    const Range rows = range_of(*q), written = range_of(*o);
    if (written.meets(rows.from, rows.to) || meets_cache(written, *cache)) return kOther;
    out = *o;
  }
  const bool many = q->size(0) > 1, heads = q->size(1) > 1;
  d.cache = *cache;
  d.q = q->data_ptr();
  d.out = out.data_ptr();
  d.block_tables = tab.at;
  d.starts = starts;
  d.lens = lens;
  d.error_flags = flags;
  d.q_token_stride = many ? q->stride(0) : 0;
  d.q_head_stride = heads ? q->stride(1) : 0;
  d.out_token_stride = many ? out.stride(0) : 0;
  d.out_head_stride = heads ? out.stride(1) : 0;
  d.table_stride = tab.stride;
  d.tokens = q->size(0);
  d.table_width = static_cast<int32_t>(tab.width);
  d.requests = static_cast<int32_t>(tab.n);
  d.q_heads = static_cast<int32_t>(q->size(1));
  d.dtype = code;
  d.max_new = static_cast<int32_t>(most_new);
  d.max_len = static_cast<int32_t>(most_len);
  return kUsual;
}

// Launches the call with a workspace of `need` bytes, whose memory goes back in stream order.
template <typename F>
PyObject* launch_attend(mkv_attend_desc_t& d, int64_t need, const at::Device& dev, PyObject* out_o,
                        const at::Tensor& out, F call) {
  at::Tensor workspace;
  if (need > 0) {
    workspace = at::empty({need}, at::TensorOptions().dtype(at::kByte).device(dev));
    d.workspace = workspace.data_ptr();
    d.workspace_bytes = need;
  }
  void* stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = call(stream);
  Py_END_ALLOW_THREADS
  if (rc != MKV_OK) return PyLong_FromLong(rc);
  if (out_o != Py_None) return (Py_INCREF(out_o), out_o);
  return THPVariable_Wrap(out);
}

// attend(cache descriptor's address, device index, q, block_tables, starts, lens, scale,
//        max_new, max_len, out, error_flags)
PyObject* attend(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 11 || g_attend == nullptr || g_attend_size == nullptr) {
    PyErr_SetString(PyExc_TypeError, "attend takes 11 arguments, after bind_scaled()");
    return nullptr;
  }
  try {
    mkv_attend_desc_t d{};
    at::Device dev(at::kCPU);
    at::Tensor out;
    const int got = read_attend(args[0], args[1], args[2], args[3], args[4], args[5], args[6], args[7],
                                args[8], args[9], args[10], d, dev, out);
    if (got == kError) return nullptr;
    if (got == kOther) Py_RETURN_NONE;
    return launch_attend(d, g_attend_size(&d), dev, args[9], out,
                         [&](void* stream) { return g_attend(&d, stream); });
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// ------------------------------------------------------- the step around the cache

typedef decltype(&mkv_norm_rotate) rotate_fn;
typedef decltype(&mkv_store_rotated) put_fn;
typedef decltype(&mkv_attend_shared) shared_fn;
typedef decltype(&mkv_attend_shared_workspace_size) shared_size_fn;
rotate_fn g_rotate = nullptr;
put_fn g_put = nullptr;
shared_fn g_shared = nullptr;
shared_size_fn g_shared_size = nullptr;

// The heads' rows, and their output, kept in `out`: a fresh one, the rows themselves, or the caller's
// apart from them.
bool rows_of(PyObject* x_o, PyObject* out_o, const at::Device& dev, int64_t d, int code,
             mkv_head_rows_t& r, at::Tensor& out) {
  const at::Tensor* x = plain(x_o);
  if (x == nullptr || x->device() != dev || x->dim() != 3 || x->size(2) != d || x->stride(2) != 1 ||
      dtype_code(x->scalar_type()) != code || x->size(1) > 65536 || needs_grad(*x))
    return false;
  if (out_o == Py_None) {
    out = at::empty(x->sizes(), at::TensorOptions().dtype(x->dtype()).device(dev));
  } else {
    const at::Tensor* o = plain(out_o);
    if (o == nullptr || o->device() != dev || o->scalar_type() != x->scalar_type() ||
        o->sizes() != x->sizes() || o->stride(2) != 1 || needs_grad(*o) ||
        !((o->data_ptr() == x->data_ptr() && o->strides() == x->strides()) || apart(*o, *x)))
      return false;
    out = *o;
  }
  const bool many = x->size(0) > 1, heads = x->size(1) > 1;
  r.x = x->data_ptr();
  r.out = out.data_ptr();
  r.token_stride = many ? x->stride(0) : 0;
  r.head_stride = heads ? x->stride(1) : 0;
  r.out_token_stride = many ? out.stride(0) : 0;
  r.out_head_stride = heads ? out.stride(1) : 0;
  r.heads = static_cast<int32_t>(x->size(1));
  return true;
}

// A contiguous vector on `dev` (of n values, unless n < 0) that needs no gradient, or null.
const at::Tensor* values_of(PyObject* o, const at::Device& dev, int64_t n) {
  const at::Tensor* t = plain(o);
  return t == nullptr || t->device() != dev || t->dim() != 1 || !t->is_contiguous() ||
                 (n >= 0 && t->size(0) != n) || needs_grad(*t)
             ? nullptr
             : t;
}

// inv_freq, q_weight, k_weight, eps.
bool turn_of(PyObject* freq, PyObject* qw, PyObject* kw, PyObject* eps, const at::Device& dev, int64_t d,
             mkv_turn_t& turn) {
  if (freq != Py_None) {
    const at::Tensor* f = values_of(freq, dev, -1);
    if (f == nullptr || f->scalar_type() != at::kFloat || f->size(0) == 0 || f->size(0) % 16 != 0 ||
        2 * f->size(0) > d)
      return false;
    turn.inv_freq = static_cast<const float*>(f->data_ptr());
    turn.rotary = static_cast<int32_t>(2 * f->size(0));
  }
  if (!PyFloat_CheckExact(eps)) return eps == Py_None && qw == Py_None && kw == Py_None;
  turn.norm = 1;
  turn.eps = static_cast<float>(PyFloat_AS_DOUBLE(eps));
  if (!(turn.eps >= 0.0f) || std::isinf(turn.eps)) return false;
  int code = -1;
  const void** to[2] = {&turn.q_weight, &turn.k_weight};
  for (int i = 0; i < 2; ++i) {
    PyObject* o = i == 0 ? qw : kw;
    if (o == Py_None) continue;
    const at::Tensor* w = values_of(o, dev, d);
    if (w == nullptr) return false;
    const int c = dtype_code(w->scalar_type());
    if ((c != MKV_BF16 && c != MKV_F16 && c != MKV_F32) || (code >= 0 && c != code)) return false;
    code = c;
    *to[i] = w->data_ptr();
  }
  turn.weight_dtype = code < 0 ? 0 : code;
  return true;
}

// Whether any of some plain tensors, read as they lie in memory, has a byte among an output's rows.
template <typename... T>
bool reads_from(const Range& r, T... read) {
  for (PyObject* o : {read...}) {
    const at::Tensor* t = plain(o);
    if (t == nullptr || t->numel() == 0) continue;
    int64_t last = 1;
    for (int64_t i = 0; i < t->dim(); ++i) last += (t->size(i) - 1) * t->stride(i);
    const uintptr_t from = reinterpret_cast<uintptr_t>(t->data_ptr());
    if (r.meets(from, from + static_cast<uintptr_t>(last) * t->element_size())) return true;
  }
  return false;
}

bool row_type(int code) { return code == MKV_BF16 || code == MKV_F16 || code == MKV_F32; }

// rotate(q, k, positions, inv_freq, q_weight, k_weight, eps, out_q, out_k)
PyObject* rotate(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 9 || g_rotate == nullptr) {
    PyErr_SetString(PyExc_TypeError, "rotate takes 9 arguments, after bind_step()");
    return nullptr;
  }
  try {
    if (at::impl::PythonTorchFunctionTLS::stack_len() != 0) Py_RETURN_NONE;
    const at::Tensor* q = plain(args[0]);
    const at::Tensor* k = plain(args[1]);
    if (q == nullptr || k == nullptr || !q->is_cuda() || q->dim() != 3 || k->dim() != 3 ||
        q->size(0) != k->size(0) || c10::hip::current_device() != q->device().index())
      Py_RETURN_NONE;
    const at::Device dev = q->device();
    const int64_t d = q->size(2), n = q->size(0);
    const int code = dtype_code(q->scalar_type());
    mkv_norm_rotate_desc_t desc{};
    at::Tensor out_q, out_k;
    if ((d != 64 && d != 128 && d != 256) || !row_type(code) ||
        !turn_of(args[3], args[4], args[5], args[6], dev, d, desc.turn))
      Py_RETURN_NONE;
    if (desc.turn.rotary > 0) {
      const at::Tensor* p = values_of(args[2], dev, n);
      if (p == nullptr || (p->scalar_type() != at::kInt && p->scalar_type() != at::kLong)) Py_RETURN_NONE;
      desc.positions = p->data_ptr();
      desc.position_bytes = p->scalar_type() == at::kInt ? 4 : 8;
    }
    if (!rows_of(args[0], args[7], dev, d, code, desc.q, out_q) ||
        !rows_of(args[1], args[8], dev, d, code, desc.k, out_k))
      Py_RETURN_NONE;
    // a caller's outputs: apart from the other rows, from each other and from what is read
    const bool mine[2] = {args[7] != Py_None, args[8] != Py_None};
    if ((mine[0] && (!apart(out_q, *k) || reads_from(range_of(out_q), args[2], args[3], args[4], args[5]))) ||
        (mine[1] && (!apart(out_k, *q) || reads_from(range_of(out_k), args[2], args[3], args[4], args[5]))) ||
        (mine[0] && mine[1] && !apart(out_q, out_k)))
      Py_RETURN_NONE;
    desc.tokens = n;
    desc.head_size = static_cast<int32_t>(d);
    desc.dtype = code;
    void* stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_rotate(&desc, stream);
    Py_END_ALLOW_THREADS
    if (rc != MKV_OK) return PyLong_FromLong(rc);
    PyObject* made = PyTuple_New(2);
    if (made == nullptr) return nullptr;
    for (int i = 0; i < 2; ++i) {
      PyObject* given = args[7 + i];
      PyObject* o = given != Py_None ? (Py_INCREF(given), given) : THPVariable_Wrap(i == 0 ? out_q : out_k);
      if (o == nullptr) {
        Py_DECREF(made);
        return nullptr;
      }
      PyTuple_SET_ITEM(made, i, o);
    }
    return made;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// put(cache descriptor's address, device index, q, k, v, block_tables, starts, lens, inv_freq,
//     q_weight, k_weight, eps, out_q, error_flags)
PyObject* put(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 14 || g_put == nullptr) {
    PyErr_SetString(PyExc_TypeError, "put takes 14 arguments, after bind_step()");
    return nullptr;
  }
  try {
    if (at::impl::PythonTorchFunctionTLS::stack_len() != 0) Py_RETURN_NONE;
    const auto* cache = static_cast<const mkv_scaled_cache_t*>(PyLong_AsVoidPtr(args[0]));
    if (cache == nullptr) return nullptr;
    int64_t index;
    const at::Tensor* q = plain(args[2]);
    const at::Tensor* k = plain(args[3]);
    const at::Tensor* v = plain(args[4]);
    if (!whole(args[1], 0, 127, index) || q == nullptr || k == nullptr || v == nullptr || !q->is_cuda())
      Py_RETURN_NONE;
    const at::Device dev(at::kCUDA, static_cast<c10::DeviceIndex>(index));
    const int code = dtype_code(q->scalar_type());
    Table tab;
    int32_t* flags;
    mkv_store_rotated_desc_t d{};
    at::Tensor out;
    if (!row_type(code) || k->dim() != 3 || v->dim() != 3 || k->sizes() != v->sizes() ||
        k->device() != dev || v->device() != dev || dtype_code(k->scalar_type()) != code ||
        dtype_code(v->scalar_type()) != code || k->size(1) != cache->heads ||
        k->size(2) != cache->head_size || k->stride(2) != 1 || v->stride(2) != 1 || needs_grad(*k) ||
        needs_grad(*v) || c10::hip::current_device() != dev.index() || !table_of(args[5], &dev, tab) ||
        flags_of(args[13], dev, flags) != kUsual || q->dim() != 3 || q->size(0) != k->size(0) ||
        !turn_of(args[8], args[9], args[10], args[11], dev, cache->head_size, d.turn))
      Py_RETURN_NONE;
    const int32_t* starts = vector_of(args[6], dev, tab.n + 1);
    const int32_t* lens = vector_of(args[7], dev, tab.n);
    if (starts == nullptr || lens == nullptr ||
        !rows_of(args[2], args[12], dev, cache->head_size, code, d.q, out))
      Py_RETURN_NONE;
    if (args[12] != Py_None) {
      const Range written = range_of(out);
      if (!apart(out, *k) || !apart(out, *v) || meets_cache(written, *cache) ||
          reads_from(written, args[5], args[6], args[7], args[8], args[9], args[10]))
        Py_RETURN_NONE;
    }
    const bool many = k->size(0) > 1, heads = k->size(1) > 1;
    d.cache = *cache;
    d.k = k->data_ptr();
    d.v = v->data_ptr();
    d.k_token_stride = many ? k->stride(0) : 0;
    d.k_head_stride = heads ? k->stride(1) : 0;
    d.v_token_stride = many ? v->stride(0) : 0;
    d.v_head_stride = heads ? v->stride(1) : 0;
    d.block_tables = tab.at;
    d.starts = starts;
    d.lens = lens;
    d.error_flags = flags;
    d.table_stride = tab.stride;
    d.tokens = q->size(0);
    d.table_width = static_cast<int32_t>(tab.width);
    d.requests = static_cast<int32_t>(tab.n);
    d.dtype = code;
    void* stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_put(&d, stream);
    Py_END_ALLOW_THREADS
    if (rc != MKV_OK) return PyLong_FromLong(rc);
    return args[12] != Py_None ? (Py_INCREF(args[12]), args[12]) : THPVariable_Wrap(out);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// attend_shared(cache descriptor's address, device index, q, block_tables, starts, lens, groups,
//               shared, scale, max_new, max_shared, max_own, out, error_flags)
PyObject* attend_shared(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 14 || g_shared == nullptr || g_shared_size == nullptr) {
    PyErr_SetString(PyExc_TypeError, "attend_shared takes 14 arguments, after bind_step()");
    return nullptr;
  }
  try {
    mkv_attend_shared_desc_t d{};
    at::Device dev(at::kCPU);
    at::Tensor out;
    int64_t most = 0;
    const int got = read_attend(args[0], args[1], args[2], args[3], args[4], args[5], args[8], args[9],
                                args[11], args[12], args[13], d.attend, dev, out);
    if (got == kError) return nullptr;
    if (got == kOther || (args[10] != Py_None && !whole(args[10], 0, INT32_MAX, most))) Py_RETURN_NONE;
    d.shared = vector_of(args[7], dev, -1);
    if (d.shared == nullptr) Py_RETURN_NONE;
    const int64_t n = THPVariable_Unpack(args[7]).size(0);
    d.groups = n <= MKV_MAX_REQUESTS ? vector_of(args[6], dev, n + 1) : nullptr;
    if (d.groups == nullptr) Py_RETURN_NONE;
    d.n_groups = static_cast<int32_t>(n);
    d.max_shared = static_cast<int32_t>(most);
    return launch_attend(d.attend, g_shared_size(&d), dev, args[12], out,
                         [&](void* stream) { return g_shared(&d, stream); });
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// The addresses that a bind takes; false with an exception set.
bool addresses(PyObject* const* args, Py_ssize_t nargs, void* (&p)[4]) {
  if (nargs != 4) {
    PyErr_SetString(PyExc_TypeError, "4 addresses");
    return false;
  }
  for (int i = 0; i < 4; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (p[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "NULL function");
      return false;
    }
  }
  return true;
}

// The addresses of mkv_norm_rotate, mkv_store_rotated, mkv_attend_shared and
// mkv_attend_shared_workspace_size.
PyObject* bind_step(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  void* p[4];
  if (!addresses(args, nargs, p)) return nullptr;
  g_rotate = reinterpret_cast<rotate_fn>(p[0]);
  g_put = reinterpret_cast<put_fn>(p[1]);
  g_shared = reinterpret_cast<shared_fn>(p[2]);
  g_shared_size = reinterpret_cast<shared_size_fn>(p[3]);
  Py_RETURN_NONE;
}

// The addresses of mkv_step_slots, mkv_store_scaled, mkv_attend_scaled and
// mkv_attend_workspace_size.
PyObject* bind_scaled(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  void* p[4];
  if (!addresses(args, nargs, p)) return nullptr;
  g_slots = reinterpret_cast<slots_fn>(p[0]);
  g_store = reinterpret_cast<store_fn>(p[1]);
  g_attend = reinterpret_cast<attend_fn>(p[2]);
  g_attend_size = reinterpret_cast<attend_size_fn>(p[3]);
  Py_RETURN_NONE;
}

PyObject* bind(PyObject*, PyObject* address) {
  void* p = PyLong_AsVoidPtr(address);
  if (p == nullptr) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "NULL function");
    return nullptr;
  }
  g_scatter = reinterpret_cast<scatter_fn>(p);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"scatter", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(scatter)), METH_FASTCALL,
     "mkv_scatter_shifted on torch tensors; None: take the general path"},
    {"bind", bind, METH_O, "the address of mkv_scatter_shifted"},
    {"slots", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(slots)), METH_FASTCALL,
     "mkv_step_slots on torch tensors; None: take the general path"},
    {"store", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(store)), METH_FASTCALL,
     "mkv_store_scaled on torch tensors; None: take the general path"},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attend)), METH_FASTCALL,
     "mkv_attend_scaled on torch tensors; None: take the general path"},
    {"bind_scaled", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind_scaled)),
     METH_FASTCALL, "the addresses that slots, store and attend call"},
    {"rotate", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rotate)), METH_FASTCALL,
     "mkv_norm_rotate on torch tensors; None: take the general path"},
    {"put", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(put)), METH_FASTCALL,
     "mkv_store_rotated on torch tensors; None: take the general path"},
    {"attend_shared", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attend_shared)),
     METH_FASTCALL, "mkv_attend_shared on torch tensors; None: take the general path"},
    {"bind_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind_step)),
     METH_FASTCALL, "the addresses that rotate, put and attend_shared call"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "marathon_binding", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_marathon_binding() {
  s_delta = PyUnicode_InternFromString("delta");
  s_cos = PyUnicode_InternFromString("cos");
  s_sgn = PyUnicode_InternFromString("sgn");
  s_emb_cos = PyUnicode_InternFromString("emb_cos");
  s_rotary = PyUnicode_InternFromString("rotary");
  if (!s_delta || !s_cos || !s_sgn || !s_emb_cos || !s_rotary) return nullptr;
  // what it was compiled against; the loader compares them before it calls anything
  PyObject* m = PyModule_Create(&module);
  if (m == nullptr || PyModule_AddIntConstant(m, "abi", MKV_ABI_VERSION) != 0 ||
      PyModule_AddStringConstant(m, "torch", MARATHON_TORCH) != 0) {
    Py_XDECREF(m);
    return nullptr;
  }
  return m;
}
