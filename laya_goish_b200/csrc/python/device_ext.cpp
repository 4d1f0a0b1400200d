// Python binding of the operators on device buffers: torch tensors in and out,
// the C entry points of laya_cuda.h below.
//
// A call of these operators is a few microseconds of GPU work, and building
// the outputs and reading eight tensors' sizes, strides and types through
// Python attributes and ctypes took two to four times as long (16-20 us a
// call, against 4-11 here), so this is the one part of the package that binds
// in C++.  It checks what a tensor says of itself; the sizes' sense is checked
// by the entry points.  The functions here are called by laya_goish_b200.device.
#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <Python.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <initializer_list>
#include <string>

#include "laya_cuda.h"

namespace {

PyObject* g_error;  // laya_goish_b200._lib.LayaError
PyObject* g_oom;    // torch.OutOfMemoryError

struct Refused {};  // a Python error is set

[[noreturn]] void raise(int code, const std::string& message) {
  PyObject* e = PyObject_CallFunction(g_error, "is", code, message.c_str());
  if (e) {
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
  }
  throw Refused{};
}
[[noreturn]] void refuse(const std::string& message) { raise(LAYA_E_INVALID, message); }
void check(int rc) {
  if (rc < 0) raise(rc, laya_last_error());
}

// A call's body; C++ errors become Python ones.
template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const Refused&) {
  } catch (const c10::OutOfMemoryError& e) {  // what callers of torch catch
    PyErr_SetString(g_oom, e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

constexpr int kAny = -1;

const char* dtype_name(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    default: return "of another type";
  }
}

// The tensor behind an argument: CUDA, strided, of `dim` dimensions, `type`
// (or kAny) and `device` (or kAny).
const at::Tensor& tensor(PyObject* o, const char* name, int64_t dim, int type, int device) {
  if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a CUDA tensor");
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.layout() != at::kStrided) refuse(std::string(name) + " must be a CUDA tensor");
  if (t.dim() != dim) refuse(std::string(name) + " must have " + std::to_string(dim) + " dimension(s)");
  if (type != kAny && t.scalar_type() != (at::ScalarType)type)
    refuse(std::string(name) + " must be " + dtype_name((at::ScalarType)type));
  if (device != kAny && t.get_device() != device) refuse(std::string(name) + " is on another device");
  if (t.requires_grad() && c10::GradMode::is_enabled())
    refuse(std::string(name) + " requires a gradient; the operators are forward only");
  if (t._fw_grad(0).defined()) refuse(std::string(name) + " has a tangent; the operators are forward only");
  if (t.is_conj() || t.is_neg()) refuse(std::string(name) + " must not be a lazily negated view");
  return t;
}
const at::Tensor& flat(PyObject* o, const char* name, int type, int device) {
  const at::Tensor& t = tensor(o, name, 1, type, device);
  if (!t.is_contiguous()) refuse(std::string(name) + " must be contiguous");
  return t;
}
// Row stride of a tensor whose rows (everything past dimension 0) are contiguous.
int64_t rows_of(const at::Tensor& t, const char* name) {
  int64_t width = 1;
  for (int64_t d = t.dim() - 1; d > 0; d--) {
    if (t.size(d) != 1 && t.stride(d) != width) refuse(std::string("the rows of ") + name + " must be contiguous");
    width *= t.size(d);
  }
  return t.size(0) > 1 ? t.stride(0) : width;
}
long long integer(PyObject* o, const char* name, long long lo, long long hi) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    if (!PyErr_ExceptionMatches(PyExc_OverflowError)) throw Refused{};
    PyErr_Clear();
    refuse(std::string(name) + " out of range");
  }
  if (v < lo || v > hi) refuse(std::string(name) + " out of range");
  return v;
}
int32_t size32(int64_t v, const char* name) {
  if (v > INT32_MAX) refuse(std::string(name) + " out of range");
  return (int32_t)v;
}
void arguments(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
    throw Refused{};
  }
}
template <typename T = void>
T* ptr(const at::Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}
// An in-place write, for autograd: a tensor saved for a backward pass and
// written since is an error there.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
at::Tensor empty(at::IntArrayRef size, at::ScalarType type, int device) {
  return at::empty(size, at::TensorOptions().dtype(type).device(at::kCUDA, device));
}
void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }
PyObject* tuple_of(std::initializer_list<at::Tensor> ts) {
  PyObject* r = PyTuple_New(ts.size());
  if (!r) throw Refused{};
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) {
    PyObject* o = THPVariable_Wrap(t);
    if (!o) {
      Py_DECREF(r);
      throw Refused{};
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}
uint32_t type_code(at::ScalarType t) {
  return t == at::kFloat ? LAYA_TYPE_F32 : t == at::kHalf ? LAYA_TYPE_F16 : LAYA_TYPE_BF16;
}
at::ScalarType scalar_type(uint32_t code) { return code == LAYA_TYPE_F16 ? at::kHalf : at::kBFloat16; }

// (past, count, free_pages, tables, capacity, base)
PyObject* page_plan(PyObject*, PyObject* const* a, Py_ssize_t na) {
  return guarded([&]() -> PyObject* {
    arguments(na, 6);
    const at::Tensor& tables = tensor(a[3], "tables", 2, (int)at::kInt, kAny);
    const int dev = tables.get_device();
    const at::Tensor& past = flat(a[0], "past", (int)at::kInt, dev);
    const at::Tensor& count = flat(a[1], "count", (int)at::kInt, dev);
    const at::Tensor& free_pages = flat(a[2], "free_pages", (int)at::kInt, dev);
    const int64_t n = tables.size(0), width = tables.size(1);
    if (past.size(0) != n || count.size(0) != n) refuse("past, count and tables must have one row per sequence");
    if (n && width > 1 && tables.stride(1) != 1) refuse("the rows of tables must be contiguous");
    const int64_t stride = n > 1 ? tables.stride(0) : width;
    if (stride < width) refuse("the rows of tables overlap");
    const int capacity = (int)integer(a[4], "capacity", 0, INT32_MAX), base = (int)integer(a[5], "base", 0, INT32_MAX);
    c10::cuda::CUDAGuard guard(dev);
    at::AutoDispatchBelowADInplaceOrView below;
    // one allocation, each output on 16 bytes (the offsets below are in 32-bit words)
    const int64_t c4 = (capacity + 3ll) / 4 * 4, n4 = (n + 4) / 4 * 4;
    at::Tensor all = empty({2 * c4 + n4 + 2}, at::kLong, dev), words = all.view(at::kInt);
    auto part = [&](int64_t size, int64_t at) { return words.as_strided({size}, {1}, at); };
    at::Tensor slots = all.as_strided({capacity}, {1}, 0), totals = all.as_strided({2}, {1}, 2 * c4 + n4),
               positions = part(capacity, 2 * c4), seqs = part(capacity, 3 * c4), offsets = part(n + 1, 4 * c4),
               lens = part(n, 4 * c4 + n4);
    check(laya_page_plan(ptr<int32_t>(past), ptr<int32_t>(count), size32(n, "sequences"), ptr<int32_t>(free_pages),
                         size32(free_pages.size(0), "free_pages"), base, ptr<int32_t>(tables), stride,
                         size32(width, "tables"), ptr<int64_t>(slots), ptr<int32_t>(positions), ptr<int32_t>(seqs),
                         capacity, ptr<int32_t>(offsets), ptr<int32_t>(lens), ptr<int64_t>(totals), stream_of(dev)));
    written(tables);
    return tuple_of({slots, positions, seqs, offsets, lens, totals});
  });
}

const laya_kv_pages* pages_at(PyObject* o) {
  void* p = PyLong_AsVoidPtr(o);
  if (!p) throw Refused{};
  return static_cast<const laya_kv_pages*>(p);
}

// The tensors behind the pages, which may have come to require a gradient, or
// been given other memory, since the pages were described.
void page_tensors(const laya_kv_pages* c, PyObject* k, PyObject* v, int device) {
  const at::Tensor& tk = tensor(k, "k pages", 4, (int)scalar_type(c->type), device);
  const at::Tensor& tv = tensor(v, "v pages", 4, (int)scalar_type(c->type), device);
  if (tk.data_ptr() != c->k || tv.data_ptr() != c->v) refuse("the pages' tensors have moved since KVPages was made");
}

// (pages address, device, pages' k, pages' v, k, v, slots)
PyObject* kv_append(PyObject*, PyObject* const* a, Py_ssize_t na) {
  return guarded([&]() -> PyObject* {
    arguments(na, 7);
    const laya_kv_pages* c = pages_at(a[0]);
    const int dev = (int)integer(a[1], "device", 0, INT32_MAX);
    page_tensors(c, a[2], a[3], dev);
    const at::Tensor& k = tensor(a[4], "k", 3, kAny, dev);
    const at::Tensor& v = tensor(a[5], "v", 3, (int)k.scalar_type(), dev);
    const at::Tensor& slots = flat(a[6], "slots", (int)at::kLong, dev);
    if (k.scalar_type() != scalar_type(c->type) && k.scalar_type() != at::kFloat)
      refuse("k and v must be of the pages' type or F32");
    if (k.sizes() != v.sizes() || k.size(0) != slots.size(0) || k.size(1) != c->kv_heads || k.size(2) != c->head_dim)
      refuse("k and v must be [rows, kv_heads, head_dim] with a slot per row");
    c10::cuda::CUDAGuard guard(dev);
    check(laya_kv_append(c, type_code(k.scalar_type()), ptr(k), ptr(v), rows_of(k, "k"), rows_of(v, "v"),
                         ptr<int64_t>(slots), size32(k.size(0), "rows"), stream_of(dev)));
    written(THPVariable_Unpack(a[2]));
    written(THPVariable_Unpack(a[3]));
    Py_RETURN_NONE;
  });
}

// (pages address, device, pages' k, pages' v, q, prefix_pages, prefix_len, tables, lens, offsets, max_q, scale or None, out or None, lse or None)
PyObject* prefix_attention(PyObject*, PyObject* const* a, Py_ssize_t na) {
  return guarded([&]() -> PyObject* {
    arguments(na, 14);
    const laya_kv_pages* c = pages_at(a[0]);
    const int dev = (int)integer(a[1], "device", 0, INT32_MAX);
    page_tensors(c, a[2], a[3], dev);
    const at::ScalarType type = scalar_type(c->type);
    const at::Tensor& q = tensor(a[4], "q", 3, (int)type, dev);
    const at::Tensor& prefix_pages = flat(a[5], "prefix_pages", (int)at::kInt, dev);
    const at::Tensor& tables = tensor(a[7], "tables", 2, (int)at::kInt, dev);
    const at::Tensor& lens = flat(a[8], "lens", (int)at::kInt, dev);
    const at::Tensor& offsets = flat(a[9], "offsets", (int)at::kInt, dev);
    const int64_t n = tables.size(0), width = tables.size(1), rows = q.size(0), heads = q.size(1), hd = q.size(2);
    if (hd != c->head_dim) refuse("q and the pages have different head_dim");
    if (!heads || heads % c->kv_heads) refuse("heads must be a multiple of kv_heads");
    if (lens.size(0) != n || offsets.size(0) != n + 1) refuse("lens, offsets and tables must fit the sequences");
    if (n && width > 1 && tables.stride(1) != 1) refuse("the rows of tables must be contiguous");
    laya_prefix_args p{};
    p.prefix_len = (int32_t)integer(a[6], "prefix_pages must hold prefix_len tokens: prefix_len", 0, INT32_MAX);
    if (p.prefix_len > prefix_pages.size(0) * LAYA_PAGE_TOKENS) refuse("prefix_pages must hold prefix_len tokens");
    p.max_q = (int32_t)integer(a[10], "max_q", 0, INT32_MAX);
    if (a[11] == Py_None) {
      p.scale = (float)(1.0 / std::sqrt((double)hd));
    } else {
      const double s = PyFloat_AsDouble(a[11]);
      if (s == -1.0 && PyErr_Occurred()) throw Refused{};
      p.scale = (float)s;
    }
    c10::cuda::CUDAGuard guard(dev);
    at::AutoDispatchBelowADInplaceOrView below;
    const bool given = a[12] != Py_None;
    at::Tensor made;
    if (!given) made = at::zeros(q.sizes(), q.options());
    const at::Tensor& out = given ? tensor(a[12], "out", 3, (int)type, dev) : made;
    if (out.sizes() != q.sizes()) refuse("out must have q's shape");
    if (a[13] != Py_None) {
      const at::Tensor& lse = tensor(a[13], "lse", 2, (int)at::kFloat, dev);
      if (lse.size(0) != rows || lse.size(1) != heads || !lse.is_contiguous())
        refuse("lse must be contiguous [rows, heads]");
      p.lse = ptr<float>(lse);
    }
    p.q = ptr(q);
    p.q_stride = rows_of(q, "q");
    p.rows = size32(rows, "rows");
    p.heads = size32(heads, "heads");
    p.offsets = ptr<int32_t>(offsets);
    p.n_seqs = size32(n, "sequences");
    p.prefix_pages = ptr<int32_t>(prefix_pages);
    p.width = size32(width, "tables");
    p.tables = ptr<int32_t>(tables);
    p.table_stride = n > 1 ? tables.stride(0) : width;
    p.lens = ptr<int32_t>(lens);
    p.out = ptr(out);
    p.out_stride = rows_of(out, "out");
    p.workspace_bytes = laya_prefix_attention_workspace(c, &p);
    at::Tensor work;
    if (p.workspace_bytes) {
      work = empty({(int64_t)p.workspace_bytes}, at::kByte, dev);
      p.workspace = ptr(work);
    }
    check(laya_prefix_attention(c, &p, stream_of(dev)));
    if (p.lse) written(THPVariable_Unpack(a[13]));
    if (!given) return THPVariable_Wrap(made);
    written(out);
    Py_INCREF(a[12]);
    return a[12];
  });
}

// (logits, tokens, top)
PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t na) {
  return guarded([&]() -> PyObject* {
    arguments(na, 3);
    const at::Tensor& x = tensor(a[0], "logits", 2, kAny, kAny);
    const int dev = x.get_device();
    const at::ScalarType type = x.scalar_type();
    if (type != at::kFloat && type != at::kHalf && type != at::kBFloat16) refuse("logits must be F32, F16 or BF16");
    const at::Tensor& tokens = tensor(a[1], "tokens", 2, (int)at::kInt, dev);
    const int64_t n = x.size(0), vocab = x.size(1), c = tokens.size(1);
    if (!vocab) refuse("empty vocabulary");
    if (tokens.size(0) != n) refuse("tokens must have a row per row of logits");
    const int top = (int)integer(a[2], "top", 0, LAYA_MAX_TOP);
    const int64_t xs = rows_of(x, "logits"), ts = c ? rows_of(tokens, "tokens") : 0;
    c10::cuda::CUDAGuard guard(dev);
    at::AutoDispatchBelowADInplaceOrView below;
    at::Tensor all = empty({n * (c + 2 + 2 * top)}, at::kFloat, dev);
    auto part = [&](const at::Tensor& t, int64_t size, int64_t at) { return t.as_strided({n, size}, {size, 1}, at); };
    at::Tensor logprobs = part(all, c, 0), entropy = all.as_strided({n}, {1}, n * c),
               lse = all.as_strided({n}, {1}, n * (c + 1)), top_lp = part(all, top, n * (c + 2)),
               ids = part(all.view(at::kInt), top, n * (c + 2 + top));
    check(laya_token_logprobs(type_code(type), ptr(x), xs, size32(n, "rows"), size32(vocab, "vocabulary"),
                              ptr<int32_t>(tokens), ts, size32(c, "tokens"), top, ptr<float>(logprobs),
                              ptr<float>(entropy), ptr<float>(lse), ptr<int32_t>(ids), ptr<float>(top_lp),
                              stream_of(dev)));
    return tuple_of({logprobs, entropy, lse, ids, top_lp});
  });
}

#define LAYA_METHOD(f) \
  { #f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr }
PyMethodDef g_methods[] = {LAYA_METHOD(page_plan), LAYA_METHOD(kv_append), LAYA_METHOD(prefix_attention),
                           LAYA_METHOD(token_logprobs), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_device", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__device(void) {
  PyObject* lib = PyImport_ImportModule("laya_goish_b200._lib");
  if (!lib) return nullptr;
  g_error = PyObject_GetAttrString(lib, "LayaError");
  Py_DECREF(lib);
  PyObject* torch = g_error ? PyImport_ImportModule("torch") : nullptr;
  if (!torch) return nullptr;
  g_oom = PyObject_GetAttrString(torch, "OutOfMemoryError");
  Py_DECREF(torch);
  if (!g_oom) return nullptr;
  return PyModule_Create(&g_module);
}
