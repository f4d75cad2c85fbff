// Calls of the 8-bit cache, the 8- and 4-bit linears and the token log probabilities from torch tensors, without Python
// between the checks and the library.
//
// A decode step's kernels take 5 to 8 us; checking their tensors attribute by attribute in Python and packing the
// C call's arguments took 13 to 18. Each function here looks at its arguments, allocates the result and the workspace
// and calls the C ABI (6 to 8 us in all, a launch included). What it does not recognise as a plain call it leaves alone: it returns None,
// and the Python function goes through its own checks, which say what is wrong or arrange what can be (a copy of
// strided rows, another stride of a table). A failed C call comes back as its status.
#include <dlfcn.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/torch.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <exception>
#include <type_traits>
#include <vector>

#include "../../include/ftx.h"

namespace {

using at::Tensor;

// The entries of the one library that the process has loaded, from wherever it came: linked to the binding they would
// be those of the library beside it, a second one with streams and buffers of its own.
struct Library {
  decltype(&ftx_kv8_append) kv8_append;
  decltype(&ftx_kv8_attention_workspace) kv8_attention_workspace;
  decltype(&ftx_kv8_attention) kv8_attention;
  decltype(&ftx_kv8_copy_pages) kv8_copy_pages;
  decltype(&ftx_int8_linear_workspace) int8_linear_workspace;
  decltype(&ftx_int8_linear) int8_linear;
  decltype(&ftx_int8_matmul_workspace) int8_matmul_workspace;
  decltype(&ftx_int8_matmul) int8_matmul;
  decltype(&ftx_kv8_append_norm) kv8_append_norm;
  decltype(&ftx_kv8_tree_attention_workspace) kv8_tree_attention_workspace;
  decltype(&ftx_kv8_tree_attention) kv8_tree_attention;
  decltype(&ftx_kv8_keep) kv8_keep;
  decltype(&ftx_int4_linear_workspace) int4_linear_workspace;
  decltype(&ftx_int4_linear) int4_linear;
  decltype(&ftx_token_logprobs_workspace) token_logprobs_workspace;
  decltype(&ftx_token_logprobs) token_logprobs;
};
Library lib{};

// The tensor behind an exact torch.Tensor or Parameter on `device` of this type, or nullptr: a subclass or a proxy is
// not plain memory.
const Tensor *plain(PyObject *o, int64_t device, at::ScalarType type) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const Tensor &t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.get_device() != device || t.scalar_type() != type) return nullptr;
  return &t;
}

const Tensor *operand(PyObject *o, int64_t device, at::ScalarType type) {  // that no gradient is asked for
  const Tensor *t = plain(o, device, type);
  return t && !(t->requires_grad() && at::GradMode::is_enabled()) ? t : nullptr;
}

bool aligned(const Tensor &t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// Strides of a [batch, token, head, d] operand read 16 bytes at a time.
bool heads(const Tensor *t, int64_t *stride) {
  if (!t || t->dim() != 4 || t->stride(3) != 1 || !aligned(*t)) return false;
  for (int i = 0; i < 3; ++i) {
    stride[i] = t->size(i) > 1 ? t->stride(i) : 0;
    if (stride[i] < 0 || stride[i] % 8 != 0) return false;
  }
  return true;
}

struct Cache {
  ftx_kv8_cache c{};
  const Tensor *codes, *scales;
};

// None, or a whole number that is not negative.
bool whole(PyObject *o, int64_t *out) {
  if (o == Py_None) return true;
  if (!PyLong_CheckExact(o)) return false;
  *out = PyLong_AsLongLong(o);
  if (*out >= 0) return true;
  PyErr_Clear();
  return false;
}

bool ints(PyObject *o, int64_t device, int64_t batch, const Tensor **out) {
  const Tensor *t = plain(o, device, at::kInt);
  if (!t || t->dim() != 1 || t->size(0) != batch || !t->is_contiguous()) return false;
  *out = t;
  return true;
}

// codes, scales, table, starts and new, for queries `q`.
bool cache(PyObject *const *args, const Tensor &q, int64_t device, Cache *out) {
  out->codes = plain(args[0], device, at::kChar);
  const bool e4m3 = !out->codes;
  if (e4m3) out->codes = operand(args[0], device, at::kFloat8_e4m3fn);
  out->scales = operand(args[1], device, at::kFloat);
  const Tensor *table = plain(args[2], device, at::kInt), *starts = nullptr, *news = nullptr;
  if (!out->codes || !out->scales || !table) return false;
  const Tensor &codes = *out->codes, &scales = *out->scales;
  const int64_t batch = q.size(0), d = q.size(3);
  if (codes.dim() != 5 || scales.dim() != 4 || !codes.is_contiguous() || !scales.is_contiguous() || !aligned(codes) ||
      !aligned(scales) || codes.size(1) != 2 || codes.size(4) != FTX_KV8_BLOCK * d || codes.size(2) < 1 ||
      q.size(2) % codes.size(2) != 0)
    return false;
  for (int i = 0; i < 4; ++i)
    if (codes.size(i) != scales.size(i)) return false;
  if (table->dim() != 2 || table->size(0) != batch || !table->is_contiguous() || !ints(args[3], device, batch, &starts))
    return false;
  if (args[4] != Py_None && !ints(args[4], device, batch, &news)) return false;
  const int64_t kMost = int64_t(1) << 30;
  if (table->size(1) > kMost || codes.size(2) > kMost || codes.size(3) > kMost / FTX_KV8_BLOCK) return false;
  out->c.codes = codes.data_ptr();
  out->c.scales = scales.data_ptr<float>();
  out->c.pages = codes.size(0);
  out->c.table = table->data_ptr<int32_t>();
  out->c.table_stride = table->size(1);
  out->c.starts = starts->data_ptr<int32_t>();
  out->c.news = news ? news->data_ptr<int32_t>() : nullptr;
  out->c.width = static_cast<int>(table->size(1));
  out->c.kv_heads = static_cast<int>(codes.size(2));
  out->c.page_tokens = static_cast<int>(codes.size(3)) * FTX_KV8_BLOCK;
  out->c.d = static_cast<int>(d);
  out->c.format = e4m3 ? FTX_KV8_E4M3 : FTX_KV8_INT8;
  return true;
}

void written(const Tensor &t) {  // as an in-place operation, for what autograd saved
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

PyObject *other_way() { Py_RETURN_NONE; }

// Arguments that the C entry refuses are for the Python checks to name.
PyObject *status(int rc) { return rc == FTX_ERR_INVALID ? other_way() : PyLong_FromLong(rc); }

PyObject *result(int rc, Tensor out) { return rc == FTX_OK ? THPVariable_Wrap(std::move(out)) : status(rc); }

int64_t device_of(PyObject *o) {  // -1, which no GPU's tensor has, for what is no number
  const int64_t device = PyLong_AsLong(o);
  PyErr_Clear();
  return device;
}

void *stream_of(PyObject *o) { return PyLong_AsVoidPtr(o); }

template <typename F>
PyObject *guarded(F f) {
  try {
    if (lib.kv8_append) return f();
    PyErr_SetString(PyExc_RuntimeError, "the binding has no library yet (use)");
    return nullptr;
  } catch (...) {  // as the Python type that torch gives it: memory that ran out is torch.OutOfMemoryError
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
}

// (q, k, v, cos, sin, codes, scales, table, starts, new, [positions, q norm, k norm, eps,] device, stream) -> rotated
// queries
PyObject *append(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (n != 12 && n != 16) return other_way();
    const int64_t device = device_of(a[n - 2]);
    int64_t stride[9];
    const Tensor *x[3];
    for (int i = 0; i < 3; ++i) {
      x[i] = operand(a[i], device, at::kBFloat16);
      if (!heads(x[i], stride + 3 * i)) return other_way();
    }
    const Tensor &q = *x[0];
    const Tensor *cos = operand(a[3], device, at::kFloat), *sin = operand(a[4], device, at::kFloat);
    Cache c;
    if (!cos || !sin || cos->dim() != 2 || cos->size(1) != q.size(3) || !cos->sizes().equals(sin->sizes()) ||
        !cos->is_contiguous() || !sin->is_contiguous() || !aligned(*cos) || !aligned(*sin) ||
        !cache(a + 5, q, device, &c))
      return other_way();
    for (int i = 1; i < 3; ++i)
      if (x[i]->size(0) != q.size(0) || x[i]->size(1) != q.size(1) || x[i]->size(2) != c.c.kv_heads ||
          x[i]->size(3) != q.size(3))
        return other_way();
    const Tensor *positions = nullptr, *weight[2] = {nullptr, nullptr};
    double eps = 0.0;
    int64_t apart = q.size(1);
    if (n == 16) {
      if (a[10] != Py_None) {
        positions = plain(a[10], device, at::kInt);
        if (!positions || positions->dim() != 2 || positions->size(0) != q.size(0) || positions->size(1) != q.size(1) ||
            (q.size(1) > 1 && positions->stride(1) != 1) || (q.size(0) > 1 && positions->stride(0) < q.size(1)))
          return other_way();
        if (q.size(0) > 1) apart = positions->stride(0);
      }
      if ((a[11] == Py_None) != (a[12] == Py_None)) return other_way();
      for (int i = 0; i < 2 && a[11] != Py_None; ++i) {
        weight[i] = operand(a[11 + i], device, at::kBFloat16);
        if (!weight[i] || weight[i]->dim() != 1 || weight[i]->size(0) != q.size(3) || !weight[i]->is_contiguous() ||
            !aligned(*weight[i]))
          return other_way();
      }
      eps = PyFloat_AsDouble(a[13]);
      if (PyErr_Occurred()) {
        PyErr_Clear();
        return other_way();
      }
    }
    Tensor out = at::empty(q.sizes(), q.options().requires_grad(false));
    written(*c.codes);
    written(*c.scales);
    int rc;
    if (n == 12)
      rc = lib.kv8_append(&c.c, q.data_ptr(), x[1]->data_ptr(), x[2]->data_ptr(), cos->data_ptr<float>(),
                          sin->data_ptr<float>(), cos->size(0), out.data_ptr(), q.size(0), q.size(1),
                          static_cast<int>(q.size(2)), stride, stream_of(a[11]));
    else
      rc = lib.kv8_append_norm(&c.c, q.data_ptr(), x[1]->data_ptr(), x[2]->data_ptr(),
                               weight[0] ? weight[0]->data_ptr() : nullptr, weight[1] ? weight[1]->data_ptr() : nullptr,
                               static_cast<float>(eps), cos->data_ptr<float>(), sin->data_ptr<float>(), cos->size(0),
                               positions ? positions->data_ptr<int32_t>() : nullptr, apart, out.data_ptr(), q.size(0),
                               q.size(1), static_cast<int>(q.size(2)), stride, stream_of(a[15]));
    return result(rc, std::move(out));
  });
}

// The attention of `q` over a cache from max tokens, scale, device and stream on; with the rows' sets of nodes over a
// tree.
PyObject *attend(const Tensor &q, int64_t *stride, const Cache &c, const Tensor *tree, int64_t tree_stride, int nodes,
                 PyObject *const *a) {
  int64_t longest = static_cast<int64_t>(c.c.width) * c.c.page_tokens, most = longest;
  if (!whole(a[0], &most)) return other_way();
  longest = std::min(longest, most);
  double scale = 1.0 / std::sqrt(static_cast<double>(q.size(3)));
  if (a[1] != Py_None) {
    scale = PyFloat_AsDouble(a[1]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      return other_way();
    }
  }
  Tensor out = at::empty_like(q);
  if (!heads(&out, stride + 3)) return other_way();
  const int h = static_cast<int>(q.size(2));
  size_t bytes = 0;
  int rc = (tree ? lib.kv8_tree_attention_workspace : lib.kv8_attention_workspace)(q.size(0), q.size(1), h, c.c.kv_heads,
                                                                                  c.c.d, longest, &bytes);
  if (rc != FTX_OK) return result(rc, out);
  Tensor ws;
  if (bytes > 0) ws = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte).requires_grad(false));
  void *scratch = bytes > 0 ? ws.data_ptr() : nullptr;
  if (tree)
    rc = lib.kv8_tree_attention(&c.c, q.data_ptr(), out.data_ptr(), tree->data_ptr<int64_t>(), tree_stride, nodes,
                                q.size(0), q.size(1), h, stride, static_cast<float>(scale), longest, scratch, bytes,
                                stream_of(a[3]));
  else
    rc = lib.kv8_attention(&c.c, q.data_ptr(), out.data_ptr(), q.size(0), q.size(1), h, stride,
                           static_cast<float>(scale), longest, scratch, bytes, stream_of(a[3]));
  return result(rc, std::move(out));
}

// (q, codes, scales, table, starts, new, max tokens, scale, device, stream) -> attended values
PyObject *attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (n != 10) return other_way();
    const int64_t device = device_of(a[8]);
    const Tensor *q = operand(a[0], device, at::kBFloat16);
    int64_t stride[6];
    Cache c;
    if (!heads(q, stride) || !cache(a + 1, *q, device, &c)) return other_way();
    return attend(*q, stride, c, nullptr, 0, 0, a + 6);
  });
}

// (q, codes, scales, table, starts, tree, new, nodes, max tokens, scale, device, stream) -> attended values
PyObject *tree_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (n != 12) return other_way();
    const int64_t device = device_of(a[10]);
    const Tensor *q = operand(a[0], device, at::kBFloat16);
    int64_t stride[6];
    Cache c;
    PyObject *const of_cache[5] = {a[1], a[2], a[3], a[4], a[6]};
    if (!heads(q, stride) || !cache(of_cache, *q, device, &c)) return other_way();
    const Tensor *tree = plain(a[5], device, at::kLong);
    int64_t nodes = q->size(1);
    if (!tree || tree->dim() != 2 || tree->size(0) != q->size(0) || tree->size(1) != q->size(1) || !whole(a[7], &nodes) ||
        nodes > 64)
      return other_way();
    const int64_t apart = tree->size(0) > 1 ? tree->stride(0) : tree->size(1);
    if ((apart != 0 && apart < tree->size(1)) || (tree->size(1) > 1 && tree->stride(1) != 1)) return other_way();
    return attend(*q, stride, c, tree, apart, static_cast<int>(nodes), a + 8);
  });
}

// (codes, scales, table, starts, path, counts, device, stream) -> True
PyObject *keep(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (n != 8) return other_way();
    const int64_t device = device_of(a[6]);
    const Tensor *codes = plain(a[0], device, at::kChar), *scales = operand(a[1], device, at::kFloat);
    const bool e4m3 = !codes;
    if (e4m3) codes = operand(a[0], device, at::kFloat8_e4m3fn);
    const Tensor *table = plain(a[2], device, at::kInt), *path = plain(a[4], device, at::kInt), *starts, *counts = nullptr;
    if (!codes || !scales || !table || !path || codes->dim() != 6 || scales->dim() != 5 || !codes->is_contiguous() ||
        !scales->is_contiguous() || !aligned(*codes) || !aligned(*scales) || codes->size(2) != 2 || path->dim() != 2 ||
        !path->is_contiguous() || table->dim() != 2 || !table->is_contiguous() || codes->size(0) < 1)
      return other_way();
    for (int i = 0; i < 5; ++i)
      if (codes->size(i) != scales->size(i)) return other_way();
    const int64_t batch = path->size(0), d = codes->size(5) / FTX_KV8_BLOCK, kMost = int64_t(1) << 30;
    if (table->size(0) != batch || !ints(a[3], device, batch, &starts) ||
        (a[5] != Py_None && !ints(a[5], device, batch, &counts)) || table->size(1) > kMost || codes->size(3) > kMost ||
        codes->size(4) > kMost / FTX_KV8_BLOCK || (d != 64 && d != 128) || codes->size(5) % FTX_KV8_BLOCK != 0)
      return other_way();
    ftx_kv8_cache c{};
    c.codes = codes->data_ptr();
    c.scales = scales->data_ptr<float>();
    c.pages = codes->size(1);
    c.table = table->data_ptr<int32_t>();
    c.table_stride = table->size(1);
    c.starts = starts->data_ptr<int32_t>();
    c.news = counts ? counts->data_ptr<int32_t>() : nullptr;
    c.width = static_cast<int>(table->size(1));
    c.kv_heads = static_cast<int>(codes->size(3));
    c.page_tokens = static_cast<int>(codes->size(4)) * FTX_KV8_BLOCK;
    c.d = static_cast<int>(d);
    c.format = e4m3 ? FTX_KV8_E4M3 : FTX_KV8_INT8;
    const int rc = lib.kv8_keep(&c, codes->size(0), path->data_ptr<int32_t>(), path->size(1), batch, path->size(1),
                                stream_of(a[7]));
    if (rc != FTX_OK) return status(rc);
    written(*codes);
    written(*scales);
    Py_RETURN_TRUE;
  });
}

// (codes, scales, source pages, target pages, device, stream) -> True
PyObject *copy_pages(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (n != 6 || !PyList_CheckExact(a[2]) || !PyList_CheckExact(a[3])) return other_way();
    const int64_t device = device_of(a[4]);
    const Tensor *codes = plain(a[0], device, at::kChar), *scales = operand(a[1], device, at::kFloat);
    if (!codes) codes = operand(a[0], device, at::kFloat8_e4m3fn);
    if (!codes || !scales || codes->dim() != 6 || scales->dim() != 5 || !codes->is_contiguous() ||
        !scales->is_contiguous() || !aligned(*codes) || !aligned(*scales) || codes->size(2) != 2)
      return other_way();
    for (int i = 0; i < 5; ++i)
      if (codes->size(i) != scales->size(i)) return other_way();
    const int64_t kMost = int64_t(1) << 30;
    const int64_t d = codes->size(5) / FTX_KV8_BLOCK;
    if (codes->size(3) > kMost || codes->size(4) > kMost / FTX_KV8_BLOCK || (d != 64 && d != 128) ||
        codes->size(5) % FTX_KV8_BLOCK != 0)
      return other_way();
    const Py_ssize_t count = PyList_GET_SIZE(a[2]);
    if (PyList_GET_SIZE(a[3]) != count) return other_way();
    std::vector<int32_t> pages[2];
    for (int side = 0; side < 2; ++side) {
      pages[side].reserve(count);
      for (Py_ssize_t i = 0; i < count; ++i) {
        PyObject *o = PyList_GET_ITEM(a[2 + side], i);
        if (!PyLong_CheckExact(o)) return other_way();
        const long v = PyLong_AsLong(o);
        if (v < 0 || v >= codes->size(1)) {
          PyErr_Clear();
          return other_way();
        }
        pages[side].push_back(static_cast<int32_t>(v));
      }
    }
    written(*codes);
    written(*scales);
    const int rc = lib.kv8_copy_pages(codes->data_ptr(), scales->data_ptr<float>(), codes->size(0), codes->size(1),
                                      static_cast<int>(codes->size(3)), static_cast<int>(codes->size(4)) * FTX_KV8_BLOCK,
                                      static_cast<int>(d), pages[0].data(), pages[1].data(), count, stream_of(a[5]));
    if (rc != FTX_OK) return status(rc);
    Py_RETURN_TRUE;
  });
}

// An int8 weight [n, k] and its fp32 scale [n].
bool weight(PyObject *w, PyObject *s, int64_t device, int64_t k, const Tensor **wt, const Tensor **st) {
  *wt = plain(w, device, at::kChar);
  *st = operand(s, device, at::kFloat);
  return *wt && *st && (*wt)->dim() == 2 && (*wt)->size(1) == k && (*st)->dim() == 1 &&
         (*st)->size(0) == (*wt)->size(0) && (*wt)->is_contiguous() && (*st)->is_contiguous() && aligned(**wt) &&
         aligned(**st);
}

// (x, weight, scale, device, stream) -> y
PyObject *int8_linear(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (n != 5) return other_way();
    const int64_t device = device_of(a[3]);
    const Tensor *x = operand(a[0], device, at::kBFloat16), *w, *s;
    if (!x || x->dim() != 2 || !aligned(*x)) return other_way();
    const int64_t m = x->size(0), k = x->size(1), stride = m > 1 ? x->stride(0) : k;
    if (k == 0 || x->stride(1) != 1 || stride < k || stride % 8 != 0 || !weight(a[1], a[2], device, k, &w, &s))
      return other_way();
    const int64_t channels = w->size(0);
    size_t bytes = 0;
    int rc = lib.int8_linear_workspace(m, channels, k, &bytes);
    if (rc != FTX_OK) return other_way();
    Tensor y = at::empty({m, channels}, x->options().requires_grad(false));
    Tensor ws = at::empty({static_cast<int64_t>(bytes)}, x->options().dtype(at::kByte).requires_grad(false));
    rc = lib.int8_linear(x->data_ptr(), stride, w->data_ptr(), s->data_ptr<float>(), y.data_ptr(), m, channels, k,
                         ws.data_ptr(), bytes, stream_of(a[4]));
    return result(rc, std::move(y));
  });
}

// (codes, row scales, weight, scale, device, stream) -> y
PyObject *int8_matmul(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (n != 6) return other_way();
    const int64_t device = device_of(a[4]);
    const Tensor *c = plain(a[0], device, at::kChar), *r = operand(a[1], device, at::kFloat), *w, *s;
    const Tensor *shape = plain(a[2], device, at::kChar);
    if (!c || !r || !shape || shape->dim() != 2 || c->dim() != 2 || r->dim() != 1 || r->size(0) != c->size(0) ||
        !c->is_contiguous() || !r->is_contiguous() || !aligned(*c) || !aligned(*r))
      return other_way();
    const int64_t m = c->size(0), k = shape->size(1);
    if (k == 0 || c->size(1) != FTX_INT8_CODE_STRIDE(k) || !weight(a[2], a[3], device, k, &w, &s)) return other_way();
    const int64_t channels = w->size(0);
    size_t bytes = 0;
    int rc = lib.int8_matmul_workspace(m, channels, k, &bytes);
    if (rc != FTX_OK) return other_way();
    Tensor y = at::empty({m, channels}, c->options().dtype(at::kBFloat16)), ws;
    if (bytes > 0) ws = at::empty({static_cast<int64_t>(bytes)}, c->options().dtype(at::kByte));
    rc = lib.int8_matmul(c->data_ptr(), r->data_ptr<float>(), w->data_ptr(), s->data_ptr<float>(), y.data_ptr(), m,
                         channels, k, bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream_of(a[5]));
    return result(rc, std::move(y));
  });
}

// (x, weight, scale, zero, channels, device, stream) -> y
PyObject *int4_linear(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (n != 7) return other_way();
    const int64_t device = device_of(a[5]);
    const Tensor *x = operand(a[0], device, at::kBFloat16), *w = plain(a[1], device, at::kByte);
    const Tensor *s = operand(a[2], device, at::kBFloat16), *z = nullptr;
    if (a[3] != Py_None && !(z = operand(a[3], device, at::kBFloat16))) return other_way();
    if (!x || !w || !s || x->dim() != 2 || !aligned(*x) || w->dim() != 3 || s->dim() != 4 || !w->is_contiguous() ||
        !s->is_contiguous() || !aligned(*w) || !aligned(*s) || (z && (!z->is_contiguous() || !aligned(*z))))
      return other_way();
    const int64_t m = x->size(0), k = x->size(1), stride = m > 1 ? x->stride(0) : k, tiles = w->size(0);
    const int64_t parts = s->size(3);
    int64_t channels = tiles * FTX_INT4_TILE;
    if (k == 0 || x->stride(1) != 1 || stride < k || (parts != 1 && parts != 2 && parts != 4) ||
        w->size(1) != (k + FTX_INT4_UNIT - 1) / FTX_INT4_UNIT || w->size(2) != FTX_INT4_TILE * FTX_INT4_UNIT / 2 ||
        s->size(0) != tiles || s->size(1) != w->size(1) || s->size(2) != FTX_INT4_TILE ||
        (z && !z->sizes().equals(s->sizes())) || !whole(a[4], &channels) ||
        (channels + FTX_INT4_TILE - 1) / FTX_INT4_TILE != tiles)
      return other_way();
    const int group = static_cast<int>(FTX_INT4_UNIT / parts);
    size_t bytes = 0;
    int rc = lib.int4_linear_workspace(m, channels, k, group, &bytes);
    if (rc != FTX_OK) return other_way();
    Tensor y = at::empty({m, channels}, x->options().requires_grad(false)), ws;
    if (bytes > 0) ws = at::empty({static_cast<int64_t>(bytes)}, x->options().dtype(at::kByte).requires_grad(false));
    rc = lib.int4_linear(x->data_ptr(), stride, w->data_ptr(), s->data_ptr(), z ? z->data_ptr() : nullptr, y.data_ptr(), m,
                         channels, k, group, bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream_of(a[6]));
    return result(rc, std::move(y));
  });
}

// (logits, tokens, top, device, stream) -> (log probabilities, entropies, top log probabilities, top tokens)
PyObject *token_logprobs(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded([&]() -> PyObject * {
    if (n != 5) return other_way();
    const int64_t device = device_of(a[3]);
    int type = FTX_LOGITS_FP32;
    const Tensor *x = operand(a[0], device, at::kFloat), *tokens = plain(a[1], device, at::kLong);
    if (!x) {
      type = FTX_LOGITS_BF16;
      x = operand(a[0], device, at::kBFloat16);
    }
    if (!x) {
      type = FTX_LOGITS_FP16;
      x = operand(a[0], device, at::kHalf);
    }
    int64_t top = -1;
    if (!x || !tokens || x->dim() != 2 || tokens->dim() != 1 || tokens->size(0) != x->size(0) ||
        !tokens->is_contiguous() || x->stride(1) != 1 || x->size(1) == 0 || !whole(a[2], &top) || top < 0 || top > 64)
      return other_way();
    const int64_t rows = x->size(0), vocab = x->size(1);
    size_t bytes = 0;
    int rc = lib.token_logprobs_workspace(rows, vocab, type, static_cast<int>(top), &bytes);
    if (rc != FTX_OK) return other_way();
    const auto floats = x->options().dtype(at::kFloat).requires_grad(false);
    Tensor given = at::empty({rows}, floats), entropy = at::empty({rows}, floats), best = at::empty({rows, top}, floats);
    Tensor index = at::empty({rows, top}, tokens->options()), ws;
    if (bytes > 0) ws = at::empty({static_cast<int64_t>(bytes)}, floats.dtype(at::kByte));
    rc = lib.token_logprobs(x->data_ptr(), rows > 1 ? x->stride(0) : vocab, type, tokens->data_ptr<int64_t>(), rows, vocab,
                            static_cast<int>(top), given.data_ptr<float>(), entropy.data_ptr<float>(),
                            best.data_ptr<float>(), index.data_ptr<int64_t>(), bytes > 0 ? ws.data_ptr() : nullptr, bytes,
                            stream_of(a[4]));
    if (rc != FTX_OK) return status(rc);
    PyObject *out = PyTuple_New(4);
    if (!out) return nullptr;
    int i = 0;
    for (Tensor *t : {&given, &entropy, &best, &index}) {
      PyObject *o = THPVariable_Wrap(std::move(*t));
      if (!o) {
        Py_DECREF(out);
        return nullptr;
      }
      PyTuple_SET_ITEM(out, i++, o);
    }
    return out;
  });
}

template <PyObject *(*F)(PyObject *, PyObject *const *, Py_ssize_t)>
PyMethodDef method(const char *name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}

// (the loaded library's handle)
PyObject *use(PyObject *, PyObject *handle) {
  void *from = PyLong_AsVoidPtr(handle);
  if (!from) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "no library");
    return nullptr;
  }
  Library found{};
  const auto entry = [&](auto &to, const char *name) {
    to = reinterpret_cast<std::remove_reference_t<decltype(to)>>(dlsym(from, name));
    if (!to) PyErr_Format(PyExc_ImportError, "the library has no %s", name);
    return to != nullptr;
  };
  if (!entry(found.kv8_append, "ftx_kv8_append") ||
      !entry(found.kv8_attention_workspace, "ftx_kv8_attention_workspace") ||
      !entry(found.kv8_attention, "ftx_kv8_attention") || !entry(found.kv8_copy_pages, "ftx_kv8_copy_pages") ||
      !entry(found.int8_linear_workspace, "ftx_int8_linear_workspace") ||
      !entry(found.int8_linear, "ftx_int8_linear") ||
      !entry(found.int8_matmul_workspace, "ftx_int8_matmul_workspace") ||
      !entry(found.int8_matmul, "ftx_int8_matmul") || !entry(found.kv8_append_norm, "ftx_kv8_append_norm") ||
      !entry(found.kv8_tree_attention_workspace, "ftx_kv8_tree_attention_workspace") ||
      !entry(found.kv8_tree_attention, "ftx_kv8_tree_attention") || !entry(found.kv8_keep, "ftx_kv8_keep") ||
      !entry(found.int4_linear_workspace, "ftx_int4_linear_workspace") ||
      !entry(found.int4_linear, "ftx_int4_linear") ||
      !entry(found.token_logprobs_workspace, "ftx_token_logprobs_workspace") ||
      !entry(found.token_logprobs, "ftx_token_logprobs"))
    return nullptr;
  lib = found;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"use", use, METH_O, nullptr},
                         method<append>("append"),           method<attention>("attention"),
                         method<copy_pages>("copy_pages"),   method<int8_linear>("int8_linear"),
                         method<int8_matmul>("int8_matmul"), method<append>("append_norm"),
                         method<tree_attention>("tree_attention"), method<keep>("keep"),
                         method<int4_linear>("int4_linear"), method<token_logprobs>("token_logprobs"),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ftx_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ftx_torch() { return PyModule_Create(&module); }
