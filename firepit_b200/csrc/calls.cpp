// The paged cache's calls (firepit_b200/paged.py) without Python's share of them: a
// decode step's calls take a few microseconds each on the GPU, and the checks of ten
// tensors and thirty arguments through ctypes 8 to 11.
//
// A function takes a call that is right in every respect and makes it on the current
// stream.  Anything else it leaves alone (NotImplemented): paged.py then checks
// again and says what is wrong.  Returns what the call returns, or the status of a call
// that the library refused.
#include <Python.h>
#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "firepit_b200.h"

namespace {

using at::Tensor;

// Plain tensors alone: a subclass may mean something else by its methods.
const Tensor *tensor(PyObject *o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

bool code_of(const Tensor &t, int *code) {
  if (t.scalar_type() == at::kFloat)
    *code = FPB_F32;
  else if (t.scalar_type() == at::kBFloat16)
    *code = FPB_BF16;
  else
    return false;
  return true;
}

// The device of a call: of its first tensor, and the current one.
struct Device {
  int index;
  explicit Device(const Tensor *t) : index(t && t->is_cuda() ? (int)t->get_device() : -1) {
    if (index >= 0 && index != (int)c10::cuda::current_device()) index = -1;
  }
  bool holds(const Tensor &t) const { return index >= 0 && t.is_cuda() && t.get_device() == index; }
  void *stream() const { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream(); }
};

// An optional argument: None, or a tensor on the device for which `good` holds.
template <typename Good>
bool optional(PyObject *o, const Device &dev, const Tensor **t, Good good) {
  *t = nullptr;
  if (o == Py_None) return true;
  *t = tensor(o);
  return *t && dev.holds(**t) && good(**t);
}

bool vector(const Tensor &t, at::ScalarType type, int64_t n) {
  return t.scalar_type() == type && t.dim() == 1 && t.size(0) == n && t.is_contiguous();
}
bool ints(PyObject *o, const Device &dev, int64_t n, const Tensor **t) {
  *t = tensor(o);
  return *t && dev.holds(**t) && vector(**t, at::kInt, n);
}

void *address(const Tensor *t) { return t ? t->data_ptr() : nullptr; }
template <typename P>
P *as(const Tensor *t) {
  return static_cast<P *>(address(t));
}

// [rows, heads, d], d contiguous.
struct Heads {
  int64_t row, head;
  bool of(const Tensor &t, int64_t n, int64_t h, int64_t d) {
    if (t.dim() != 3 || t.size(0) != n || t.size(1) != h || t.size(2) != d || t.stride(2) != 1) return false;
    row = n > 1 ? t.stride(0) : h * d;
    head = h > 1 ? t.stride(1) : d;
    return true;
  }
};

struct Pages {
  const Tensor *k, *v;
  int code;
  int64_t n, p, h, d, page, row, head;
  bool of(PyObject *k_pages, PyObject *v_pages) {
    k = tensor(k_pages);
    v = tensor(v_pages);
    if (!k || !v || k->dim() != 4 || !code_of(*k, &code) || v->scalar_type() != k->scalar_type() ||
        v->sizes() != k->sizes() || v->strides() != k->strides() || k->stride(3) != 1)
      return false;
    n = k->size(0), p = k->size(1), h = k->size(2), d = k->size(3);
    if (n < 1 || p < 1 || h < 1 || d < 16) return false;
    page = n > 1 ? k->stride(0) : p * h * d;
    row = p > 1 ? k->stride(1) : h * d;
    head = h > 1 ? k->stride(2) : d;
    const int64_t el = code == FPB_F32 ? 4 : 2;
    return d % 16 == 0 && d <= 256 && page >= d && row >= d && head >= d && (page | row | head) * el % 16 == 0;
  }
};

struct Table {
  const Tensor *t;
  int64_t pitch, batch, width;
  bool of(PyObject *o, const Device &dev) {
    t = tensor(o);
    if (!t || !dev.holds(*t) || t->dim() != 2 || t->scalar_type() != at::kInt) return false;
    batch = t->size(0), width = t->size(1);
    if (batch < 1 || width < 1 || (width > 1 && t->stride(1) != 1)) return false;
    pitch = batch > 1 ? t->stride(0) : width;
    return true;
  }
};

bool whole(PyObject *o, int64_t *x) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  *x = PyLong_AsLongLongAndOverflow(o, &over);
  return !over && *x >= 0;
}
bool real(PyObject *o, double *x) {
  if (PyFloat_CheckExact(o)) {
    *x = PyFloat_AS_DOUBLE(o);
    return true;
  }
  int64_t n;
  if (!whole(o, &n)) return false;
  *x = (double)n;
  return true;
}

Tensor empty(at::IntArrayRef shape, at::ScalarType type, const Device &dev) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(at::Device(at::kCUDA, (c10::DeviceIndex)dev.index)));
}

// n elements of a vector from `at` on: a tensor of its own over the same memory (a view
// through the dispatcher takes a microsecond).
Tensor part(const Tensor &t, int64_t at, int64_t n) {
  Tensor r = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(t.storage()), t.key_set(), t.dtype());
  r.unsafeGetTensorImpl()->set_storage_offset(at);
  r.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return r;
}

PyObject *leave() {
  Py_INCREF(Py_NotImplemented);
  return Py_NotImplemented;
}

struct WithoutGil {
  PyThreadState *state = PyEval_SaveThread();
  ~WithoutGil() { PyEval_RestoreThread(state); }
};
template <typename Call>
int without_gil(Call call) {
  WithoutGil released;
  return call();
}

// table, lengths, free, free_count, page_size
struct Tables {
  Device dev;
  Table table;
  const Tensor *lengths, *free, *free_count;
  int64_t page_size;
  explicit Tables(PyObject *const *a) : dev(tensor(a[0])) {}
  bool of(PyObject *const *a) {
    if (!table.of(a[0], dev) || !ints(a[1], dev, table.batch, &lengths) || !whole(a[4], &page_size) || page_size < 1)
      return false;
    free = tensor(a[2]);
    return free && dev.holds(*free) && free->numel() > 0 && vector(*free, at::kInt, free->numel()) &&
           ints(a[3], dev, 1, &free_count);
  }
};

// (tables..., counts, rows, padded, slots, positions, requests, starts): the last four
// all None, or as PageMap holds them
PyObject *page_extend(PyObject *, PyObject *const *a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 12) return leave();
  Tables t(a);
  const Tensor *counts, *out[4];
  int64_t rows;
  if (!t.of(a) || !ints(a[5], t.dev, t.table.batch, &counts) || !whole(a[6], &rows) || rows < 1 ||
      rows > FPB_PAGE_MAX_ROWS || !PyBool_Check(a[7]))
    return leave();
  const bool padded = a[7] == Py_True, fresh = a[8] == Py_None;
  const int64_t b = t.table.batch;
  if (padded && rows % b) return leave();
  Tensor made[4];
  if (fresh) {
    // one allocation: three rows of a multiple of four, and the starts
    if (a[9] != Py_None || a[10] != Py_None || a[11] != Py_None) return leave();
    const int64_t up = (rows + 3) / 4 * 4;
    const Tensor flat = empty({3 * up + b + 1}, at::kInt, t.dev);
    for (int i = 0; i < 4; ++i) {
      made[i] = part(flat, i * up, i < 3 ? rows : b + 1);
      out[i] = &made[i];
    }
  } else {
    for (int i = 0; i < 4; ++i)
      if (!optional(a[8 + i], t.dev, &out[i], [&](const Tensor &x) { return vector(x, at::kInt, i < 3 ? rows : b + 1); }) ||
          (i < 2 && !out[i]))
        return leave();
  }
  void *stream = t.dev.stream();
  const int status = without_gil([&] {
    return fpb_page_extend(as<int32_t>(t.table.t), t.table.pitch, b, t.table.width, as<int32_t>(t.lengths),
                           as<int32_t>(counts), as<int32_t>(t.free), as<int32_t>(t.free_count), t.free->numel(),
                           t.page_size, rows, padded, as<int32_t>(out[0]), as<int32_t>(out[1]), as<int32_t>(out[2]),
                           as<int32_t>(out[3]), stream);
  });
  if (status) return PyLong_FromLong(status);
  if (!fresh) Py_RETURN_NONE;
  PyObject *r = PyTuple_New(4);
  if (!r) return nullptr;
  for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(made[i]));
  return r;
  END_HANDLE_TH_ERRORS
}

// (tables..., lengths)
PyObject *page_truncate(PyObject *, PyObject *const *a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 6) return leave();
  Tables t(a);
  const Tensor *to;
  if (!t.of(a) || !ints(a[5], t.dev, t.table.batch, &to)) return leave();
  void *stream = t.dev.stream();
  const int status = without_gil([&] {
    return fpb_page_truncate(as<int32_t>(t.table.t), t.table.pitch, t.table.batch, t.table.width, as<int32_t>(t.lengths),
                             as<int32_t>(to), as<int32_t>(t.free), as<int32_t>(t.free_count), t.free->numel(),
                             t.page_size, stream);
  });
  if (status) return PyLong_FromLong(status);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// (k pages, v pages, slots, positions, k, v, q, q_gamma, k_gamma, eps, rotary_dim, theta, q_out)
PyObject *paged_append(PyObject *, PyObject *const *a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 13) return leave();
  Pages c;
  if (!c.of(a[0], a[1])) return leave();
  const Device dev(c.k);
  const Tensor *slots, *positions, *k = tensor(a[4]), *v = tensor(a[5]), *q, *q_gamma, *k_gamma, *q_out;
  if (!k || !v || !dev.holds(*c.v) || !dev.holds(*k) || !dev.holds(*v) || k->dim() != 3) return leave();
  const int64_t n = k->size(0);
  int code, out_code = 0;
  Heads hk, hv, hq{0, 0};
  if (n < 1 || !code_of(*k, &code) || v->scalar_type() != k->scalar_type() || !hk.of(*k, n, c.h, c.d) ||
      !hv.of(*v, n, c.h, c.d) || hk.head != c.d || hv.head != c.d || !ints(a[2], dev, n, &slots) ||
      !ints(a[3], dev, n, &positions))
    return leave();
  auto gamma = [&](const Tensor &g) { return vector(g, at::kFloat, c.d); };
  int64_t q_heads = 0, rotary_dim;
  if (!optional(a[6], dev, &q, [&](const Tensor &x) {
        return x.dim() == 3 && x.scalar_type() == k->scalar_type() && (q_heads = x.size(1)) > 0 &&
               hq.of(x, n, q_heads, c.d);
      }) || !optional(a[7], dev, &q_gamma, gamma) || !optional(a[8], dev, &k_gamma, gamma) ||
      !optional(a[12], dev, &q_out, [&](const Tensor &x) {
        return q && x.sizes() == q->sizes() && x.is_contiguous() && code_of(x, &out_code);
      }))
    return leave();
  double eps, theta;
  if (!real(a[9], &eps) || !whole(a[10], &rotary_dim) || !real(a[11], &theta)) return leave();
  Tensor made;
  if (q && !q_out) {
    made = empty(q->sizes(), q->scalar_type(), dev);
    out_code = code;
  }
  void *stream = dev.stream();
  const int status = without_gil([&] {
    return fpb_paged_append(address(q), hq.row, hq.head, address(k), hk.row, address(v), hv.row, code,
                            as<float>(q_gamma), as<float>(k_gamma), as<int32_t>(slots), as<int32_t>(positions), n,
                            q_heads, c.h, c.d, rotary_dim, (float)theta, (float)eps,
                            made.defined() ? made.data_ptr() : address(q_out), out_code, address(c.k), address(c.v),
                            c.code, c.n, c.p, c.page, c.row, c.head, stream);
  });
  if (status) return PyLong_FromLong(status);
  if (!q) Py_RETURN_NONE;
  return THPVariable_Wrap(made.defined() ? made : *q_out);
  END_HANDLE_TH_ERRORS
}

// (q, k pages, v pages, table, lengths, gate, scale, out, workspace)
PyObject *paged_attention(PyObject *, PyObject *const *a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 9) return leave();
  Pages c;
  if (!c.of(a[1], a[2])) return leave();
  const Device dev(c.k);
  const Tensor *q = tensor(a[0]), *lengths, *gate, *out, *workspace;
  Table table;
  if (!q || !dev.holds(*c.v) || !dev.holds(*q) || q->dim() != 3 || !table.of(a[3], dev)) return leave();
  const int64_t b = q->size(0), h = q->size(1);
  int q_code, out_code = c.code;
  Heads hq, hg{0, 0};
  if (b < 1 || h < 1 || h % c.h || table.batch != b || !code_of(*q, &q_code) || !hq.of(*q, b, h, c.d) ||
      !ints(a[4], dev, b, &lengths) ||
      !optional(a[5], dev, &gate, [&](const Tensor &x) { return x.scalar_type() == at::kFloat && hg.of(x, b, h, c.d); }) ||
      !optional(a[7], dev, &out, [&](const Tensor &x) {
        return x.sizes() == q->sizes() && x.is_contiguous() && code_of(x, &out_code);
      }) ||
      !optional(a[8], dev, &workspace, [&](const Tensor &x) { return x.scalar_type() == at::kByte && x.is_contiguous(); }))
    return leave();
  double scale;
  if (a[6] == Py_None)
    scale = 1.0 / std::sqrt((double)c.d);
  else if (!real(a[6], &scale))
    return leave();
  Tensor space, made;
  if (!workspace) space = empty({(int64_t)fpb_paged_attn_workspace_bytes(b, h, c.h, c.d)}, at::kByte, dev);
  if (!out) made = empty({b, h, c.d}, c.k->scalar_type(), dev);
  const Tensor *w = workspace ? workspace : &space, *to = out ? out : &made;
  void *stream = dev.stream();
  const int status = without_gil([&] {
    return fpb_paged_attn(address(q), q_code, hq.row, hq.head, address(c.k), address(c.v), c.code, c.n, c.p, c.page, c.row,
                          c.head, as<int32_t>(table.t), table.pitch, table.width, as<int32_t>(lengths), as<float>(gate),
                          hg.row, hg.head, b, h, c.h, c.d, (float)scale, address(w), w->numel(), address(to), out_code,
                          stream);
  });
  return status ? PyLong_FromLong(status) : THPVariable_Wrap(*to);
  END_HANDLE_TH_ERRORS
}

// (logits, temperature, noise, top_k, top_p, min_p, logprobs, out)
PyObject *sample(PyObject *, PyObject *const *a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 8) return leave();
  const Tensor *logits = tensor(a[0]), *noise = tensor(a[2]), *row[3], *top_k, *out;
  const Device dev(logits);
  int code;
  if (!logits || !noise || !dev.holds(*logits) || !dev.holds(*noise) || logits->dim() != 2 || !code_of(*logits, &code) ||
      noise->scalar_type() != at::kFloat || noise->sizes() != logits->sizes() || !PyBool_Check(a[6]))
    return leave();
  const int64_t b = logits->size(0), vocab = logits->size(1);
  if (b < 1 || vocab < 1 || (vocab > 1 && (logits->stride(1) != 1 || noise->stride(1) != 1))) return leave();
  auto floats = [&](const Tensor &x) { return vector(x, at::kFloat, b); };
  auto whole_ones = [&](const Tensor &x) { return vector(x, at::kInt, b); };
  if (!optional(a[1], dev, &row[0], floats) || !optional(a[3], dev, &top_k, whole_ones) ||
      !optional(a[4], dev, &row[1], floats) || !optional(a[5], dev, &row[2], floats) ||
      !optional(a[7], dev, &out, whole_ones))
    return leave();
  Tensor tokens, logs;
  if (!out) tokens = empty({b}, at::kInt, dev);
  if (a[6] == Py_True) logs = empty({b}, at::kFloat, dev);
  const Tensor *to = out ? out : &tokens;
  void *stream = dev.stream();
  const int status = without_gil([&] {
    return fpb_sample(address(logits), code, b > 1 ? logits->stride(0) : vocab, as<float>(row[0]), as<int32_t>(top_k),
                      as<float>(row[1]), as<float>(row[2]), as<float>(noise), b > 1 ? noise->stride(0) : vocab, b, vocab,
                      as<int32_t>(to), logs.defined() ? static_cast<float *>(logs.data_ptr()) : nullptr, stream);
  });
  if (status) return PyLong_FromLong(status);
  if (!logs.defined()) return THPVariable_Wrap(*to);
  PyObject *r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(*to));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(logs));
  return r;
  END_HANDLE_TH_ERRORS
}

template <PyObject *(*F)(PyObject *, PyObject *const *, Py_ssize_t)>
PyMethodDef method(const char *name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(F)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<page_extend>("page_extend"),
                         method<page_truncate>("page_truncate"),
                         method<paged_append>("paged_append"),
                         method<paged_attention>("paged_attention"),
                         method<sample>("sample"),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// Torch's tensors are read by the layout that this was compiled for: "<torch's version>
// <Python's cache tag>", or the import fails.
PyMODINIT_FUNC PyInit__calls() {
  PyObject *torch = PyImport_ImportModule("torch"), *sys = PyImport_ImportModule("sys");
  PyObject *version = torch ? PyObject_GetAttrString(torch, "__version__") : nullptr;
  PyObject *python = sys ? PyObject_GetAttrString(sys, "implementation") : nullptr;
  PyObject *tag = python ? PyObject_GetAttrString(python, "cache_tag") : nullptr;
  PyObject *here = version && tag ? PyUnicode_FromFormat("%S %S", version, tag) : nullptr, *made = nullptr;
  if (here && PyUnicode_CompareWithASCIIString(here, FPB_CALLS_FOR) == 0)
    made = PyModule_Create(&module);
  else if (here)
    PyErr_Format(PyExc_ImportError, "_calls is built for \"%s\", this is \"%U\"", FPB_CALLS_FOR, here);
  for (PyObject *o : {torch, sys, version, python, tag, here}) Py_XDECREF(o);
  return made;
}
