// The paged K/V cache's calls from Python on torch tensors: checks and argument
// blocks for chonk_kv_* (include/chonk.h). A step of a small model calls these a few
// dozen times a token, a few microseconds of device work each, so the host's share
// counts: through ctypes a call took 8 to 9 us, here 4 to 5 (3 of them the launch).
// chonklm_amd/paged_kv.py documents the class and adds what need not be fast.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <structmember.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstddef>
#include <stdexcept>
#include <string>

#include "chonk.h"

namespace {

PyObject* g_error = nullptr;   // chonklm_amd._lib.ChonkError(status, message)
PyObject* g_stream = nullptr;  // device index -> hipStream_t of torch's current stream, as an int
PyObject* g_f32 = nullptr;     // torch.float32
PyObject* g_f16 = nullptr;     // torch.float16

struct Refused {
  int status;
  std::string message;
};
[[noreturn]] void refuse(const std::string& m) { throw Refused{CHONK_EINVAL, "paged K/V cache: " + m}; }
struct PythonError {};  // a Python exception is set

template <class F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const Refused& e) {
    if (PyObject* x = PyObject_CallFunction(g_error, "is", e.status, e.message.c_str())) {
      PyErr_SetObject(g_error, x);
      Py_DECREF(x);
    }
  } catch (const PythonError&) {
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "paged K/V cache: unknown error");
  }
  return nullptr;
}

// Positional and keyword arguments into `out` (borrowed; null: not given).
void arguments(const char* what, PyObject* const* args, Py_ssize_t n, PyObject* kw, const char* const* names, int total,
               int positional, int required, PyObject** out) {
  if (n > positional) {
    PyErr_Format(PyExc_TypeError, "%s() takes at most %d positional arguments (%zd given)", what, positional, n);
    throw PythonError{};
  }
  for (int i = 0; i < total; ++i) out[i] = i < n ? args[i] : nullptr;
  const Py_ssize_t nk = kw ? PyTuple_GET_SIZE(kw) : 0;
  for (Py_ssize_t k = 0; k < nk; ++k) {
    PyObject* name = PyTuple_GET_ITEM(kw, k);
    int i = 0;
    while (i < total && PyUnicode_CompareWithASCIIString(name, names[i]) != 0) ++i;
    if (i == total || out[i]) {
      PyErr_Format(PyExc_TypeError, i == total ? "%s() got an unexpected keyword argument %R"
                                               : "%s() got multiple values for argument %R", what, name);
      throw PythonError{};
    }
    out[i] = args[n + k];
  }
  for (int i = 0; i < required; ++i)
    if (!out[i]) {
      PyErr_Format(PyExc_TypeError, "%s() missing argument '%s'", what, names[i]);
      throw PythonError{};
    }
}

const at::Tensor* tensor_or_none(PyObject* o, const char* name) {
  if (!o || o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a tensor", name);
    throw PythonError{};
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.requires_grad() && c10::GradMode::is_enabled())
    refuse(std::string(name) + " requires a gradient, and these operators have none");
  return &t;
}
const at::Tensor& tensor(PyObject* o, const char* name) {
  const at::Tensor* t = tensor_or_none(o, name);
  if (!t) refuse(std::string(name) + " is missing");
  return *t;
}
double number(PyObject* o, double otherwise) {
  if (!o || o == Py_None) return otherwise;
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PythonError{};
  return v;
}
int64_t integer(PyObject* o, int64_t otherwise) {
  if (!o || o == Py_None) return otherwise;
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PythonError{};
  return v;
}
bool truth(PyObject* o) {
  const int v = o ? PyObject_IsTrue(o) : 0;
  if (v < 0) throw PythonError{};
  return v != 0;
}
void status(int rc) {
  if (rc != CHONK_OK) throw Refused{rc, chonk_last_error()};
}

std::string dims(std::initializer_list<int64_t> d) {
  std::string s = "[";
  for (int64_t v : d) s += (s.size() > 1 ? ", " : "") + std::to_string(v);
  return s + "]";
}

struct Cache {
  PyObject_HEAD
  PyObject *pages, *table, *fault;
  chonk_kv_cache c;
  at::Device device;
};

void* stream_of(const Cache* k) {
  PyObject* at = PyLong_FromLong(k->c.device);
  PyObject* s = at ? PyObject_CallOneArg(g_stream, at) : nullptr;
  Py_XDECREF(at);
  if (!s) throw PythonError{};
  void* p = PyLong_AsVoidPtr(s);
  Py_DECREF(s);
  if (!p && PyErr_Occurred()) throw PythonError{};
  return p;
}

int act(const at::Tensor& t, const char* name) {
  const auto d = t.scalar_type();
  if (d == at::kFloat) return CHONK_F32;
  if (d == at::kHalf) return CHONK_F16;
  refuse(std::string(name) + " must be float32 or float16");
}

const int32_t* index(const Cache* k, const at::Tensor& t, int64_t n, const char* name) {
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != n || !t.is_contiguous() || t.device() != k->device)
    refuse(std::string(name) + " must be contiguous int32 " + dims({n}) + " on " + k->device.str());
  return (const int32_t*)t.data_ptr();
}

// Rows [n, heads, head_dim] of `type`, each contiguous; returns the elements from row to row.
int64_t rows(const Cache* k, const at::Tensor& t, int64_t n, int64_t heads, int type, const char* name) {
  const int64_t hd = k->c.head_dim;
  if (t.dim() != 3 || t.size(0) != n || t.size(1) != heads || t.size(2) != hd)
    refuse(std::string(name) + " must be " + dims({n, heads, hd}));
  if (act(t, name) != type) refuse(std::string(name) + " must be of the other rows' type");
  if (t.device() != k->device) refuse(std::string(name) + " must be on " + k->device.str());
  if (n == 0) return heads * hd;
  if (t.stride(2) != 1 || (heads > 1 && t.stride(1) != hd)) refuse(std::string("a row of ") + name + " must be contiguous");
  return n > 1 ? t.stride(0) : heads * hd;
}

const float* weights(const Cache* k, const at::Tensor* t, const char* name) {
  if (!t) return nullptr;
  if (t->scalar_type() != at::kFloat || t->dim() != 1 || t->size(0) != k->c.head_dim || !t->is_contiguous() ||
      t->device() != k->device)
    refuse(std::string(name) + " must be contiguous float32 " + dims({k->c.head_dim}) + " on " + k->device.str());
  return (const float*)t->data_ptr();
}

int32_t count(int64_t n) {
  if (n > INT32_MAX) refuse("too many rows");
  return (int32_t)n;
}

int cache_init(PyObject* self, PyObject* args, PyObject* kwargs) {
  static const char* names[] = {"pages", "table", "kv_heads", "head_dim", "kv_type", "fault", nullptr};
  PyObject *pages, *table, *fault = nullptr;
  long long heads, hd, type;
  if (!PyArg_ParseTupleAndKeywords(args, kwargs, "OOLLL|O", const_cast<char**>(names), &pages, &table, &heads, &hd, &type,
                                   &fault))
    return -1;
  PyObject* done = guarded([&]() -> PyObject* {
    Cache* k = (Cache*)self;
    const at::Tensor &p = tensor(pages, "pages"), &t = tensor(table, "table");
    const at::Tensor* f = tensor_or_none(fault, "fault");
    if (heads <= 0 || heads > INT32_MAX || hd <= 0 || hd > INT32_MAX || type < 0 || type > INT32_MAX) refuse("bad sizes");
    const int64_t size = chonk_kv_page_bytes((int32_t)type, (int32_t)heads, (int32_t)hd);
    if (size < 0) status((int)size);
    if (p.scalar_type() != at::kByte || p.dim() != 2 || p.size(1) != size || !p.is_contiguous())
      refuse("pages must be contiguous uint8 [n_pages, " + std::to_string(size) + "]");
    if (t.scalar_type() != at::kInt || t.dim() != 2 || !t.is_contiguous())
      refuse("table must be contiguous int32 [n_seqs, max_pages]");
    if (!p.is_cuda()) refuse("pages must be on a GPU");
    if (t.device() != p.device() || (f && f->device() != p.device())) refuse("table and fault must be on the pages' device");
    if (f && (f->scalar_type() != at::kInt || f->numel() != 1)) refuse("fault must be int32 [1]");
    k->c.kv_type = (int32_t)type;
    k->c.kv_heads = (int32_t)heads;
    k->c.head_dim = (int32_t)hd;
    k->c.n_pages = count(p.size(0));
    k->c.pages = p.data_ptr();
    k->c.n_seqs = count(t.size(0));
    k->c.max_pages = count(t.size(1));
    k->c.table = (const int32_t*)t.data_ptr();
    k->c.fault = f ? (int32_t*)f->data_ptr() : nullptr;
    k->c.device = p.device().index();
    k->device = p.device();
    PyObject* held[3] = {pages, table, f ? fault : Py_None};
    PyObject** at[3] = {&k->pages, &k->table, &k->fault};
    for (int i = 0; i < 3; ++i) {
      Py_INCREF(held[i]);
      Py_XSETREF(*at[i], held[i]);
    }
    Py_RETURN_NONE;
  });
  Py_XDECREF(done);
  return done ? 0 : -1;
}

PyObject* cache_new(PyTypeObject* type, PyObject*, PyObject*) {
  Cache* k = (Cache*)type->tp_alloc(type, 0);
  if (k) {
    k->pages = k->table = k->fault = nullptr;
    k->c = chonk_kv_cache{};
    new (&k->device) at::Device(at::kCPU);
  }
  return (PyObject*)k;
}
int cache_traverse(PyObject* self, visitproc visit, void* arg) {
  Cache* k = (Cache*)self;
  Py_VISIT(Py_TYPE(self));
  Py_VISIT(k->pages);
  Py_VISIT(k->table);
  Py_VISIT(k->fault);
  return 0;
}
int cache_clear(PyObject* self) {
  Cache* k = (Cache*)self;
  k->c = chonk_kv_cache{};  // (a later call is refused: an empty pool)
  Py_CLEAR(k->pages);
  Py_CLEAR(k->table);
  Py_CLEAR(k->fault);
  return 0;
}
void cache_dealloc(PyObject* self) {
  PyTypeObject* type = Py_TYPE(self);
  PyObject_GC_UnTrack(self);
  cache_clear(self);
  type->tp_free(self);
  Py_DECREF(type);
}

const Cache* made(PyObject* self) {
  const Cache* k = (const Cache*)self;
  if (!k->pages) refuse("the cache was not made");
  return k;
}

PyObject* cache_append(PyObject* self, PyObject* const* args, Py_ssize_t n_args, PyObject* kw) {
  return guarded([&]() -> PyObject* {
    static const char* names[] = {"q", "k", "v", "seqs", "positions", "q_norm", "k_norm", "eps", "rope", "interleaved", "out"};
    PyObject* x[11];
    arguments("append", args, n_args, kw, names, 11, 5, 5, x);
    const Cache* c = made(self);
    const at::Tensor *q = tensor_or_none(x[0], "q"), *out = tensor_or_none(x[10], "out"), *rope = tensor_or_none(x[8], "rope");
    const at::Tensor &k = tensor(x[1], "k"), &v = tensor(x[2], "v");
    const int64_t n = k.dim() ? k.size(0) : 0;
    chonk_kv_append_args a{};
    a.type = act(k, "k");
    a.k_stride = rows(c, k, n, c->c.kv_heads, a.type, "k");
    a.v_stride = rows(c, v, n, c->c.kv_heads, a.type, "v");
    const chonk_kv_rows r{count(n), index(c, tensor(x[3], "seqs"), n, "seqs"),
                          index(c, tensor(x[4], "positions"), n, "positions")};
    a.q_norm = weights(c, tensor_or_none(x[5], "q_norm"), "q_norm");
    a.k_norm = weights(c, tensor_or_none(x[6], "k_norm"), "k_norm");
    a.eps = number(x[7], 1e-6);
    if (rope) {
      if (rope->scalar_type() != at::kFloat || rope->dim() != 3 || rope->size(2) != 2 || !rope->is_contiguous() ||
          rope->device() != c->device)
        refuse("rope must be contiguous float32 [positions, rope_dim / 2, 2] on " + c->device.str());
      a.rope = (const float*)rope->data_ptr();
      a.rope_dim = count(2 * rope->size(1));
      a.rope_positions = count(rope->size(0));
    }
    a.interleaved = truth(x[9]);
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    at::Tensor result;
    if (q) {
      if (q->dim() != 3) refuse("q must be [n, heads, head_dim]");
      a.heads = count(q->size(1));
      a.q_stride = rows(c, *q, n, a.heads, a.type, "q");
      if (!out) {
        result = at::empty(q->sizes(), q->options());
        out = &result;
      }
      a.q_out_stride = rows(c, *out, n, a.heads, a.type, "out");
      a.q = q->data_ptr();
      a.q_out = out->data_ptr();
    } else if (out) {
      refuse("out without q");
    }
    status(chonk_kv_append(&c->c, &r, &a, stream_of(c)));
    if (!q) Py_RETURN_NONE;
    if (result.defined()) return THPVariable_Wrap(std::move(result));
    Py_INCREF(x[10]);
    return x[10];
  });
}

PyObject* cache_read(PyObject* self, PyObject* const* args, Py_ssize_t n_args, PyObject* kw) {
  return guarded([&]() -> PyObject* {
    static const char* names[] = {"seqs", "positions", "dtype"};
    PyObject* x[3];
    arguments("read", args, n_args, kw, names, 3, 3, 2, x);
    const Cache* c = made(self);
    const bool f32 = x[2] == g_f32;
    if (x[2] && !f32 && x[2] != g_f16) refuse("dtype must be float32 or float16");
    const at::Tensor& s = tensor(x[0], "seqs");
    const int64_t n = s.dim() ? s.size(0) : 0;
    const chonk_kv_rows r{count(n), index(c, s, n, "seqs"), index(c, tensor(x[1], "positions"), n, "positions")};
    const int64_t heads = c->c.kv_heads, hd = c->c.head_dim;
    const auto options = at::TensorOptions().dtype(f32 ? at::kFloat : at::kHalf).device(c->device);
    at::Tensor k = at::empty({n, heads, hd}, options), v = at::empty({n, heads, hd}, options);
    status(chonk_kv_read(&c->c, &r, f32 ? CHONK_F32 : CHONK_F16, k.data_ptr(), v.data_ptr(), heads * hd, hd, stream_of(c)));
    PyObject* pk = THPVariable_Wrap(std::move(k));
    PyObject* pv = pk ? THPVariable_Wrap(std::move(v)) : nullptr;
    if (!pv) {
      Py_XDECREF(pk);
      throw PythonError{};
    }
    PyObject* both = PyTuple_Pack(2, pk, pv);
    Py_DECREF(pk);
    Py_DECREF(pv);
    return both;
  });
}

PyObject* cache_attend(PyObject* self, PyObject* const* args, Py_ssize_t n_args, PyObject* kw) {
  return guarded([&]() -> PyObject* {
    static const char* names[] = {"q", "seqs", "lengths", "scale", "window", "out"};
    PyObject* x[6];
    arguments("attend", args, n_args, kw, names, 6, 3, 3, x);
    const Cache* c = made(self);
    const at::Tensor& q = tensor(x[0], "q");
    const at::Tensor* out = tensor_or_none(x[5], "out");
    if (q.dim() != 3) refuse("q must be [n, heads, head_dim]");
    const int64_t n = q.size(0), hd = c->c.head_dim;
    chonk_kv_attend_args a{};
    a.type = act(q, "q");
    a.heads = count(q.size(1));
    a.n = count(n);
    a.q_stride = rows(c, q, n, a.heads, a.type, "q");
    a.seq = index(c, tensor(x[1], "seqs"), n, "seqs");
    a.lengths = index(c, tensor(x[2], "lengths"), n, "lengths");
    const double least = 1.0 / std::sqrt((double)hd);
    a.scale = (float)number(x[3], least);
    const int64_t window = integer(x[4], 0);
    if (window < 0 || window > INT32_MAX) refuse("bad window " + std::to_string(window));
    a.window = (int32_t)window;
    a.workspace_bytes = chonk_kv_attend_workspace(&c->c, a.n, a.heads);
    if (a.workspace_bytes < 0) status((int)a.workspace_bytes);
    at::Tensor result, work;
    if (!out) {
      result = at::empty(q.sizes(), q.options());
      out = &result;
    }
    a.out_stride = rows(c, *out, n, a.heads, a.type, "out");
    if (a.workspace_bytes) {
      work = at::empty({a.workspace_bytes}, at::TensorOptions().dtype(at::kByte).device(c->device));
      a.workspace = work.data_ptr();
    }
    a.q = q.data_ptr();
    a.out = out->data_ptr();
    status(chonk_kv_attend(&c->c, &a, stream_of(c)));
    if (result.defined()) return THPVariable_Wrap(std::move(result));
    Py_INCREF(x[5]);
    return x[5];
  });
}

PyObject* bind(PyObject*, PyObject* args) {
  PyObject* o[4];
  if (!PyArg_ParseTuple(args, "OOOO", &o[0], &o[1], &o[2], &o[3])) return nullptr;
  PyObject** at[4] = {&g_error, &g_stream, &g_f32, &g_f16};
  for (int i = 0; i < 4; ++i) {
    Py_INCREF(o[i]);
    Py_XSETREF(*at[i], o[i]);
  }
  Py_RETURN_NONE;
}

PyMethodDef cache_methods[] = {
    {"append", (PyCFunction)(void (*)(void))cache_append, METH_FASTCALL | METH_KEYWORDS, nullptr},
    {"read", (PyCFunction)(void (*)(void))cache_read, METH_FASTCALL | METH_KEYWORDS, nullptr},
    {"attend", (PyCFunction)(void (*)(void))cache_attend, METH_FASTCALL | METH_KEYWORDS, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyMemberDef cache_members[] = {
    {"pages", T_OBJECT, offsetof(Cache, pages), READONLY, nullptr},
    {"table", T_OBJECT, offsetof(Cache, table), READONLY, nullptr},
    {"fault", T_OBJECT, offsetof(Cache, fault), READONLY, nullptr},
    {"kv_heads", T_INT, offsetof(Cache, c) + offsetof(chonk_kv_cache, kv_heads), READONLY, nullptr},
    {"head_dim", T_INT, offsetof(Cache, c) + offsetof(chonk_kv_cache, head_dim), READONLY, nullptr},
    {nullptr, 0, 0, 0, nullptr}};
PyType_Slot cache_slots[] = {{Py_tp_new, (void*)cache_new},           {Py_tp_init, (void*)cache_init},
                             {Py_tp_dealloc, (void*)cache_dealloc},   {Py_tp_traverse, (void*)cache_traverse},
                             {Py_tp_clear, (void*)cache_clear},       {Py_tp_methods, cache_methods},
                             {Py_tp_members, cache_members},          {0, nullptr}};
PyType_Spec cache_spec = {"chonklm_amd._paged_kv.Cache", sizeof(Cache), 0,
                          Py_TPFLAGS_DEFAULT | Py_TPFLAGS_BASETYPE | Py_TPFLAGS_HAVE_GC, cache_slots};

PyMethodDef module_methods[] = {{"bind", bind, METH_VARARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_paged_kv", nullptr, -1, module_methods};

}  // namespace

PyMODINIT_FUNC PyInit__paged_kv(void) {
  PyObject* m = PyModule_Create(&module_def);
  PyObject* t = m ? PyType_FromSpec(&cache_spec) : nullptr;
  if (!t || PyModule_AddObject(m, "Cache", t) < 0) {
    Py_XDECREF(t);
    Py_XDECREF(m);
    return nullptr;
  }
  return m;
}
