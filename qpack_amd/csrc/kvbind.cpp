// The Python side of the kv entry points (qpack_amd._kvbind, used by qpack_amd/kvcache.py): checks tensors and calls the C ABI.  A step's
// kernels take 3 to 8 us each; the checks through ctypes took 10 us a call (15 with scratch), through the tensors' Python attributes
// 4.5 (8.5 with scratch and a second launch), from torch's own structures 3.5 (7.7); each launch is about 3 of it.
// torch is loaded before this module is.
#define PY_SSIZE_T_CLEAN
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>
#include <initializer_list>

#include "../../include/qpack_hip.h"

namespace {
PyObject *g_error, *g_stream, *g_device, *g_guard;   // QphError, functions
PyObject *s_new_empty;

struct Ref {   // owned reference
  PyObject *p;
  explicit Ref(PyObject *q) : p(q) {}
  ~Ref() { Py_XDECREF(p); }
  Ref(const Ref &) = delete;
  Ref &operator=(const Ref &) = delete;
  operator PyObject *() const { return p; }
};

struct Cache {
  PyObject_HEAD
  qph_kv c;
  int64_t device, item;
  PyObject *data, *data_v;   // tensors of the cache's memory (4-bit: the one of them), item bytes an element: scratch is a new one like data
};

bool fail(const char *fmt, const char *a, const char *b = "") {
  PyErr_Format(g_error, fmt, a, b);
  return false;
}
bool tensor(const Cache *c, PyObject *x, const char *name, const at::Tensor **t) {   // on the cache's device
  if (!THPVariable_Check(x)) return fail("kv: %s must be a tensor%s", name);
  *t = &THPVariable_Unpack(x);
  if ((*t)->requires_grad() && c10::GradMode::is_enabled()) return fail("kv: %s requires a gradient, and no call here passes one on: detach it, or call under torch.no_grad()%s", name);
  if (!(*t)->is_cuda() || (*t)->get_device() != c->device) return fail("kv: %s is not on the cache's device%s", name);
  return true;
}
// what a call has written, for autograd's check that nothing saved was changed (inference tensors are not checked)
void written(const at::Tensor &t) { if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version(); }
// a tensor [nseq, n, heads, head_dim] with consecutive dims
bool rows(const Cache *c, PyObject *x, const char *name, qph_rows *r, int64_t *n, int64_t *heads) try {
  const at::Tensor *t;
  if (!tensor(c, x, name, &t)) return false;
  switch (t->scalar_type()) {
    case at::kFloat: r->type = QPH_F32; break;
    case at::kHalf: r->type = QPH_F16; break;
    case at::kBFloat16: r->type = QPH_BF16; break;
    default: return fail("kv: %s must be float32, float16 or bfloat16%s", name);
  }
  if (t->layout() != at::kStrided || t->dim() != 4 || t->size(0) != c->c.nseq || t->size(3) != c->c.head_dim) {
    PyErr_Format(g_error, "kv: %s must be [%d, n, heads, %d]", name, c->c.nseq, c->c.head_dim);
    return false;
  }
  if (t->stride(3) != 1) return fail("kv: the last dimension of %s must be contiguous%s", name);
  *n = t->size(1); *heads = t->size(2);
  r->seq = t->stride(0); r->tok = t->stride(1); r->head = t->stride(2);
  r->p = t->data_ptr();
  if (*n == 0 && !r->p) r->p = (void *)16;   // a tensor without elements may have no memory: nothing of it is read
  return true;
} catch (...) { return fail("kv: %s is not a plain tensor%s", name); }   // (nested or fake ones: torch throws)
bool index(const Cache *c, PyObject *x, const char *name, const int **p) try {   // int32 [nseq]; None: NULL
  if (x == Py_None && !strcmp(name, "lens")) { *p = nullptr; return true; }
  const at::Tensor *t;
  if (!tensor(c, x, name, &t)) return false;
  if (t->scalar_type() != at::kInt || t->layout() != at::kStrided || t->dim() != 1 || t->size(0) != c->c.nseq || !t->is_contiguous()) {
    PyErr_Format(g_error, "kv: %s must be a contiguous int32 tensor [%d]", name, c->c.nseq);
    return false;
  }
  *p = (const int *)t->data_ptr();
  return true;
} catch (...) { return fail("kv: %s is not a plain tensor%s", name); }
bool stream_of(const Cache *c, void **st) {
  Ref d(PyLong_FromLongLong(c->device));
  Ref v(PyObject_CallOneArg(g_stream, d));
  if (!v.p) return false;
  *st = PyLong_AsVoidPtr(v);
  return !PyErr_Occurred();
}
// runs f on the cache's device; a switch only where another one is current
bool current(const Cache *c, bool *yes) {
  Ref now(PyObject_CallNoArgs(g_device));
  if (!now.p) return false;
  *yes = PyLong_AsLongLong(now) == c->device;
  return !PyErr_Occurred();
}
template <typename F>
bool launch(const Cache *c, bool here, void *st, const F &f) {
  int rc;
  if (here) rc = f(st);
  else {
    Ref d(PyLong_FromLongLong(c->device));
    Ref guard(PyObject_CallOneArg(g_guard, d));
    Ref in(guard.p ? PyObject_CallMethod(guard, "__enter__", nullptr) : nullptr);
    if (!in.p) return false;
    rc = f(st);
    Ref out(PyObject_CallMethod(guard, "__exit__", "OOO", Py_None, Py_None, Py_None));
    if (!out.p) return false;
  }
  return rc == 0 || fail("%s%s", qph_last_error());
}
bool integer(PyObject *x, const char *name, int *v) {
  const long long y = PyLong_AsLongLong(x);
  if (PyErr_Occurred()) return false;
  if (y < INT32_MIN || y > INT32_MAX) return fail("kv: %s is out of range%s", name);
  *v = (int)y;
  return true;
}
bool nargs(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
  return n == want;
}

// write / read (k, v, pos, lens)
template <bool WRITE>
PyObject *io(PyObject *self, PyObject *const *arg, Py_ssize_t na) {
  const Cache *c = (const Cache *)self;
  qph_rows k, v;
  int64_t nk, nv, hk, hv;
  const int *pos, *lens;
  if (!nargs(na, 4) || !rows(c, arg[0], "k", &k, &nk, &hk) || !rows(c, arg[1], "v", &v, &nv, &hv) || !index(c, arg[2], "pos", &pos) || !index(c, arg[3], "lens", &lens))
    return nullptr;
  if (nk != nv) { fail("kv: k and v have different numbers of tokens%s%s", ""); return nullptr; }
  if (hk != c->c.kv_heads || hv != c->c.kv_heads) { PyErr_Format(g_error, "kv: k and v must have %d heads", c->c.kv_heads); return nullptr; }
  if (nk > INT32_MAX) { fail("kv: too many tokens%s%s", ""); return nullptr; }
  bool here;
  void *st;
  if (!current(c, &here) || !stream_of(c, &st)) return nullptr;
  if (!launch(c, here, st, [&](void *st) { return (WRITE ? qph_kv_write : qph_kv_read)(&c->c, &k, &v, (int)nk, pos, lens, st); })) return nullptr;
  for (PyObject *t : {WRITE ? c->data : arg[0], WRITE ? c->data_v : arg[1]})
    if (t) written(THPVariable_Unpack(t));
  Py_RETURN_NONE;
}
// attention(q, out, pos, lens, window, sinks, scale)
PyObject *attention(PyObject *self, PyObject *const *arg, Py_ssize_t na) {
  const Cache *c = (const Cache *)self;
  qph_rows q, o;
  int64_t n, n2, h, h2, bytes = 0;
  const int *pos, *lens;
  int window, sinks;
  if (!nargs(na, 7) || !rows(c, arg[0], "q", &q, &n, &h) || !rows(c, arg[1], "out", &o, &n2, &h2) || !index(c, arg[2], "pos", &pos) || !index(c, arg[3], "lens", &lens) ||
      !integer(arg[4], "window", &window) || !integer(arg[5], "sinks", &sinks))
    return nullptr;
  const double scale = PyFloat_AsDouble(arg[6]);
  if (PyErr_Occurred()) return nullptr;
  if (scale != 0 && (float)scale == 0.f) { fail("kv: scale is too small%s%s", ""); return nullptr; }   // (0 means the default)
  if (n != n2 || h != h2) { fail("kv: out must have q's shape%s%s", ""); return nullptr; }
  if (n > INT32_MAX || h > INT32_MAX) { fail("kv: q is too large%s%s", ""); return nullptr; }
  if (qph_kv_attention_work(&c->c, q.type, (int)h, (int)n, window, sinks, &bytes) != 0) { fail("%s%s", qph_last_error()); return nullptr; }
  bool here;
  void *st, *w = nullptr;
  if (!current(c, &here) || !stream_of(c, &st)) return nullptr;
  // scratch of this call alone: the allocator gives it to the stream's later work, or to the graph that is being captured
  Ref size(bytes ? PyLong_FromLongLong((bytes + c->item - 1) / c->item) : nullptr), work(bytes ? PyObject_CallMethodOneArg(c->data, s_new_empty, size) : nullptr);
  if (bytes && !work.p) return nullptr;
  if (bytes) w = THPVariable_Unpack(work.p).data_ptr();
  if (!launch(c, here, st, [&](void *st) { return qph_kv_attention(&c->c, &q, &o, (int)h, (int)n, pos, lens, window, sinks, (float)scale, w, bytes, st); })) return nullptr;
  written(THPVariable_Unpack(arg[1]));
  Py_RETURN_NONE;
}

int init(PyObject *self, PyObject *args, PyObject *) {   // (kind, nseq, kv_heads, head_dim, ctx, k, v, seq, row, device, data[, the fp16 V's])
  Cache *c = (Cache *)self;
  long long ctx, k, v, seq, row, device;
  PyObject *data, *data_v = nullptr;
  if (!PyArg_ParseTuple(args, "iiiiLLLLLLO|O", &c->c.kind, &c->c.nseq, &c->c.kv_heads, &c->c.head_dim, &ctx, &k, &v, &seq, &row, &device, &data, &data_v)) return -1;
  if (!THPVariable_Check(data) || (data_v && !THPVariable_Check(data_v))) { PyErr_SetString(PyExc_TypeError, "data must be tensors"); return -1; }
  Py_INCREF(data);
  Py_XINCREF(data_v);
  Py_XDECREF(c->data);
  Py_XDECREF(c->data_v);
  c->data = data; c->data_v = data_v; c->item = c->c.kind == QPH_Q4 ? 1 : 2;
  c->c.ctx = ctx; c->c.k = (void *)k; c->c.v = (void *)v; c->c.seq = seq; c->c.row = row; c->device = device;
  return 0;
}
void dealloc(PyObject *self) {
  Py_XDECREF(((Cache *)self)->data);
  Py_XDECREF(((Cache *)self)->data_v);
  Py_TYPE(self)->tp_free(self);
}

PyMethodDef cache_methods[] = {
    {"write", (PyCFunction)(void (*)(void))io<true>, METH_FASTCALL, "write(k, v, pos, lens)"},
    {"read", (PyCFunction)(void (*)(void))io<false>, METH_FASTCALL, "read(k, v, pos, lens)"},
    {"attention", (PyCFunction)(void (*)(void))attention, METH_FASTCALL, "attention(q, out, pos, lens, window, sinks, scale)"},
    {nullptr, nullptr, 0, nullptr}};
PyTypeObject cache_type = {PyVarObject_HEAD_INIT(nullptr, 0)};

// setup(QphError, raw stream of a device, current device, device guard)
PyObject *setup(PyObject *, PyObject *args) {
  if (!PyArg_ParseTuple(args, "OOOO", &g_error, &g_stream, &g_device, &g_guard)) return nullptr;
  for (PyObject *p : {g_error, g_stream, g_device, g_guard}) Py_INCREF(p);
  Py_RETURN_NONE;
}
PyMethodDef module_methods[] = {{"setup", setup, METH_VARARGS, "the names that the module uses of Python's side"}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kvbind", nullptr, -1, module_methods};
}  // namespace

PyMODINIT_FUNC PyInit__kvbind(void) {
  s_new_empty = PyUnicode_InternFromString("new_empty");
  cache_type.tp_name = "qpack_amd._kvbind.Cache";
  cache_type.tp_basicsize = sizeof(Cache);
  cache_type.tp_flags = Py_TPFLAGS_DEFAULT;
  cache_type.tp_new = PyType_GenericNew;
  cache_type.tp_init = init;
  cache_type.tp_dealloc = dealloc;
  cache_type.tp_methods = cache_methods;
  if (PyType_Ready(&cache_type) < 0) return nullptr;
  PyObject *m = PyModule_Create(&module);
  if (!m) return nullptr;
  Py_INCREF(&cache_type);
  PyModule_AddObject(m, "Cache", (PyObject *)&cache_type);
  return m;
}
