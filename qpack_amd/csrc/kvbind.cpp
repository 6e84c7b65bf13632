// The Python side of the kv entry points and of qph_logprobs (qpack_amd._kvbind, used by qpack_amd/kvcache.py and tokenprobs.py): checks tensors and calls the C ABI.  A step's
// kernels take 3 to 8 us each; the checks through ctypes took 10 us a call (15 with scratch), through the tensors' Python attributes
// 4.5 (8.5 with scratch and a second launch), from torch's own structures 3.3 (6.5, 7.8 with scratch by way of a Python call); each launch is about 3 of it.
// torch is loaded before this module is.
#define PY_SSIZE_T_CLEAN
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>
#include <initializer_list>

#include "../../include/qpack_hip.h"

namespace {
PyObject *g_error, *g_stream, *g_device, *g_guard;   // QphError, functions

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
  int64_t device;
  PyObject *data, *data_v;   // tensors of the cache's memory (4-bit: the one of them)
};

bool fail(const char *fmt, const char *a, const char *b = "") {
  PyErr_Format(g_error, fmt, a, b);
  return false;
}
// whether t, whose autograd data m is, has a forward-mode tangent.  Its own question takes a lock and, of a view, its base's: asked only where one of them had a tangent
// (three views a call: 0.1 us of 3.7)
bool tangent(const at::Tensor &t, const torch::autograd::AutogradMeta *m) {
  const auto may_have = [](const torch::autograd::AutogradMeta *x) { return x && x->fw_grad_; };
  const auto *v = m->is_view_ ? static_cast<const torch::autograd::DifferentiableViewMeta *>(m) : nullptr;
  return (may_have(m) || (v && v->has_fw_view() && may_have(torch::autograd::impl::get_autograd_meta(v->get_forward_view().base_)))) && t._fw_grad(0).defined();
}
bool tensor(PyObject *x, const char *name, const at::Tensor **t, const char *call = "kv") {
  if (!THPVariable_Check(x)) return fail("%s: %s must be a tensor", call, name);
  *t = &THPVariable_Unpack(x);
  const torch::autograd::AutogradMeta *m = torch::autograd::impl::get_autograd_meta(**t);   // (plain tensors have none)
  if (!m) return true;
  if (m->requires_grad() && c10::GradMode::is_enabled()) return fail("%s: %s requires a gradient, and no call here passes one on: detach it, or call under torch.no_grad()", call, name);
  if (tangent(**t, m)) return fail("%s: %s has a forward-mode tangent, and no call here passes one on: take unpack_dual's primal", call, name);
  return true;
}
bool tensor(const Cache *c, PyObject *x, const char *name, const at::Tensor **t) {   // on the cache's device
  if (!tensor(x, name, t)) return false;
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
// a tensor whose memory was given back would be NULL, and so taken as not given
bool there(const at::Tensor &t, const void *p, const char *name) { return p || !t.numel() || fail("kv: %s has no memory%s", name); }
bool index(const Cache *c, PyObject *x, const char *name, const int **p, bool may_lack = false, int64_t n = -1) try {   // int32 [n], or [nseq]; None: NULL
  if (n < 0) n = c->c.nseq;
  if (x == Py_None && may_lack) { *p = nullptr; return true; }
  const at::Tensor *t;
  if (!tensor(c, x, name, &t)) return false;
  if (t->scalar_type() != at::kInt || t->layout() != at::kStrided || t->dim() != 1 || t->size(0) != n || !t->is_contiguous()) {
    PyErr_Format(g_error, "kv: %s must be a contiguous int32 tensor [%lld]", name, (long long)n);
    return false;
  }
  *p = (const int *)t->data_ptr();
  return there(*t, *p, name);
} catch (...) { return fail("kv: %s is not a plain tensor%s", name); }
// float32, contiguous, of these sizes (last < 0: any); None: NULL
bool floats(const Cache *c, PyObject *x, const char *name, int64_t dims, int64_t last, const float **p, const at::Tensor **t) try {
  if (x == Py_None && dims == 1) { *p = nullptr; return true; }
  if (!tensor(c, x, name, t)) return false;
  if ((*t)->scalar_type() != at::kFloat || (*t)->layout() != at::kStrided || (*t)->dim() != dims || (last >= 0 && (*t)->size(dims - 1) != last) || !(*t)->is_contiguous())
    return fail("kv: %s must be a contiguous float32 tensor %s", name, dims == 1 ? "[head_dim]" : "[places, half the rotated dims], cos and sin alike");
  *p = (const float *)(*t)->data_ptr();
  return there(**t, *p, name);
} catch (...) { return fail("kv: %s is not a plain tensor%s", name); }
bool stream_of(int64_t device, void **st) {
  Ref d(PyLong_FromLongLong(device));
  Ref v(PyObject_CallOneArg(g_stream, d));
  if (!v.p) return false;
  *st = PyLong_AsVoidPtr(v);
  return !PyErr_Occurred();
}
// runs f on the tensors' device; a switch only where another one is current.  f does not throw, which would leave the switch in place: tensors say where their
// memory is (functorch's, without storage, throw) before
bool current(int64_t device, bool *yes) {
  Ref now(PyObject_CallNoArgs(g_device));
  if (!now.p) return false;
  *yes = PyLong_AsLongLong(now) == device;
  return !PyErr_Occurred();
}
template <typename F>
bool launch(int64_t device, const F &f) {
  bool here;
  void *st;
  if (!current(device, &here) || !stream_of(device, &st)) return false;
  int rc;
  if (here) rc = f(st);
  else {
    Ref d(PyLong_FromLongLong(device));
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
  if (!nargs(na, 4) || !rows(c, arg[0], "k", &k, &nk, &hk) || !rows(c, arg[1], "v", &v, &nv, &hv) || !index(c, arg[2], "pos", &pos) || !index(c, arg[3], "lens", &lens, true))
    return nullptr;
  if (nk != nv) { fail("kv: k and v have different numbers of tokens%s%s", ""); return nullptr; }
  if (hk != c->c.kv_heads || hv != c->c.kv_heads) { PyErr_Format(g_error, "kv: k and v must have %d heads", c->c.kv_heads); return nullptr; }
  if (nk > INT32_MAX) { fail("kv: too many tokens%s%s", ""); return nullptr; }
  if (!launch(c->device, [&](void *st) { return (WRITE ? qph_kv_write : qph_kv_read)(&c->c, &k, &v, (int)nk, pos, lens, st); })) return nullptr;
  for (PyObject *t : {WRITE ? c->data : arg[0], WRITE ? c->data_v : arg[1]})
    if (t) written(THPVariable_Unpack(t));
  Py_RETURN_NONE;
}
// scratch of this call alone: the allocator gives it to the stream's later work, or to the graph that is being captured
bool scratch(const Cache *c, int64_t bytes, at::Tensor *work, void **p) try {
  *p = nullptr;
  if (!bytes) return true;
  *work = at::empty({bytes}, at::TensorOptions().device(THPVariable_Unpack(c->data).device()).dtype(at::kByte));
  *p = work->data_ptr();
  return true;
} catch (...) { torch::translate_exception_to_python(std::current_exception()); return false; }
bool scale_of(PyObject *x, float *scale) {
  const double y = PyFloat_AsDouble(x);
  if (PyErr_Occurred()) return false;
  *scale = (float)y;
  return y == 0 || *scale != 0.f || fail("kv: scale is too small%s%s", "");   // (0 means the default)
}
bool attend_rows(const Cache *c, PyObject *const *arg, qph_rows *q, qph_rows *o, int64_t *n, int64_t *h, const int **pos, const int **lens) {   // (q, out, pos, lens)
  int64_t n2, h2;
  if (!rows(c, arg[0], "q", q, n, h) || !rows(c, arg[1], "out", o, &n2, &h2) || !index(c, arg[2], "pos", pos) || !index(c, arg[3], "lens", lens, true)) return false;
  if (*n != n2 || *h != h2) return fail("kv: out must have q's shape%s%s", "");
  return (*n <= INT32_MAX && *h <= INT32_MAX) || fail("kv: q is too large%s%s", "");
}
// attention(q, out, pos, lens, window, sinks, scale)
PyObject *attention(PyObject *self, PyObject *const *arg, Py_ssize_t na) {
  const Cache *c = (const Cache *)self;
  qph_rows q, o;
  int64_t n, h, bytes = 0;
  const int *pos, *lens;
  int window, sinks;
  float scale;
  if (!nargs(na, 7) || !attend_rows(c, arg, &q, &o, &n, &h, &pos, &lens) || !integer(arg[4], "window", &window) || !integer(arg[5], "sinks", &sinks) || !scale_of(arg[6], &scale)) return nullptr;
  if (qph_kv_attention_work(&c->c, q.type, (int)h, (int)n, window, sinks, &bytes) != 0) { fail("%s%s", qph_last_error()); return nullptr; }
  at::Tensor work;
  void *w;
  if (!scratch(c, bytes, &work, &w)) return nullptr;
  if (!launch(c->device, [&](void *st) { return qph_kv_attention(&c->c, &q, &o, (int)h, (int)n, pos, lens, window, sinks, scale, w, bytes, st); })) return nullptr;
  written(THPVariable_Unpack(arg[1]));
  Py_RETURN_NONE;
}
PyTypeObject cache_type = {PyVarObject_HEAD_INIT(nullptr, 0)};
bool cache_of(const Cache *c, PyObject *x, const char *name, const Cache **y) {
  if (!PyObject_TypeCheck(x, &cache_type)) { PyErr_Format(PyExc_TypeError, "%s must be a cache", name); return false; }
  *y = (const Cache *)x;
  return (*y)->device == c->device || fail("kv: %s is not on the cache's device%s", name);
}
// attention_prefix(q, out, pos, lens, scale, prefix, prefix_len)
PyObject *attention_prefix(PyObject *self, PyObject *const *arg, Py_ssize_t na) {
  const Cache *c = (const Cache *)self, *p;
  qph_rows q, o;
  int64_t n, h, bytes = 0;
  const int *pos, *lens, *plen;
  float scale;
  if (!nargs(na, 7) || !attend_rows(c, arg, &q, &o, &n, &h, &pos, &lens) || !scale_of(arg[4], &scale) || !cache_of(c, arg[5], "prefix", &p) || !index(c, arg[6], "prefix_len", &plen, true, 1)) return nullptr;
  if (qph_kv_attention_prefix_work(&c->c, &p->c, q.type, (int)h, (int)n, &bytes) != 0) { fail("%s%s", qph_last_error()); return nullptr; }
  at::Tensor work;
  void *w;
  if (!scratch(c, bytes, &work, &w)) return nullptr;
  if (!launch(c->device, [&](void *st) { return qph_kv_attention_prefix(&c->c, &p->c, plen, &q, &o, (int)h, (int)n, pos, lens, scale, w, bytes, st); })) return nullptr;
  written(THPVariable_Unpack(arg[1]));
  Py_RETURN_NONE;
}
// append(q, k, v, out, pos, lens, cos, sin, at, q_weight, k_weight, eps)
PyObject *append(PyObject *self, PyObject *const *arg, Py_ssize_t na) {
  const Cache *c = (const Cache *)self;
  qph_rows r[4];
  int64_t n[4], h[4];
  const char *names[4] = {"q", "k", "v", "out"};
  const int *pos, *lens;
  qph_turn t{};
  const at::Tensor *cos, *sin, *w;
  if (!nargs(na, 12)) return nullptr;
  for (int i = 0; i < 4; i++)
    if (!rows(c, arg[i], names[i], &r[i], &n[i], &h[i])) return nullptr;
  if (!index(c, arg[4], "pos", &pos) || !index(c, arg[5], "lens", &lens, true) || !floats(c, arg[6], "cos", 2, -1, &t.cos, &cos) || !floats(c, arg[7], "sin", 2, cos->size(1), &t.sin, &sin) ||
      !index(c, arg[8], "at", &t.at, true) || !floats(c, arg[9], "q_weight", 1, c->c.head_dim, &t.q_norm, &w) || !floats(c, arg[10], "k_weight", 1, c->c.head_dim, &t.k_norm, &w)) return nullptr;
  const double eps = PyFloat_AsDouble(arg[11]);
  if (PyErr_Occurred()) return nullptr;
  if (n[1] != n[0] || n[2] != n[0]) { fail("kv: q, k and v have different numbers of tokens%s%s", ""); return nullptr; }
  if (n[3] != n[0] || h[3] != h[0]) { fail("kv: out must have q's shape%s%s", ""); return nullptr; }
  if (h[1] != c->c.kv_heads || h[2] != c->c.kv_heads) { PyErr_Format(g_error, "kv: k and v must have %d heads", c->c.kv_heads); return nullptr; }
  if (sin->size(0) != cos->size(0)) { fail("kv: cos and sin must have the same shape%s%s", ""); return nullptr; }
  if (n[0] > INT32_MAX || h[0] > INT32_MAX || cos->size(1) > INT32_MAX) { fail("kv: q or cos is too large%s%s", ""); return nullptr; }
  t.places = cos->size(0); t.half = (int)cos->size(1); t.eps = (float)eps;
  if (!launch(c->device, [&](void *st) { return qph_kv_append(&c->c, &r[0], &r[1], &r[2], &r[3], (int)h[0], (int)n[0], pos, lens, &t, st); })) return nullptr;
  for (PyObject *x : {c->data, c->data_v, (PyObject *)arg[3]})
    if (x) written(THPVariable_Unpack(x));
  Py_RETURN_NONE;
}
// copy(source, index, pos, lens, seqs, apart)
PyObject *copy(PyObject *self, PyObject *const *arg, Py_ssize_t na) try {
  const Cache *c = (const Cache *)self, *src;
  const at::Tensor *x;
  const int *pos, *lens, *seqs;
  int64_t bytes = 0;
  if (!nargs(na, 6) || !cache_of(c, arg[0], "source", &src) || !tensor(c, arg[1], "index", &x) || !index(c, arg[2], "pos", &pos) || !index(c, arg[3], "lens", &lens, true) ||
      !index(c, arg[4], "seqs", &seqs, true)) return nullptr;
  const int apart = PyObject_IsTrue(arg[5]);
  if (apart < 0) return nullptr;
  if (x->scalar_type() != at::kInt || x->layout() != at::kStrided || x->dim() != 2 || x->size(0) != c->c.nseq || (x->size(1) > 1 && x->stride(1) != 1)) {
    PyErr_Format(g_error, "kv: index must be an int32 tensor [%d, n] with contiguous rows", c->c.nseq);
    return nullptr;
  }
  const int64_t n = x->size(1);
  if (n > INT32_MAX) { fail("kv: too many tokens%s%s", ""); return nullptr; }
  const int *at = n ? (const int *)x->data_ptr() : (const int *)16;
  const int64_t stride = x->stride(0);
  if (qph_kv_copy_work(&c->c, &src->c, (int)n, apart, &bytes) != 0) { fail("%s%s", qph_last_error()); return nullptr; }
  at::Tensor work;
  void *w;
  if (!scratch(c, bytes, &work, &w)) return nullptr;
  if (!launch(c->device, [&](void *st) { return qph_kv_copy(&c->c, &src->c, at, stride, (int)n, pos, lens, seqs, apart, w, bytes, st); })) return nullptr;
  for (PyObject *y : {c->data, c->data_v})
    if (y) written(THPVariable_Unpack(y));
  Py_RETURN_NONE;
} catch (...) { fail("kv: index is not a plain tensor%s%s", ""); return nullptr; }

// logprobs(logits, tokens, top) -> (logp, entropy, rank, top_index, top_logp)
PyObject *logprobs(PyObject *, PyObject *const *arg, Py_ssize_t na) try {
  const at::Tensor *x, *tok = nullptr;
  int top, type;
  if (!nargs(na, 3) || !tensor(arg[0], "logits", &x, "logprobs") || (arg[1] != Py_None && !tensor(arg[1], "tokens", &tok, "logprobs")) || !integer(arg[2], "top", &top)) return nullptr;
  switch (x->scalar_type()) {
    case at::kFloat: type = QPH_F32; break;
    case at::kHalf: type = QPH_F16; break;
    case at::kBFloat16: type = QPH_BF16; break;
    default: fail("logprobs: logits must be float32, float16 or bfloat16%s%s", ""); return nullptr;
  }
  if (x->layout() != at::kStrided || x->dim() != 2 || (x->size(1) > 1 && x->stride(1) != 1) || x->size(1) > INT32_MAX) { fail("logprobs: logits must be [rows, vocab] with contiguous rows%s%s", ""); return nullptr; }
  if (!x->is_cuda()) { fail("logprobs: logits must be on a GPU%s%s", ""); return nullptr; }
  const int64_t rows = x->size(0), device = x->get_device();
  if (tok && (tok->scalar_type() != at::kInt || tok->layout() != at::kStrided || tok->dim() != 1 || tok->size(0) != rows || !tok->is_contiguous())) {
    PyErr_Format(g_error, "logprobs: tokens must be a contiguous int32 tensor [%lld]", (long long)rows);
    return nullptr;
  }
  if (tok && (!tok->is_cuda() || tok->get_device() != device)) { fail("logprobs: tokens are not on the logits' device%s%s", ""); return nullptr; }
  const void *from, *ids;
  try { from = x->data_ptr(); ids = tok ? tok->data_ptr() : nullptr; }
  catch (...) { fail("logprobs: logits and tokens must be plain tensors%s%s", ""); return nullptr; }
  int64_t bytes = 0;
  if (qph_logprobs_work(type, rows, (int)x->size(1), top, &bytes) != 0) { fail("%s%s", qph_last_error()); return nullptr; }
  // the results side by side in one allocation, each from a multiple of 64 bytes on (an allocation each takes as long as the rest of the call)
  const auto f32 = at::TensorOptions().device(x->device()).dtype(at::kFloat);
  const int64_t one = (rows + 15) / 16 * 16, list = (rows * top + 15) / 16 * 16;
  const at::Tensor all = at::empty({(tok ? 3 : 1) * one + 2 * list}, f32);
  int64_t used = 0;
  auto part = [&](at::ScalarType t, at::IntArrayRef sizes, int64_t room) {
    at::Tensor y = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), c10::scalarTypeToTypeMeta(t));
    y.unsafeGetTensorImpl()->set_storage_offset(used);
    y.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    used += room;
    return y;
  };
  at::Tensor logp, rank, work, entropy = part(at::kFloat, {rows}, one);
  if (tok) { logp = part(at::kFloat, {rows}, one); rank = part(at::kInt, {rows}, one); }
  at::Tensor ti = part(at::kInt, {rows, top}, list), tl = part(at::kFloat, {rows, top}, list);
  if (bytes) work = at::empty({(bytes + 3) / 4}, f32);
  void *to[6], **next = to;
  for (const at::Tensor *t : {&logp, &entropy, &rank, &ti, &tl, &work}) *next++ = t->defined() ? t->data_ptr() : nullptr;
  const int vocab = (int)x->size(1);
  const int64_t ld = x->stride(0);
  if (!launch(device, [&](void *st) {
        return qph_logprobs(from, type, rows, vocab, ld, (const int *)ids, top, (float *)to[0], (float *)to[1], (int *)to[2], (int *)to[3], (float *)to[4], to[5], bytes, st);
      }))
    return nullptr;
  PyObject *out = PyTuple_New(5);
  if (!out) return nullptr;
  int i = 0;
  for (at::Tensor *t : {&logp, &entropy, &rank, &ti, &tl}) {
    PyObject *y = t->defined() ? THPVariable_Wrap(*t) : Py_NewRef(Py_None);
    if (!y) { Py_DECREF(out); return nullptr; }
    PyTuple_SET_ITEM(out, i++, y);
  }
  return out;
} catch (...) { if (!PyErr_Occurred()) torch::translate_exception_to_python(std::current_exception()); return nullptr; }

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
  c->data = data; c->data_v = data_v;
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
    {"attention_prefix", (PyCFunction)(void (*)(void))attention_prefix, METH_FASTCALL, "attention_prefix(q, out, pos, lens, scale, prefix, prefix_len)"},
    {"append", (PyCFunction)(void (*)(void))append, METH_FASTCALL, "append(q, k, v, out, pos, lens, cos, sin, at, q_weight, k_weight, eps)"},
    {"copy", (PyCFunction)(void (*)(void))copy, METH_FASTCALL, "copy(source, index, pos, lens, seqs, apart)"},
    {nullptr, nullptr, 0, nullptr}};

// setup(QphError, raw stream of a device, current device, device guard)
PyObject *setup(PyObject *, PyObject *args) {
  if (!PyArg_ParseTuple(args, "OOOO", &g_error, &g_stream, &g_device, &g_guard)) return nullptr;
  for (PyObject *p : {g_error, g_stream, g_device, g_guard}) Py_INCREF(p);
  Py_RETURN_NONE;
}
PyMethodDef module_methods[] = {{"setup", setup, METH_VARARGS, "the names that the module uses of Python's side"},
                                {"logprobs", (PyCFunction)(void (*)(void))logprobs, METH_FASTCALL, "logprobs(logits, tokens, top)"}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kvbind", nullptr, -1, module_methods};
}  // namespace

PyMODINIT_FUNC PyInit__kvbind(void) {
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
