// extern "C" entry points of libqpack_hip.so (declared in include/qpack_hip.h).  Each one catches every C++ exception
// and turns it into status -1 plus a thread-local message, so no exception crosses the C boundary.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "../../include/qpack_hip.h"
#include "hip/launch.hpp"
#include "hip/model.hpp"
#include "host/container.hpp"
#include "host/rans.hpp"
#include "host/synth.hpp"

struct qph_model {
  std::unique_ptr<qph::HipLlama> m;
};

static thread_local std::string g_err;

#define QPH_API_TRY(...)                  \
  try {                                   \
    __VA_ARGS__;                          \
    return 0;                             \
  } catch (std::exception & e) {          \
    g_err = e.what();                     \
    return -1;                            \
  } catch (...) {                         \
    g_err = "unknown C++ exception";      \
    return -1;                            \
  }

static void need(const void *p, const char *what) {
  if (!p) throw std::invalid_argument(std::string(what) + " is NULL");
}
// ---- the kv entry points' arguments
static int kv_kind(const qph_kv *c) { return c->kind == QPH_Q4 ? qph::MK_Q4 : qph::MK_F32; }
static void kv_fits(__int128 bytes) {
  if (bytes > INT64_MAX) throw std::invalid_argument("kv: the cache's bytes must be below 2^63");
}
static void kv_check(int kind, int nseq, int kv_heads, int head_dim, int64_t ctx) {
  if (kind != QPH_F16 && kind != QPH_Q4) throw std::invalid_argument("kv: kind must be QPH_F16 or QPH_Q4");
  if (nseq < 1 || nseq > 65535 || kv_heads < 1 || kv_heads > 4096) throw std::invalid_argument("kv: nseq must be in [1, 65535] and kv_heads in [1, 4096]");
  if (head_dim != 64 && head_dim != 128) throw std::invalid_argument("kv: head_dim must be 64 or 128");
  if (ctx < 1 || ctx > (int64_t)1 << 30) throw std::invalid_argument("kv: ctx must be in [1, 2^30]");
  // within the limits above the product reaches 2^65
  kv_fits(kind == QPH_Q4 ? (__int128)nseq * kv_heads * qph::kv4_records(ctx) * 9 * head_dim : (__int128)4 * nseq * ctx * kv_heads * head_dim);
}
// the cache's strides
static void kv_cache(const qph_kv *c, int64_t *seq, int64_t *row) {
  need(c, "cache");
  kv_check(c->kind, c->nseq, c->kv_heads, c->head_dim, c->ctx);
  need(c->k, "cache k");
  *seq = *row = 0;
  if ((uintptr_t)c->k % 16) throw std::invalid_argument("kv: the cache must be 16-byte aligned");
  if (c->kind == QPH_Q4) return;
  need(c->v, "cache v");
  const int64_t d = (int64_t)c->kv_heads * c->head_dim;
  *row = c->row ? c->row : d;
  const __int128 between = c->seq ? c->seq : (__int128)c->ctx * *row, span = (__int128)(c->ctx - 1) * *row + d;   // of sequences; of one's rows
  if ((uintptr_t)c->v % 16 || *row % 8 || between % 8) throw std::invalid_argument("kv: an fp16 cache must be 16-byte aligned and its strides multiples of 8");
  if (*row < d || (c->nseq > 1 && between < span)) throw std::invalid_argument("kv: the cache's rows or sequences overlap");
  kv_fits(2 * ((c->nseq - 1) * between + span));
  *seq = (int64_t)between;
  if (c->k == c->v) throw std::invalid_argument("kv: the cache's k and v overlap");
}
// the launches count an fp16 cache's threads, 8 dims each, in 32 bits
static void kv_threads(const qph_kv *c, int n) {
  if (c->kind == QPH_F16 && (int64_t)n * c->kv_heads * c->head_dim > (int64_t)1 << 34) throw std::invalid_argument("kv: n * kv_heads * head_dim must not pass 2^34 for an fp16 cache");
}
static qph::KvRows kv_rows(const qph_rows *r, const char *what, bool out, int nseq, int n, int heads, int hd) {
  need(r, what); need(r->p, what);
  if (r->type != QPH_F32 && r->type != QPH_F16 && r->type != QPH_BF16) throw std::invalid_argument(std::string("kv: the type of ") + what + " must be QPH_F32, QPH_F16 or QPH_BF16");
  if ((uintptr_t)r->p % (r->type == QPH_F32 ? 4 : 2)) throw std::invalid_argument(std::string("kv: ") + what + " is not aligned to its type");
  if (r->seq < 0 || r->tok < 0 || r->head < 0) throw std::invalid_argument(std::string("kv: negative strides of ") + what);
  if (out) {   // rows that are written lie apart: by rising strides, each step is past what the smaller ones cover
    std::pair<int64_t, int> d[3] = {{r->seq, nseq}, {r->tok, n}, {r->head, heads}};
    std::sort(d, d + 3);
    __int128 covered = hd;
    for (const auto &[stride, count] : d) {
      if (count <= 1) continue;
      if (stride < covered) throw std::invalid_argument(std::string("kv: the rows of ") + what + " overlap");
      covered += (__int128)stride * (count - 1);
    }
  }
  return {r->p, r->type == QPH_F32 ? qph::RT_F32 : r->type == QPH_F16 ? qph::RT_F16 : qph::RT_BF16, r->seq, r->tok, r->head};
}
static qph::KvIoArgs kv_io(const qph_kv *c, const qph_rows *k, const qph_rows *v, bool out, int n, const int *pos, const int *lens) {
  qph::KvIoArgs a{};
  kv_cache(c, &a.cseq, &a.crow);
  if (n < 0 || n > 1 << 20) throw std::invalid_argument("kv: n must be in [0, 2^20]");
  need(pos, "pos");
  a.cache = c->k; a.cache_v = c->v; a.ctx = c->ctx; a.nrec = qph::kv4_records(c->ctx);
  a.nseq = c->nseq; a.nkv = c->kv_heads; a.hd = c->head_dim; a.n = n; a.pos = pos; a.lens = lens;
  a.k = kv_rows(k, "k", out, c->nseq, n, c->kv_heads, c->head_dim); a.v = kv_rows(v, "v", out, c->nseq, n, c->kv_heads, c->head_dim);
  if (a.k.type != a.v.type) throw std::invalid_argument("kv: k and v must have the same type");
  if (out && n && k->p == v->p) throw std::invalid_argument("kv: the rows of k and v overlap");
  kv_threads(c, n);
  return a;
}
static void kv_attn_args(const qph_kv *c, int heads, int n, int window, int sinks, qph::KvAttnArgs &a) {
  kv_cache(c, &a.cseq, &a.crow);
  if (heads < 1 || heads % c->kv_heads) throw std::invalid_argument("kv: heads must be a positive multiple of kv_heads");
  if (n < 0 || n > 1 << 20 || (int64_t)n * (heads / c->kv_heads) > 1 << 23 || heads > 65535) throw std::invalid_argument("kv: n must be in [0, 2^20], heads <= 65535 and n * heads / kv_heads <= 2^23");
  if (window < 0 || sinks < 0) throw std::invalid_argument("kv: window and sinks must not be negative");
  a.kind = kv_kind(c); a.cache = c->k; a.cache_v = c->v; a.ctx = c->ctx; a.nrec = qph::kv4_records(c->ctx);
  a.nseq = c->nseq; a.nkv = c->kv_heads; a.hd = c->head_dim; a.heads = heads; a.rep = heads / c->kv_heads; a.n = n;
  a.window = window; a.sinks = sinks; a.few = qph::kv_few();
}
// attention over a common prefix and the sequences' own caches: both passes' arguments without their rows
static void kv_prefix_args(const qph_kv *c, const qph_kv *prefix, const int *prefix_len, int heads, int n, qph::KvAttnArgs &a, qph::KvPreArgs &p) {
  kv_attn_args(c, heads, n, 0, 0, a);
  int64_t seq, row;
  kv_cache(prefix, &seq, &row);
  if (prefix->kind != c->kind || prefix->kv_heads != c->kv_heads || prefix->head_dim != c->head_dim || prefix->nseq != 1)
    throw std::invalid_argument("kv: the prefix must be a cache of one sequence, with the kind, kv_heads and head_dim of the sequences' own");
  const int64_t tokens = (int64_t)c->nseq * n;
  if (tokens * a.rep > 1 << 23 || tokens * heads > 1 << 30) throw std::invalid_argument("kv: with a prefix nseq * n * heads / kv_heads must be <= 2^23 and nseq * n * heads <= 2^30");
  kv_attn_args(prefix, heads, 0, 0, 0, p);
  p.n = (int)tokens;
  p.prefix = {prefix_len, prefix->ctx, c->ctx, std::max(n, 1)};
}
// over q: every workgroup stores where it has read, which takes the same rows in the same places
static void kv_over(const qph_rows *q, const qph_rows *out, int nseq, int n, int heads) {
  if (n && q->p == out->p && ((nseq > 1 && q->seq != out->seq) || (n > 1 && q->tok != out->tok) || (heads > 1 && q->head != out->head)))
    throw std::invalid_argument("kv: out over q must have q's strides");
}
// what both attention calls check and set besides their caches
static void kv_attn_rows(const qph_kv *c, const qph_rows *q, const qph_rows *out, int heads, int n, const int *pos, const int *lens, float scale, qph::KvAttnArgs &a) {
  need(pos, "pos");
  a.q = kv_rows(q, "q", false, c->nseq, n, heads, c->head_dim); a.out = kv_rows(out, "out", true, c->nseq, n, heads, c->head_dim);
  if (a.q.type != a.out.type) throw std::invalid_argument("kv: q and out must have the same type");
  if (!(scale >= 0.f) || std::isinf(scale)) throw std::invalid_argument("kv: scale must be finite and not negative (0: 1 / sqrt(head_dim))");
  a.pos = pos; a.lens = lens;
  a.scale2 = 1.4426950408889634f * (scale > 0.f ? scale : 1.f / std::sqrt((float)c->head_dim));
  if (std::isinf(a.scale2)) throw std::invalid_argument("kv: scale is too large");
  kv_over(q, out, c->nseq, n, heads);
}
static int kv_row_type(int type) {
  if (type != QPH_F32 && type != QPH_F16 && type != QPH_BF16) throw std::invalid_argument("kv: the type of q must be QPH_F32, QPH_F16 or QPH_BF16");
  return type == QPH_F32 ? qph::RT_F32 : type == QPH_F16 ? qph::RT_F16 : qph::RT_BF16;
}
// what two caches' memory covers, K and V
static bool kv_overlap(const qph_kv *x, const qph_kv *y) {
  auto span = [](const qph_kv *c, bool v) {
    int64_t seq, row;
    kv_cache(c, &seq, &row);
    const uintptr_t p = (uintptr_t)(v ? c->v : c->k), d = (uintptr_t)c->kv_heads * c->head_dim;
    const uintptr_t n = c->kind == QPH_Q4 ? (uintptr_t)qph::kv4_bytes(c->nseq, c->kv_heads, c->head_dim, c->ctx) : 2 * ((c->nseq - 1) * (uintptr_t)seq + (c->ctx - 1) * (uintptr_t)row + d);
    return std::pair<uintptr_t, uintptr_t>(p, p + n);
  };
  for (int i = 0; i < (x->kind == QPH_Q4 ? 1 : 4); i++) {
    const auto a = span(x, i & 1), b = span(y, i >> 1);
    if (a.first < b.second && b.first < a.second) return true;
  }
  return false;
}
static void kv_copy_args(const qph_kv *dst, const qph_kv *src, int n, qph::KvCopyArgs &a) {
  kv_cache(dst, &a.cseq, &a.crow);
  kv_cache(src, &a.src_cseq, &a.src_crow);
  if (dst->kind != src->kind || dst->kv_heads != src->kv_heads || dst->head_dim != src->head_dim) throw std::invalid_argument("kv: caches that are copied between must have the same kind, kv_heads and head_dim");
  if (n < 0 || n > 1 << 20) throw std::invalid_argument("kv: n must be in [0, 2^20]");
  kv_threads(dst, n);
  a.cache = dst->k; a.cache_v = dst->v; a.ctx = dst->ctx; a.nrec = qph::kv4_records(dst->ctx);
  a.src = src->k; a.src_v = src->v; a.src_ctx = src->ctx; a.src_nrec = qph::kv4_records(src->ctx);
  a.nseq = dst->nseq; a.src_nseq = src->nseq; a.nkv = dst->kv_heads; a.hd = dst->head_dim; a.n = n;
}
static int64_t kv_copy_bytes(const qph_kv *dst, const qph_kv *src, int n, int apart) {
  if (!n || apart || !kv_overlap(dst, src)) return 0;
  const __int128 bytes = (__int128)dst->nseq * dst->kv_heads * dst->head_dim * (dst->kind == QPH_Q4 ? 9 * qph::kv4_records(n) : 4 * (int64_t)n);
  kv_fits(bytes);
  return (int64_t)bytes;
}
static void kv_work(const void *work, int64_t have, int64_t bytes, const char *call) {
  if (bytes && (!work || have < bytes || (uintptr_t)work % 16)) throw std::invalid_argument("kv: work must have the " + std::to_string(bytes) + " bytes that " + call + " gives, 16-byte aligned");
}
static void hck(hipError_t e, const char *what) {
  if (e == hipSuccess) return;
  (void)hipGetLastError();   // as QPH_CK
  throw std::runtime_error(std::string("hip: ") + hipGetErrorString(e) + " (" + what + ")");
}

extern "C" {

const char *qph_last_error(void) { return g_err.c_str(); }

int qph_device_count(int *n) {
  QPH_API_TRY({
    need(n, "n"); int c = 0;
    if (hipGetDeviceCount(&c) != hipSuccess) { (void)hipGetLastError(); c = 0; }
    *n = c;
  });
}

// a model's cache: MK_Q4, or MK_F32 for fp16
static int cache_kind(int kind) {
  if (kind != QPH_F16 && kind != QPH_Q4) throw std::invalid_argument("cache: kind must be QPH_F16 or QPH_Q4");
  return kind == QPH_Q4 ? qph::MK_Q4 : qph::MK_F32;
}
int qph_create(const qph_config *cfg, const qph_tensor *tensors, int n_tensors, int max_ctx, qph_model **out) {
  return qph_create_kv(cfg, tensors, n_tensors, max_ctx, QPH_F16, out);
}
int qph_create_kv(const qph_config *cfg, const qph_tensor *tensors, int n_tensors, int max_ctx, int cache, qph_model **out) {
  QPH_API_TRY({
    need(cfg, "cfg"); need(tensors, "tensors"); need(out, "out");
    *out = nullptr;
    const int kind = cache_kind(cache);
    auto *h = new qph_model;
    try { h->m.reset(new qph::HipLlama(*cfg, tensors, n_tensors, max_ctx, kind)); } catch (...) { delete h; throw; }
    *out = h;
  });
}

int qph_load(const char *path, int max_ctx, qph_model **out) { return qph_load_kv(path, max_ctx, QPH_F16, out); }
int qph_load_kv(const char *path, int max_ctx, int cache, qph_model **out) {
  QPH_API_TRY({
    need(path, "path"); need(out, "out");
    *out = nullptr;
    const int kind = cache_kind(cache);
    qph::Container c(path);
    const qph::JNode &j = c.config();
    if (j.get("arch").text() != "llama") throw std::runtime_error(std::string(path) + ": arch '" + j.get("arch").text() + "' is not a Llama-family model");
    qph_config cfg{};
    cfg.hidden = (int)j.get("hidden_size").int_or(0); cfg.layers = (int)j.get("num_hidden_layers").int_or(0);
    cfg.heads = (int)j.get("num_attention_heads").int_or(0); cfg.kv_heads = (int)j.get("num_key_value_heads").int_or(0);
    cfg.head_dim = (int)j.get("head_dim").int_or(cfg.heads > 0 ? cfg.hidden / cfg.heads : 0);
    cfg.ffn = (int)j.get("intermediate_size").int_or(0); cfg.vocab = (int)j.get("vocab_size").int_or(0);
    cfg.rms_eps = (float)j.get("rms_norm_eps").num_or(1e-6); cfg.rope_theta = j.get("rope_theta").num_or(10000);
    cfg.tied = j.get("tie_embeddings").bool_or(false) ? 1 : 0;
    cfg.max_pos = (int)j.get("max_position_embeddings").int_or(1 << 20);
    std::vector<qph_tensor> ts;
    for (const qph::JNode &e : c.manifest().get("tensors").items()) {
      const qph::TensorView &t = c.at(e.get("name").text());
      if (t.kind == qph::Kind::F16) continue;   // 2-D f16 matrices are not on the HIP path; a required one is reported missing
      qph_tensor q{}; q.name = t.name.c_str(); q.data = t.data; q.scale = t.scale;
      if (t.shape.size() == 1) { q.rows = t.shape[0]; q.cols = 1; } else { q.rows = t.rows(); q.cols = t.cols(); }
      q.kind = t.kind == qph::Kind::Q8 ? QPH_Q8 : t.kind == qph::Kind::Q4 ? QPH_Q4 : t.kind == qph::Kind::Q1 ? QPH_Q1 : QPH_F32;
      q.data_coded = (int64_t)t.data_coded; q.scale_coded = (int64_t)t.scale_coded;
      ts.push_back(q);
    }
    cfg.qkv_bias = c.get("layers.0.bq") ? 1 : 0;
    auto *h = new qph_model;
    try { h->m.reset(new qph::HipLlama(cfg, ts.data(), (int)ts.size(), max_ctx, kind)); } catch (...) { delete h; throw; }
    *out = h;
  });
}

void qph_destroy(qph_model *m) { delete m; }

int qph_load_stats_of(const qph_model *m, qph_load_stats *out) {
  QPH_API_TRY({
    need(m, "model"); need(out, "out");
    const qph::RansTiming &t = m->m->load_timing();
    out->planes = t.planes; out->coded_bytes = (int64_t)t.coded; out->raw_bytes = (int64_t)t.raw;
    out->upload_ms = t.upload_ms; out->decode_ms = t.decode_ms; out->total_ms = t.total_ms; out->rounds = t.rounds;
  });
}

int qph_vocab(const qph_model *m) { return m ? m->m->config().vocab : -1; }
int qph_hidden(const qph_model *m) { return m ? m->m->config().hidden : -1; }
int qph_max_ctx(const qph_model *m) { return m ? m->m->max_ctx() : -1; }
int qph_pos(const qph_model *m) { return m ? m->m->pos() : -1; }
int qph_config_of(const qph_model *m, qph_config *out) { QPH_API_TRY({ need(m, "model"); need(out, "out"); *out = m->m->config(); }); }

int qph_step(qph_model *m, int token, int want, float *out) {
  QPH_API_TRY({
    need(m, "model");
    if (want < 0 || want > 2) throw std::invalid_argument("want must be 0, 1 or 2");
    if (want) need(out, "out");
    m->m->step(token, want, out);
  });
}
int qph_prefill(qph_model *m, const int *tokens, int n, int want, float *out) {
  QPH_API_TRY({
    need(m, "model"); need(tokens, "tokens");
    if (want < 0 || want > 2) throw std::invalid_argument("want must be 0, 1 or 2");
    if (want) need(out, "out");
    m->m->prefill(tokens, n, want, out);
  });
}
int qph_greedy_run(qph_model *m, int token, int n, int *out, int *produced) {
  QPH_API_TRY({
    need(m, "model"); need(out, "out");
    const int r = m->m->greedy_run(token, n, out);
    if (produced) *produced = r;
  });
}
int qph_verify_batches(const qph_model *m, int64_t *n) {
  QPH_API_TRY({ need(m, "model"); need(n, "n"); *n = m->m->verify_batches(); });
}
int qph_prefill_all(qph_model *m, const int *tokens, int n, float *logits) {
  QPH_API_TRY({ need(m, "model"); need(tokens, "tokens"); need(logits, "logits"); m->m->prefill_all(tokens, n, logits); });
}
int qph_score(qph_model *m, const int *tokens, const int *targets, int n, int top, float *logp, float *entropy, int *rank, int *top_index, float *top_logp) {
  QPH_API_TRY({
    need(m, "model"); need(tokens, "tokens");
    m->m->score(tokens, targets, n, top, {logp, entropy, rank, top_index, top_logp});
  });
}
int qph_step_topk(qph_model *m, int token, int M, int *idx, float *val) {
  QPH_API_TRY({ need(m, "model"); need(idx, "idx"); need(val, "val"); m->m->step_topk(token, M, idx, val); });
}
int qph_prefill_topk(qph_model *m, const int *tokens, int n, int M, int *idx, float *val) {
  QPH_API_TRY({
    need(m, "model"); need(tokens, "tokens"); need(idx, "idx"); need(val, "val");
    m->m->prefill_topk(tokens, n, M, idx, val);
  });
}
int qph_reset(qph_model *m) { QPH_API_TRY({ need(m, "model"); m->m->reset(); }); }
int qph_rewind(qph_model *m, int pos, int *ok) {
  QPH_API_TRY({ need(m, "model"); const bool r = m->m->rewind(pos); if (ok) *ok = r ? 1 : 0; });
}
int qph_set_pos(qph_model *m, int pos) { QPH_API_TRY({ need(m, "model"); m->m->set_pos(pos); }); }
int qph_snapshot_size(const qph_model *m, int64_t *bytes) { QPH_API_TRY({ need(m, "model"); need(bytes, "bytes"); *bytes = m->m->snapshot_size(); }); }
int qph_snapshot(qph_model *m, uint8_t *buf, int64_t cap) { QPH_API_TRY({ need(m, "model"); need(buf, "buf"); m->m->snapshot(buf, cap); }); }
int qph_restore(qph_model *m, const uint8_t *buf, int64_t n) { QPH_API_TRY({ need(m, "model"); need(buf, "buf"); m->m->restore(buf, n); }); }

int qph_set_cache(qph_model *m, int kind) { QPH_API_TRY({ need(m, "model"); m->m->set_cache(cache_kind(kind)); }); }
int qph_set_window(qph_model *m, int window, int sinks) { QPH_API_TRY({ need(m, "model"); m->m->set_window(window, sinks); }); }
int qph_set_order(qph_model *m, int mode) { QPH_API_TRY({ need(m, "model"); m->m->set_order(mode); }); }

int qph_time_greedy(qph_model *m, int token, int n, float *ms) {
  QPH_API_TRY({ need(m, "model"); need(ms, "ms"); *ms = m->m->time_greedy(token, n); });
}
int qph_time_kernel(qph_model *m, int which, int iters, float *ms, double *bytes) {
  QPH_API_TRY({ need(m, "model"); need(ms, "ms"); need(bytes, "bytes"); *ms = m->m->time_kernel(which, iters, bytes); });
}

int qph_time_copy(int64_t bytes, int iters, float *ms) {
  QPH_API_TRY({
    need(ms, "ms");
    if (bytes <= 0 || bytes % 16) throw std::invalid_argument("time_copy: bytes must be a positive multiple of 16");
    if (iters <= 0) iters = 1;
    void *src = nullptr, *dst = nullptr;
    hipStream_t st = nullptr;
    hipEvent_t e0 = nullptr, e1 = nullptr;
    auto cleanup = [&]() {
      if (e0) (void)hipEventDestroy(e0);
      if (e1) (void)hipEventDestroy(e1);
      if (st) (void)hipStreamDestroy(st);
      if (src) (void)hipFree(src);
      if (dst) (void)hipFree(dst);
    };
    try {
      QPH_CK(hipMalloc(&src, bytes)); QPH_CK(hipMalloc(&dst, bytes));
      QPH_CK(hipStreamCreateWithFlags(&st, hipStreamNonBlocking));
      QPH_CK(hipMemsetAsync(src, 1, bytes, st));
      QPH_CK(hipEventCreate(&e0)); QPH_CK(hipEventCreate(&e1));
      QPH_CK(qph::launch_copy(src, dst, bytes / 16, st));   // warm-up
      QPH_CK(hipEventRecord(e0, st));
      for (int i = 0; i < iters; i++) QPH_CK(qph::launch_copy(src, dst, bytes / 16, st));
      QPH_CK(hipEventRecord(e1, st));
      QPH_CK(hipEventSynchronize(e1));
      QPH_CK(hipEventElapsedTime(ms, e0, e1));
      *ms /= iters;
    } catch (...) { cleanup(); throw; }
    cleanup();
  });
}

int qph_kernel_matvec(int kind, const void *q, const void *scale, int rows, int cols, const float *x, float *y,
                      int32_t *sums, int16_t *xq, float *bs) {
  QPH_API_TRY({
    need(q, "q"); need(scale, "scale"); need(x, "x"); need(y, "y");
    if (rows <= 0 || cols <= 0 || cols % 128) throw std::invalid_argument("matvec: rows > 0 and cols a positive multiple of 128 required");
    if (kind != QPH_Q8 && kind != QPH_Q4 && kind != QPH_Q1) throw std::invalid_argument("matvec: kind must be QPH_Q8, QPH_Q4 or QPH_Q1");
    const size_t qb = kind == QPH_Q8 ? (size_t)rows * cols : kind == QPH_Q4 ? (size_t)rows * cols / 2 : (size_t)rows * cols / 8;
    const size_t sb = kind == QPH_Q8 ? 4ull * rows : kind == QPH_Q4 ? 2ull * rows * (cols / 32) : 2ull * rows * (cols / 128);
    const size_t nsum = kind == QPH_Q4 ? (size_t)rows * (cols / 32) : (size_t)rows * (cols / 128);
    std::vector<void *> bufs;
    auto alloc = [&](size_t n) { void *p = nullptr; hck(hipMalloc(&p, n), "hipMalloc"); bufs.push_back(p); return p; };
    try {
      void *dq = alloc(qb), *ds = alloc(sb); float *dx = (float *)alloc(4ull * cols), *dy = (float *)alloc(4ull * rows);
      int32_t *dsum = sums ? (int32_t *)alloc(4 * nsum) : nullptr;
      int16_t *dxq = xq ? (int16_t *)alloc(2ull * cols) : nullptr;
      float *dbs = bs ? (float *)alloc(4ull * (cols / 128)) : nullptr;
      hck(hipMemcpy(dq, q, qb, hipMemcpyHostToDevice), "upload q");
      hck(hipMemcpy(ds, scale, sb, hipMemcpyHostToDevice), "upload scale");
      hck(hipMemcpy(dx, x, 4ull * cols, hipMemcpyHostToDevice), "upload x");
      qph::MvArgs a{}; a.m[0].q = dq; a.m[0].s = ds; a.m[0].rows = rows; a.m[0].cols = cols; a.m[0].kind = kind == QPH_Q8 ? qph::MK_Q8 : kind == QPH_Q4 ? qph::MK_Q4 : qph::MK_Q1;
      a.nseg = 1; a.x = dx; a.out[0] = dy; a.dbg_sums = dsum; a.dbg_xq = dxq; a.dbg_bs = dbs;
      qph::mv_plan(a, qph::EPI_STORE);
      hck(qph::launch_matvec(qph::PRO_QUANT, qph::EPI_STORE, a, 256, nullptr), "launch matvec");
      hck(hipDeviceSynchronize(), "matvec");
      hck(hipMemcpy(y, dy, 4ull * rows, hipMemcpyDeviceToHost), "download y");
      if (sums) hck(hipMemcpy(sums, dsum, 4 * nsum, hipMemcpyDeviceToHost), "download sums");
      if (xq) hck(hipMemcpy(xq, dxq, 2ull * cols, hipMemcpyDeviceToHost), "download xq");
      if (bs) hck(hipMemcpy(bs, dbs, 4ull * (cols / 128), hipMemcpyDeviceToHost), "download bs");
    } catch (...) { for (void *p : bufs) (void)hipFree(p); throw; }
    for (void *p : bufs) (void)hipFree(p);
  });
}

int qph_kernel_topk(const float *x, int n, int M, int *idx, float *val) {
  QPH_API_TRY({
    need(x, "x"); need(idx, "idx"); need(val, "val");
    if (n <= 0 || M < 1 || M > qph::kTopkMax || M > n) throw std::invalid_argument("topk: 1 <= M <= min(512, n) required");
    std::vector<void *> bufs;
    auto alloc = [&](size_t b) { void *p = nullptr; hck(hipMalloc(&p, b), "hipMalloc"); bufs.push_back(p); return p; };
    try {
      const size_t keys = qph::topk_scratch_keys(n, M);
      float *dx = (float *)alloc(4ull * n), *dv = (float *)alloc(4ull * M);
      int *di = (int *)alloc(4ull * M);
      uint64_t *ka = (uint64_t *)alloc(8 * keys), *kb = (uint64_t *)alloc(8 * keys);
      hck(hipMemcpy(dx, x, 4ull * n, hipMemcpyHostToDevice), "upload x");
      hck(qph::launch_topk(dx, n, M, ka, kb, di, dv, nullptr), "launch topk");
      hck(hipDeviceSynchronize(), "topk");
      hck(hipMemcpy(idx, di, 4ull * M, hipMemcpyDeviceToHost), "download idx");
      hck(hipMemcpy(val, dv, 4ull * M, hipMemcpyDeviceToHost), "download val");
    } catch (...) { for (void *p : bufs) (void)hipFree(p); throw; }
    for (void *p : bufs) (void)hipFree(p);
  });
}
int qph_topk_noalloc(const float *x, int n, int M, int *idx, float *val, void *stream) {
  QPH_API_TRY({
    need(x, "x"); need(idx, "idx"); need(val, "val");
    if (n <= 0 || n > 262144) throw std::invalid_argument("topk_noalloc: n must be in [1, 262144] (the size of its fixed device buffers)");
    if (M < 1 || M > qph::kTopkMax || M > n) throw std::invalid_argument("topk_noalloc: 1 <= M <= min(512, n) required");
    hck(qph::launch_topk_noalloc(x, n, M, idx, val, (hipStream_t)stream), "launch topk");
  });
}
static void logprob_args(int type, int64_t rows, int vocab, int top, qph::LogprobArgs &a) {
  if (type != QPH_F32 && type != QPH_F16 && type != QPH_BF16) throw std::invalid_argument("logprobs: the type must be QPH_F32, QPH_F16 or QPH_BF16");
  if (rows < 0 || rows > 1 << 23) throw std::invalid_argument("logprobs: rows must be in [0, 2^23]");   // (256 threads each, counted in 32 bits)
  if (vocab < 1 || vocab > 1 << 28) throw std::invalid_argument("logprobs: vocab must be in [1, 2^28]");
  if (top < 0 || top > std::min(qph::kLpTop, vocab)) throw std::invalid_argument("logprobs: top must be in [0, min(64, vocab)]");
  a.type = type == QPH_F32 ? qph::RT_F32 : type == QPH_F16 ? qph::RT_F16 : qph::RT_BF16;
  a.rows = rows; a.vocab = vocab; a.top = top;
}
int qph_logprobs_work(int type, int64_t rows, int vocab, int top, int64_t *bytes) {
  QPH_API_TRY({
    need(bytes, "bytes");
    qph::LogprobArgs a{};
    logprob_args(type, rows, vocab, top, a);
    *bytes = rows ? (int64_t)qph::logprobs_plan(a) : 0;
  });
}
int qph_logprobs(const void *x, int type, int64_t rows, int vocab, int64_t ld, const int *tokens, int top, float *logp, float *entropy, int *rank, int *top_index,
                 float *top_logp, void *work, int64_t work_bytes, void *stream) {
  QPH_API_TRY({
    qph::LogprobArgs a{};
    logprob_args(type, rows, vocab, top, a);
    if (rows) {
      need(x, "x");
      if ((uintptr_t)x % (type == QPH_F32 ? 4 : 2)) throw std::invalid_argument("logprobs: x is not aligned to its type");
      if (ld < 0) throw std::invalid_argument("logprobs: negative stride");
      if (!tokens && (logp || rank)) throw std::invalid_argument("logprobs: logp and rank need tokens");
      if (top) { need(top_index, "top_index"); need(top_logp, "top_logp"); }
      a.x = x; a.ld = ld; a.tokens = tokens; a.logp = logp; a.entropy = entropy; a.rank = rank; a.top_index = top_index; a.top_logp = top_logp;
      const int64_t bytes = (int64_t)qph::logprobs_plan(a);
      if (bytes && (!work || work_bytes < bytes || (uintptr_t)work % 16)) throw std::invalid_argument("logprobs: work must have the " + std::to_string(bytes) + " bytes that qph_logprobs_work gives, 16-byte aligned");
      a.work = work;
      hck(qph::launch_logprobs(a, (hipStream_t)stream), "logprobs");
    }
  });
}
int qph_kernel_matmul(int kind, const void *q, const void *scale, int rows, int cols, const float *X, int B, float *Y) {
  QPH_API_TRY({
    need(q, "q"); need(scale, "scale"); need(X, "X"); need(Y, "Y");
    if (rows <= 0 || B <= 0 || cols <= 0 || cols % 128) throw std::invalid_argument("matmul: rows, B > 0 and cols a positive multiple of 128 required");
    if (kind != QPH_Q8 && kind != QPH_Q4 && kind != QPH_Q1) throw std::invalid_argument("matmul: kind must be QPH_Q8, QPH_Q4 or QPH_Q1");
    const int nb = cols / 128, ldb = (nb + 7) / 8 * 8, G = cols / 32, mk = kind == QPH_Q8 ? qph::MK_Q8 : kind == QPH_Q4 ? qph::MK_Q4 : qph::MK_Q1;
    const size_t qb = kind == QPH_Q8 ? (size_t)rows * cols : kind == QPH_Q4 ? (size_t)rows * cols / 2 : (size_t)rows * cols / 8;
    const size_t sb = kind == QPH_Q8 ? 4ull * rows : kind == QPH_Q4 ? 2ull * rows * G : 2ull * rows * nb;
    std::vector<void *> bufs;
    auto alloc = [&](size_t n) { void *p = nullptr; hck(hipMalloc(&p, n), "hipMalloc"); bufs.push_back(p); return p; };
    try {
      void *dq = alloc(qb), *ds = alloc(sb);
      float *dx = (float *)alloc(4ull * B * cols), *dy = (float *)alloc(4ull * B * rows), *dxb = (float *)alloc(4ull * B * ldb);
      const int ldbt = (B + 63) / 64 * 64;
      float *dxbt = (float *)alloc(4ull * ldbt * nb);
      int8_t *dxh = (int8_t *)alloc((size_t)B * cols), *dxl = (int8_t *)alloc((size_t)B * cols);
      hck(hipMemcpy(dq, q, qb, hipMemcpyHostToDevice), "upload q");
      hck(hipMemcpy(ds, scale, sb, hipMemcpyHostToDevice), "upload scale");
      hck(hipMemcpy(dx, X, 4ull * B * cols, hipMemcpyHostToDevice), "upload X");
      qph::GemmArgs ga{}; ga.kind = mk; ga.w = (const int8_t *)dq; ga.scale = (const float *)ds;
      ga.rows = rows; ga.cols = cols; ga.xh = dxh; ga.xl = dxl; ga.xb = dxb; ga.ntok = B; ga.ldq = cols; ga.ldb = ldb;
      ga.y = dy; ga.ldy = rows; ga.xbt = dxbt; ga.ldbt = ldbt;
      qph::PfQuantArgs qa{}; qa.x = dx; qa.ldx = cols; qa.cols = cols; qa.xh = dxh; qa.xl = dxl; qa.ldq = cols; qa.xb = dxb; qa.ldb = ldb;
      qa.xbt = dxbt; qa.ldbt = ldbt;
      if (qph::gemm_wants_tiles(ga)) {   // the few-token kernel: the planes in 16-token tiles
        const size_t tb = (size_t)(B + 15) / 16 * 16 * cols;
        qa.th = (int8_t *)alloc(tb); qa.tl = (int8_t *)alloc(tb); qa.xh = qa.xl = nullptr;
        ga.th = qa.th; ga.tl = qa.tl;
      }
      if (kind != QPH_Q8) {
        qa.fp = (uint16_t *)alloc((size_t)(B + 15) / 16 * 16 * cols * (kind == QPH_Q4 ? 4 : 2));
        qa.fkind = mk; ga.fp = qa.fp;
      }
      hck(qph::launch_pf_quant(qph::PRO_QUANT, qa, B, nullptr), "launch quant");
      if (kind == QPH_Q8) {
        int *dws = (int *)alloc(4ull * qph::ws_pitch(rows) * nb);
        hck(qph::launch_rowsum_q8((const int8_t *)dq, rows, cols, dws, nullptr), "launch rowsum");
        ga.wsum = dws;
      } else {
        uint16_t *dst = (uint16_t *)alloc(sb);
        hck(qph::launch_scale_blocks(mk, (const uint16_t *)ds, rows, cols, dst, nullptr), "launch scale blocks");
        ga.st = dst;
      }
      hck(qph::launch_gemm(ga, nullptr), "launch gemm");
      hck(hipDeviceSynchronize(), "matmul");
      hck(hipMemcpy(Y, dy, 4ull * B * rows, hipMemcpyDeviceToHost), "download Y");
    } catch (...) { for (void *p : bufs) (void)hipFree(p); throw; }
    for (void *p : bufs) (void)hipFree(p);
  });
}

int qph_kernel_matmul_ref(int kind, const void *q, const void *scale, int rows, int cols, const float *X, int B, float *Y) {
  QPH_API_TRY({
    need(q, "q"); need(scale, "scale"); need(X, "X"); need(Y, "Y");
    if (rows <= 0 || B <= 0 || cols <= 0 || cols % 128) throw std::invalid_argument("matmul: rows, B > 0 and cols a positive multiple of 128 required");
    if (kind != QPH_Q8 && kind != QPH_Q4 && kind != QPH_Q1) throw std::invalid_argument("matmul: kind must be QPH_Q8, QPH_Q4 or QPH_Q1");
    const int nb = cols / 128, G = cols / 32;
    const size_t qb = kind == QPH_Q8 ? (size_t)rows * cols : kind == QPH_Q4 ? (size_t)rows * cols / 2 : (size_t)rows * cols / 8;
    const size_t sb = kind == QPH_Q8 ? 4ull * rows : kind == QPH_Q4 ? 2ull * rows * G : 2ull * rows * nb;
    std::vector<void *> bufs;
    auto alloc = [&](size_t n) { void *p = nullptr; hck(hipMalloc(&p, n), "hipMalloc"); bufs.push_back(p); return p; };
    try {
      void *dq = alloc(qb), *ds = alloc(sb);
      float *dx = (float *)alloc(4ull * B * cols), *dy = (float *)alloc(4ull * B * rows), *dxb = (float *)alloc(4ull * B * nb);
      int8_t *dxh = (int8_t *)alloc((size_t)B * cols), *dxl = (int8_t *)alloc((size_t)B * cols);
      hck(hipMemcpy(dq, q, qb, hipMemcpyHostToDevice), "upload q");
      hck(hipMemcpy(ds, scale, sb, hipMemcpyHostToDevice), "upload scale");
      hck(hipMemcpy(dx, X, 4ull * B * cols, hipMemcpyHostToDevice), "upload X");
      qph::PfQuantArgs qa{}; qa.x = dx; qa.ldx = cols; qa.cols = cols; qa.xh = dxh; qa.xl = dxl; qa.ldq = cols; qa.xb = dxb; qa.ldb = nb;
      hck(qph::launch_pf_quant(qph::PRO_QUANT, qa, B, nullptr), "launch quant");
      qph::ExGemmArgs ga{}; ga.kind = kind == QPH_Q8 ? qph::MK_Q8 : kind == QPH_Q4 ? qph::MK_Q4 : qph::MK_Q1; ga.w = dq; ga.scale = (const float *)ds;
      ga.s16 = (const uint16_t *)ds; ga.rows = rows; ga.cols = cols; ga.xh = dxh; ga.xl = dxl; ga.ldq = cols; ga.xb = dxb;
      ga.ldb = nb; ga.ntok = B; ga.mm_below = B - B % 4; ga.tt = B == 1 ? 1 : 16; ga.y = dy; ga.ldy = rows;
      hck(qph::launch_ex_gemm(ga, nullptr), "launch gemm");
      hck(hipDeviceSynchronize(), "matmul");
      hck(hipMemcpy(Y, dy, 4ull * B * rows, hipMemcpyDeviceToHost), "download Y");
    } catch (...) { for (void *p : bufs) (void)hipFree(p); throw; }
    for (void *p : bufs) (void)hipFree(p);
  });
}

int qph_kv_bytes(int kind, int nseq, int kv_heads, int head_dim, int64_t ctx, int64_t *bytes) {
  QPH_API_TRY({
    need(bytes, "bytes");
    kv_check(kind, nseq, kv_heads, head_dim, ctx);
    *bytes = kind == QPH_Q4 ? qph::kv4_bytes(nseq, kv_heads, head_dim, ctx) : 4 * nseq * ctx * kv_heads * head_dim;
  });
}
int qph_kv_write(const qph_kv *c, const qph_rows *k, const qph_rows *v, int n, const int *pos, const int *lens, void *stream) {
  QPH_API_TRY({
    const qph::KvIoArgs a = kv_io(c, k, v, false, n, pos, lens);
    if (n) hck(qph::launch_kv_write(kv_kind(c), a, (hipStream_t)stream), "kv write");
  });
}
int qph_kv_read(const qph_kv *c, const qph_rows *k, const qph_rows *v, int n, const int *pos, const int *lens, void *stream) {
  QPH_API_TRY({
    const qph::KvIoArgs a = kv_io(c, k, v, true, n, pos, lens);
    if (n) hck(qph::launch_kv_read(kv_kind(c), a, (hipStream_t)stream), "kv read");
  });
}
int qph_kv_append(const qph_kv *c, const qph_rows *q, const qph_rows *k, const qph_rows *v, const qph_rows *out, int heads, int n, const int *pos, const int *lens,
                  const qph_turn *turn, void *stream) {
  QPH_API_TRY({
    qph::KvAppendArgs a{};
    a.io = kv_io(c, k, v, false, n, pos, lens);
    need(turn, "turn");
    if (heads < 1 || heads % c->kv_heads || heads > 65535) throw std::invalid_argument("kv: heads must be a positive multiple of kv_heads, at most 65535");
    if ((int64_t)n * (heads + 2 * c->kv_heads) > 1 << 26) throw std::invalid_argument("kv: n * (heads + 2 * kv_heads) must not pass 2^26");
    a.q = kv_rows(q, "q", false, c->nseq, n, heads, c->head_dim); a.out = kv_rows(out, "out", true, c->nseq, n, heads, c->head_dim);
    if (a.q.type != a.out.type || a.q.type != a.io.k.type) throw std::invalid_argument("kv: q, k, v and out must have the same type");
    kv_over(q, out, c->nseq, n, heads);
    if (turn->half < 0 || 2 * turn->half > c->head_dim || turn->half % (c->head_dim / 8)) throw std::invalid_argument("kv: half the rotated dims must be a multiple of head_dim / 8, and at most head_dim / 2");
    if (turn->places < 1 || turn->places > (int64_t)1 << 31) throw std::invalid_argument("kv: places must be in [1, 2^31]");
    if (turn->half) { need(turn->cos, "cos"); need(turn->sin, "sin"); }
    if (!(turn->eps >= 0.f) || std::isinf(turn->eps)) throw std::invalid_argument("kv: eps must be finite and not negative");
    for (const float *p : {turn->cos, turn->sin, turn->q_norm, turn->k_norm}) if ((uintptr_t)p % 4) throw std::invalid_argument("kv: cos, sin and the norms' weights must be aligned to 4 bytes");
    a.heads = heads; a.half = turn->half; a.cos_t = turn->cos; a.sin_t = turn->sin; a.places = turn->places;
    a.qw = turn->q_norm; a.kw = turn->k_norm; a.eps = turn->eps; a.at = turn->at;
    if (n) hck(qph::launch_kv_append(kv_kind(c), a, (hipStream_t)stream), "kv append");
  });
}
int qph_kv_copy_work(const qph_kv *dst, const qph_kv *src, int n, int apart, int64_t *bytes) {
  QPH_API_TRY({
    need(bytes, "bytes");
    qph::KvCopyArgs a{};
    kv_copy_args(dst, src, n, a);
    *bytes = kv_copy_bytes(dst, src, n, apart);
  });
}
int qph_kv_copy(const qph_kv *dst, const qph_kv *src, const int *index, int64_t index_seq, int n, const int *pos, const int *lens, const int *seqs, int apart, void *work,
                int64_t work_bytes, void *stream) {
  QPH_API_TRY({
    qph::KvCopyArgs a{};
    kv_copy_args(dst, src, n, a);
    need(index, "index"); need(pos, "pos");
    if (index_seq < 0) throw std::invalid_argument("kv: negative stride of index");
    a.index = index; a.index_seq = index_seq; a.pos = pos; a.lens = lens; a.seqs = seqs;
    const int64_t bytes = kv_copy_bytes(dst, src, n, apart);
    kv_work(work, work_bytes, bytes, "qph_kv_copy_work");
    a.work = bytes ? work : nullptr;
    if (n) hck(qph::launch_kv_copy(kv_kind(dst), a, (hipStream_t)stream), "kv copy");
  });
}
int qph_kv_attention_work(const qph_kv *c, int type, int heads, int n, int window, int sinks, int64_t *bytes) {
  QPH_API_TRY({
    need(bytes, "bytes");
    qph::KvAttnArgs a{};
    a.q.type = kv_row_type(type);
    kv_attn_args(c, heads, n, window, sinks, a);
    *bytes = n ? (int64_t)qph::kv_attn_plan(a) : 0;
  });
}
int qph_kv_attention(const qph_kv *c, const qph_rows *q, const qph_rows *out, int heads, int n, const int *pos, const int *lens,
                     int window, int sinks, float scale, void *work, int64_t work_bytes, void *stream) {
  QPH_API_TRY({
    qph::KvAttnArgs a{};
    kv_attn_args(c, heads, n, window, sinks, a);
    kv_attn_rows(c, q, out, heads, n, pos, lens, scale, a);
    if (n) {
      const int64_t bytes = (int64_t)qph::kv_attn_plan(a);
      kv_work(work, work_bytes, bytes, "qph_kv_attention_work");
      a.part = (float *)work;
      hck(qph::launch_kv_attn(a, (hipStream_t)stream), "kv attention");
    }
  });
}
int qph_kv_attention_prefix_work(const qph_kv *c, const qph_kv *prefix, int type, int heads, int n, int64_t *bytes) {
  QPH_API_TRY({
    need(bytes, "bytes");
    qph::KvAttnArgs a{};
    qph::KvPreArgs p{};
    a.q.type = p.q.type = kv_row_type(type);
    kv_prefix_args(c, prefix, nullptr, heads, n, a, p);
    *bytes = n ? (int64_t)qph::kv_prefix_plan(a, p) : 0;
  });
}
int qph_kv_attention_prefix(const qph_kv *c, const qph_kv *prefix, const int *prefix_len, const qph_rows *q, const qph_rows *out, int heads, int n, const int *pos,
                            const int *lens, float scale, void *work, int64_t work_bytes, void *stream) {
  QPH_API_TRY({
    qph::KvAttnArgs a{};
    qph::KvPreArgs p{};
    kv_prefix_args(c, prefix, prefix_len, heads, n, a, p);
    kv_attn_rows(c, q, out, heads, n, pos, lens, scale, a);
    if (n) {
      p.q = a.q; p.out = a.out; p.pos = pos; p.lens = lens; p.scale2 = a.scale2;
      const int64_t bytes = (int64_t)qph::kv_prefix_plan(a, p);
      kv_work(work, work_bytes, bytes, "qph_kv_attention_prefix_work");
      a.part = p.part = (float *)work;
      hck(qph::launch_kv_prefix(a, p, (hipStream_t)stream), "kv attention");
    }
  });
}

int qph_kernel_rans_decode(const uint8_t *blob, int64_t len, uint8_t *out, int64_t cap, int64_t *raw, float *ms) {
  QPH_API_TRY({
    need(blob, "blob"); need(out, "out");
    if (len < 0 || cap < 0) throw std::invalid_argument("rans: negative length");
    const uint64_t n = qph::rans::raw_size(blob, (size_t)len);
    if (raw) *raw = (int64_t)n;
    if ((int64_t)n > cap) throw std::invalid_argument("rans: output buffer smaller than the raw length");
    void *d = nullptr;
    hck(hipMalloc(&d, n + 16), "hipMalloc");
    try {
      qph::RansBatch b;
      qph::RansTiming tm;
      b.add(blob, (size_t)len, d, n);
      b.run(nullptr, &tm, qph::RansBatch::default_round());
      if (n) hck(hipMemcpy(out, d, n, hipMemcpyDeviceToHost), "download");
      if (ms) *ms = tm.decode_ms;
    } catch (...) { (void)hipFree(d); throw; }
    hck(hipFree(d), "hipFree");
  });
}

int qph_pack(const char *src, const char *dst, int threads, int *coded) {
  QPH_API_TRY({
    need(src, "src"); need(dst, "dst");
    const int c = qph::rans::pack(src, dst, threads);
    if (coded) *coded = c;
  });
}

int qph_synth_write(const qph_synth_spec *spec, const char *path, int threads) {
  QPH_API_TRY({ need(spec, "spec"); need(path, "path"); qph::synth_write(*spec, path, threads); });
}

}  // extern "C"
