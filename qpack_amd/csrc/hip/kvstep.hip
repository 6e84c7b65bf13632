// What a server does to its caches besides kvcache.hip's write, read and attention: append (norms of queries and keys for each head, the position
// rotation, keys and values into the cache, in one pass) and copy (positions from places of one cache to places of another, or of the same).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kvrec.hpp"
#include "launch.hpp"

namespace qph {

namespace {
// ------------------------------------------------------------------ append
// Rows x of head_dim values, w the norm's weights (or none), c and s the cosines and sines of the token's place:
//   y = x w / sqrt(mean(x^2) + eps);  y[i], y[i + half] = y[i] c[i] - y[i + half] s[i], y[i + half] c[i] + y[i] s[i], i < half
// All in fp32, rounded once: queries to their type, keys and values as the cache holds them.
//
// Rows that are stored as they are lie on HD / 8 lanes, 4 dims and those that they are turned with each (pairs_of); what a 4-bit cache takes has the dims of a lane consecutive, as its
// scales and codes want them (turned).  Bound by a launch for a step (a token each of 64 sequences 3.5 us), by HBM for prompts: 4001 tokens of 28 and 2 x 4 heads of 128 dims into an
// fp16 cache, 75 MB, 14.8 us, 5.05 TB/s (8 consecutive dims a lane and their partners loaded too, by twice the instructions 16.7); 2048 of 32 and 2 x 8 into 4 bits 14.9 us, of which some
// 5 are the codes of 2056 records, bound by issue
template <int HD, int EL>
__device__ __forceinline__ float row_sum(float v) {   // over the HD / EL lanes of a row
  static_assert(HD / EL == 8 || HD / EL == 16 || HD / EL == 64, "lanes of a row");
  if constexpr (HD / EL == 64) return wave_sum(v);
  v += dpp_f<kDppQuadXor1>(v);
  v += dpp_f<kDppQuadXor2>(v);
  v += dpp_f<kDppHalfMirror>(v);
  if constexpr (HD / EL == 16) v += dpp_f<kDppMirror>(v);
  return v;
}
template <int T, int N>
__device__ __forceinline__ void load_some(const KvRows &r, int64_t at, float *x) {   // as load_elems, any N
  if constexpr (N % 8 == 0) load_elems<T, N>(r, at, x);
  else {
#pragma unroll
    for (int i = 0; i < N; i++) {
      if constexpr (T == RT_F32) x[i] = ((const float *)r.p)[at + i];
      else { const uint16_t h = ((const uint16_t *)r.p)[at + i]; x[i] = T == RT_F16 ? half_bits_to_float(h) : bf16_to_f(h); }
    }
  }
}
// EL consecutive dims, from d0 on, of a row on HD / EL consecutive lanes.  The pair's other dims lie in another lane: they are loaded as well (from
// L1), which keeps the lanes' order free; half is a multiple of EL, so they too follow each other
template <int HD, int EL, int T>
__device__ __forceinline__ void turned(const KvAppendArgs &a, const KvRows &r, int64_t row, const float *w, int64_t place, int d0, float *y) {
  float x[EL], o[EL], c[EL], s[EL];
  const bool pair = d0 < 2 * a.half, low = d0 < a.half;
  const int d1 = low ? d0 + a.half : d0 - a.half, i0 = low ? d0 : d1;   // the other dims; the pair's number
#pragma unroll
  for (int i = 0; i < EL; i++) o[i] = s[i] = 0.f, c[i] = 1.f;
  load_some<T, EL>(r, row + d0, x);
  if (pair) {
    load_some<T, EL>(r, row + d1, o);
#pragma unroll
    for (int i = 0; i < EL; i++) { c[i] = a.cos_t[place * a.half + i0 + i]; s[i] = a.sin_t[place * a.half + i0 + i]; }
  }
  if (w) {
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < EL; i++) q = __builtin_fmaf(x[i], x[i], q);
    const float f = 1.f / sqrtf(row_sum<HD, EL>(q) * (1.f / HD) + a.eps);
#pragma unroll
    for (int i = 0; i < EL; i++) x[i] = x[i] * f * w[d0 + i];
    if (pair) {
#pragma unroll
      for (int i = 0; i < EL; i++) o[i] = o[i] * f * w[d1 + i];
    }
  }
  // (a dim that has no pair is x itself, whatever it is: 0 x NaN and -0 + 0 would change it)
#pragma unroll
  for (int i = 0; i < EL; i++) y[i] = pair ? __builtin_fmaf(x[i], c[i], low ? -(o[i] * s[i]) : o[i] * s[i]) : x[i];
}
// Lane j of a row's HD / 8 has dims d .. d + 3 and e .. e + 3: a pair's, d + half = e, or 8 consecutive ones behind the pairs.  `mine`: the row takes part (all
// its lanes alike)
struct Pairs { int d, e; float x[4], y[4]; };
template <int T>
__device__ __forceinline__ void load_four(const KvRows &r, int64_t at, float *x) {
  if constexpr (T == RT_F32) load_elems<T, 4>(r, at, x);
  else {
    const u32x2 v = *(const u32x2_any *)((const uint16_t *)r.p + at);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint16_t h = (uint16_t)(v[i / 2] >> 16 * (i & 1));
      x[i] = T == RT_F16 ? half_bits_to_float(h) : bf16_to_f(h);
    }
  }
}
template <int HD, int T>
__device__ __forceinline__ Pairs pairs_of(const KvAppendArgs &a, const KvRows &r, int64_t row, const float *w, int64_t place, int j, bool mine) {
  Pairs p;
  const bool pair = 4 * j < a.half;
  p.d = pair ? 4 * j : 8 * j;   // (behind the pairs: 2 half + 8 (j - half / 4))
  p.e = pair ? 4 * j + a.half : 8 * j + 4;
  float c[4], s[4];
#pragma unroll
  for (int i = 0; i < 4; i++) p.x[i] = p.y[i] = s[i] = 0.f, c[i] = 1.f;
  if (mine) {
    load_four<T>(r, row + p.d, p.x);
    load_four<T>(r, row + p.e, p.y);
    if (pair) {
      const KvRows ct{(void *)a.cos_t, RT_F32, 0, 0, 0}, st{(void *)a.sin_t, RT_F32, 0, 0, 0};
      load_four<RT_F32>(ct, place * a.half + p.d, c);
      load_four<RT_F32>(st, place * a.half + p.d, s);
    }
  }
  if (w) {
    float q = 0.f, u[4], v[4];
    const KvRows wt{(void *)w, RT_F32, 0, 0, 0};
    load_four<RT_F32>(wt, p.d, u);
    load_four<RT_F32>(wt, p.e, v);
#pragma unroll
    for (int i = 0; i < 4; i++) q = __builtin_fmaf(p.y[i], p.y[i], __builtin_fmaf(p.x[i], p.x[i], q));
    const float f = 1.f / sqrtf(row_sum<HD, 8>(q) * (1.f / HD) + a.eps);
#pragma unroll
    for (int i = 0; i < 4; i++) { p.x[i] = p.x[i] * f * u[i]; p.y[i] = p.y[i] * f * v[i]; }
  }
  if (pair) {   // (others are themselves, whatever they are: 0 x NaN and -0 + 0 would change them)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float x = p.x[i], y = p.y[i];
      p.x[i] = __builtin_fmaf(x, c[i], -(y * s[i]));
      p.y[i] = __builtin_fmaf(y, c[i], x * s[i]);
    }
  }
  return p;
}
// a sequence's first position and place, and its tokens that take part
struct Seq { int P0, at; int64_t cnt; };
__device__ __forceinline__ Seq seq_of(const KvAppendArgs &a, int b) {
  Seq s;
  s.P0 = a.io.pos[b];
  s.at = a.at ? a.at[b] : s.P0;
  s.cnt = s.P0 < 0 || s.at < 0 ? 0 : min(min((int64_t)tokens_of(a.io.lens, b, a.io.n), a.io.ctx - s.P0), a.places - s.at);
  return s;
}
// the query rows i = token x heads + head, a row on HD / 8 lanes
template <int HD, int T>
__device__ __forceinline__ void query(const KvAppendArgs &a, const Seq &s, int b, int i, int lane) {
  const int t = i / a.heads, h = i - t * a.heads;
  const bool mine = t < s.cnt;
  const Pairs p = pairs_of<HD, T>(a, a.q, b * a.q.seq + (int64_t)t * a.q.tok + (int64_t)h * a.q.head, a.qw, (int64_t)s.at + t, lane % (HD / 8), mine);
  if (!mine) return;
  const int64_t o = b * a.out.seq + (int64_t)t * a.out.tok + (int64_t)h * a.out.head;
  store_elems<T, 4>(a.out, o + p.d, p.x);
  store_elems<T, 4>(a.out, o + p.e, p.y);
}

// an fp16 cache: the rows of a token - queries, keys, values - one after the other, 8 dims a thread
template <int HD, int T>
__global__ __launch_bounds__(256) void k_append16(KvAppendArgs a) {
  const int b = blockIdx.z, per = a.heads + 2 * a.io.nkv, lane = threadIdx.x & 63;
  const Seq s = seq_of(a, b);
  const int i = blockIdx.x * (256 * 8 / HD) + threadIdx.x / (HD / 8), t = i / per, h = i - t * per;
  if (t >= s.cnt) return;   // (whole rows)
  if (h < a.heads) {
    query<HD, T>(a, s, b, t * a.heads + h, lane);
    return;
  }
  const bool v = h >= a.heads + a.io.nkv;
  const int g = h - a.heads - (v ? a.io.nkv : 0);
  uint16_t *o = (uint16_t *)(v ? a.io.cache_v : a.io.cache) + b * a.io.cseq + ((int64_t)s.P0 + t) * a.io.crow + g * HD;
  auto halves = [](float x, float y) { return float_to_half_bits(x) | (uint32_t)float_to_half_bits(y) << 16; };
  if (v) {
    const int d0 = 8 * (lane % (HD / 8));
    float y[8];
    load_elems<T, 8>(a.io.v, b * a.io.v.seq + (int64_t)t * a.io.v.tok + (int64_t)g * a.io.v.head + d0, y);
    *(u32x4 *)(o + d0) = (u32x4){halves(y[0], y[1]), halves(y[2], y[3]), halves(y[4], y[5]), halves(y[6], y[7])};
  } else {
    const Pairs p = pairs_of<HD, T>(a, a.io.k, b * a.io.k.seq + (int64_t)t * a.io.k.tok + (int64_t)g * a.io.k.head, a.kw, (int64_t)s.at + t, lane % (HD / 8), true);
    *(u32x2 *)(o + p.d) = (u32x2){halves(p.x[0], p.x[1]), halves(p.x[2], p.x[3])};
    *(u32x2 *)(o + p.e) = (u32x2){halves(p.y[0], p.y[1]), halves(p.y[2], p.y[3])};
  }
}

// a 4-bit cache: the first workgroups have a record each (ONE: one token a sequence, a position), waves K and V as k_kv4_write's and k_kv4_write1's; the
// others query rows
template <int HD, int T, bool ONE>
__global__ __launch_bounds__(128) void k_append4(KvAppendArgs a, int records) {
  __shared__ __align__(16) uint8_t codes[kRec][HD];
  const int b = blockIdx.z, lane = threadIdx.x & 63, vside = threadIdx.x >> 6;
  const Seq s = seq_of(a, b);
  if (s.cnt <= 0) return;
  if ((int)blockIdx.x >= records) {
    const int i = (blockIdx.x - records) * (128 * 8 / HD) + threadIdx.x / (HD / 8);
    if (i / a.heads < s.cnt) query<HD, T>(a, s, b, i, lane);
    return;
  }
  const int g = blockIdx.x % (uint32_t)a.io.nkv;
  const int64_t rec = s.P0 / kRec + (int64_t)(blockIdx.x / (uint32_t)a.io.nkv), last = s.P0 + s.cnt;
  if (rec * kRec >= last) return;
  uint8_t *o = (uint8_t *)a.io.cache + (((int64_t)b * a.io.nkv + g) * a.io.nrec + rec) * (9 * HD);
  const KvRows &r = vside ? a.io.v : a.io.k;
  if constexpr (ONE) {
    constexpr int EL = HD / 64;
    const int64_t row = b * r.seq + g * r.head;
    float x[EL];
    if (vside) { load_some<T, EL>(r, row + EL * lane, x); store_one<HD, T>(o, s.P0 % kRec, x, true, lane); }
    else { turned<HD, EL, T>(a, r, row, a.kw, s.at, EL * lane, x); store_one<HD, RT_F32>(o, s.P0 % kRec, x, false, lane); }
  } else {
    constexpr int EL = HD / 8;
    const int row = lane >> 3, part = lane & 7;
    const int64_t p = rec * kRec + row, t = p - s.P0, at = b * r.seq + t * r.tok + g * r.head;
    const bool mine = p >= s.P0 && p < last;
    auto record = [&]() { return o; };
    if (vside) store_record<HD, T>([&](float *x) { load_elems<T, EL>(r, at + EL * part, x); }, record, mine, true, row, part, rec * kRec, s.P0, last, codes);
    else store_record<HD, RT_F32>([&](float *x) { turned<HD, EL, T>(a, r, at, a.kw, s.at + t, EL * part, x); }, record, mine, false, row, part, rec * kRec, s.P0, last, codes);
  }
}

// ------------------------------------------------------------------ copy
// Position pos[b] + t of sequence b becomes position index[b][t] of the source's sequence seqs[b].  What lies outside either cache takes no part
struct Place { int seq, p; };   // the source's; p < 0: none
__device__ __forceinline__ Place place_of(const KvCopyArgs &a, int b, int t) {
  Place s{a.seqs ? a.seqs[b] : b, a.index[b * a.index_seq + t]};
  const int P0 = a.pos[b];
  if (P0 < 0 || t >= tokens_of(a.lens, b, a.n) || (int64_t)P0 + t >= a.ctx || s.seq < 0 || s.seq >= a.src_nseq || s.p >= a.src_ctx) s.p = -1;
  return s;
}
// By way of scratch (what is read and what is written may be the same memory): STAGE 1 gathers the rows into scratch, position t of sequence b, 2 brings
// them from there; 0 does both at once
template <int STAGE, bool ONCE>
__global__ __launch_bounds__(256) void k_copy16(KvCopyArgs a) {
  const int b = blockIdx.z, per = a.nkv * a.hd / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, t = i / per;
  if (t >= a.n) return;
  const int d = 8 * (int)(i - t * per);
  const Place s = place_of(a, b, (int)t);
  if (s.p < 0) return;
  const int64_t staged = (((int64_t)blockIdx.y * a.nseq + b) * a.n + t) * (8 * per) + d;
  const uint16_t *src = STAGE == 2 ? (const uint16_t *)a.work + staged : (const uint16_t *)(blockIdx.y ? a.src_v : a.src) + s.seq * a.src_cseq + (int64_t)s.p * a.src_crow + d;
  uint16_t *dst = STAGE == 1 ? (uint16_t *)a.work + staged : (uint16_t *)(blockIdx.y ? a.cache_v : a.cache) + b * a.cseq + ((int64_t)a.pos[b] + t) * a.crow + d;
  // ONCE: where no sources are named each picks from its own, and what is picked is read once: past the caches, 4096 of 16384 positions of 4 sequences, 134 MB, 28.4 -> 24.2 us, with the attention that
  // reads them 42.6 -> 41.8.  (A fork of 4000 positions into 8 27.6 -> 43 that way; stores past the caches 28.4 -> 23.7, with that attention 45.6)
  *(u32x4 *)dst = ONCE ? __builtin_nontemporal_load((const u32x4 *)src) : *(const u32x4 *)src;
}
// A workgroup has RECS records of one kv head, and a thread a position to look up.  Records that come from one whole record, as all but the last of a fork do, are
// copied as they are, 16 bytes a thread.  Of others a wave has one: lanes 0 .. have 16 bytes of a position's K, lanes 32 .. four words of V, whose
// 8 codes come from a word each of up to 8 records; V words that hold positions outside the call are merged.  Bound by HBM: 6001 positions of 8 heads of 128 dims
// forked into 8 sequences, 62 MB, 12.3 us, 5.1 TB/s.  Where positions are picked too: a V word holds 8 positions, so nine tenths of the source's V are read for a quarter of its positions, 4000 of 16384 of 16 sequences some
// 250 MB for 147 of what is picked and written, 48 of 58.8 us
template <int HD, int STAGE, int RECS>
__global__ __launch_bounds__(256) void k_copy4(KvCopyArgs a) {
  constexpr int P = 9 * HD / 16, NP = (RECS * P + 255) / 256;   // 16-byte pieces of a record, of a thread
  __shared__ int place[RECS * kRec], whole[RECS];   // where positions come from; whole records' first, -1: of several, -2: none
  const int b = blockIdx.z, g = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int P0 = a.pos[b];
  if (P0 < 0) return;
  const int64_t rec = (STAGE == 1 ? 0 : P0 / kRec) + (int64_t)blockIdx.x * RECS;   // in scratch tokens lie from position 0 on
  const int64_t t0 = rec * kRec - (STAGE == 1 ? 0 : P0), wrec = (a.n + kRec - 1) / kRec;
  const int64_t head = (int64_t)b * a.nkv + g;
  uint8_t *dst = STAGE == 1 ? (uint8_t *)a.work + (head * wrec + rec) * (9 * HD) : (uint8_t *)a.cache + (head * a.nrec + rec) * (9 * HD);
  const uint8_t *src;
  {
    const int64_t t = t0 + tid;
    const bool mine = tid < RECS * kRec;
    const Place s = mine && t >= 0 && t < a.n ? place_of(a, b, (int)t) : Place{0, -1};
    const int p = s.p < 0 ? -1 : STAGE == 2 ? (int)t : s.p, p0 = __shfl(p, lane & ~7);
    if (mine) place[tid] = p;
    const uint32_t there = (uint32_t)(__ballot(p >= 0) >> (lane & ~7)) & 255, run = (uint32_t)(__ballot(p >= 0 && p == p0 + (lane & 7) && p0 % kRec == 0) >> (lane & ~7)) & 255;
    if (mine && (lane & 7) == 0) whole[tid / kRec] = run == 255 ? p0 : there ? -1 : -2;
    const int seq = a.seqs ? a.seqs[b] : b;   // (outside the source: no position is there)
    src = STAGE == 2 ? (const uint8_t *)a.work + head * wrec * (9 * HD) : (const uint8_t *)a.src + ((int64_t)seq * a.nkv + g) * a.src_nrec * (9 * HD);
  }
  __syncthreads();
  u32x4 piece[NP];
#pragma unroll
  for (int i = 0; i < NP; i++) {
    const int id = tid + 256 * i, r = id / P;
    const int from = r < RECS ? whole[r] : -1;
    if (from >= 0) piece[i] = *(const u32x4 *)(src + (int64_t)(from / kRec) * (9 * HD) + id % P * 16);
  }
#pragma unroll
  for (int i = 0; i < NP; i++) {
    const int id = tid + 256 * i, r = id / P;
    if (r < RECS && whole[r] >= 0) *(u32x4 *)(dst + id * 16) = piece[i];
  }
  for (int r = tid / 64; r < RECS; r += 4) {
    if (whole[r] != -1) continue;
    const int *at = place + kRec * r;
    uint8_t *o = dst + r * (9 * HD);
    const bool v = lane >= 32;
    const int l = lane & 31, j = l / (HD / 32);   // (K: the position; the piece of its row is l % (HD / 32))
    u32x4 w = {0, 0, 0, 0};
    uint32_t keep = 0;
    uint16_t sc[2] = {0, 0};
    auto record = [&](int p) { return src + (int64_t)(p / kRec) * (9 * HD); };
    if (l < HD / 4) {
      if (v) {
        u32x4 x[kRec], old = *(const u32x4 *)(o + 4 * HD + 16 * l);
#pragma unroll
        for (int k = 0; k < kRec; k++) x[k] = at[k] >= 0 ? *(const u32x4 *)(record(at[k]) + 4 * HD + 16 * l) : (u32x4){0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < kRec; k++) {
          const int q = at[k] & 7;
          if (at[k] < 0) keep |= 15u << nib(k);
          w |= (x[k] >> (uint32_t)(16 * (q & 1) + 4 * (q >> 1)) & 15u) << (uint32_t)nib(k);
        }
        w = (w & ~keep) | (old & keep);
      } else if (at[j] >= 0) {
        w = *(const u32x4 *)(record(at[j]) + at[j] % kRec * (HD / 2) + l % (HD / 32) * 16);
      }
    }
    // the scales: of position lane % 8 and group lane / 8 of K, then of V
    const int k = lane & 7, q = lane >> 3;
    const bool scale = q < HD / 32 && at[k] >= 0;
    if (scale) {
      const uint8_t *x = record(at[k]) + 8 * HD;
      sc[0] = *(const uint16_t *)(x + 2 * (at[k] % kRec * (HD / 32) + q));
      sc[1] = *(const uint16_t *)(x + HD / 2 + 2 * (q * kRec + at[k] % kRec));
    }
    if (l < HD / 4) {
      if (v) *(u32x4 *)(o + 4 * HD + 16 * l) = w;
      else if (at[j] >= 0) *(u32x4 *)(o + 16 * l) = w;
    }
    if (scale) {
      *(uint16_t *)(o + 8 * HD + 2 * (k * (HD / 32) + q)) = sc[0];
      *(uint16_t *)(o + 8 * HD + HD / 2 + 2 * (q * kRec + k)) = sc[1];
    }
  }
}
}  // namespace

hipError_t launch_kv_append(int kind, const KvAppendArgs &a, hipStream_t st) {
  const int64_t rows = (int64_t)a.io.n * (kind == MK_Q4 ? a.heads : a.heads + 2 * a.io.nkv), threads = kind == MK_Q4 ? 128 : 256;
  const int64_t blocks = (rows * (a.io.hd / 8) + threads - 1) / threads;
  const int records = kind != MK_Q4 ? 0 : a.io.n == 1 ? a.io.nkv : ((a.io.n + kRec - 1) / kRec + 1) * a.io.nkv;
  const dim3 grid((unsigned)(records + blocks), 1, a.io.nseq), thr((unsigned)threads);
#define QPH_APPEND(HD, T)                                                                                  \
  do {                                                                                                     \
    if (kind != MK_Q4) hipLaunchKernelGGL((k_append16<HD, T>), grid, thr, 0, st, a);                       \
    else if (a.io.n == 1) hipLaunchKernelGGL((k_append4<HD, T, true>), grid, thr, 0, st, a, records);      \
    else hipLaunchKernelGGL((k_append4<HD, T, false>), grid, thr, 0, st, a, records);                      \
  } while (0)
  if (a.io.hd == 128) {
    if (a.q.type == RT_F32) QPH_APPEND(128, RT_F32);
    else if (a.q.type == RT_F16) QPH_APPEND(128, RT_F16);
    else QPH_APPEND(128, RT_BF16);
  } else {
    if (a.q.type == RT_F32) QPH_APPEND(64, RT_F32);
    else if (a.q.type == RT_F16) QPH_APPEND(64, RT_F16);
    else QPH_APPEND(64, RT_BF16);
  }
#undef QPH_APPEND
  return hipGetLastError();
}

template <int STAGE>
static void launch_copy(int kind, const KvCopyArgs &a, hipStream_t st) {
  if (kind == MK_Q4) {
    const int recs = (a.n + kRec - 1) / kRec + (STAGE == 1 ? 0 : 1);
    // A record a wave up to eight workgroups of two a wave a CU: of 4 sequences' 1000 positions picked from 4000 (8 heads of 128 dims) 5.6 us with one, 6.6 with two, 14.2 with eight; 250
    // forked into 32 6.0, 5.7 and 7.6.  Past them two, 4000 picked for each of 16 57.4, 58.7 and 71.6, but eight where the call names source sequences: they are forked or change
    // places, in whole records as a rule, 6001 positions into 8 14.0, 12.3 and 12.1 (62.8 and 60.8 with the caches read back each time).  Positions
    // that are picked from named sources lose by it: those 4000 70.7 for 58.0 (and 97 for 76 in fp16, whose loads past the caches go by the same)
    auto grid = [&](int each) { return dim3((unsigned)((recs + each - 1) / each), a.nkv, a.nseq); };
#define QPH_COPY(RECS)                                                                                          \
  do {                                                                                                          \
    if (a.hd == 128) hipLaunchKernelGGL((k_copy4<128, STAGE, RECS>), grid(RECS), dim3(256), 0, st, a);          \
    else hipLaunchKernelGGL((k_copy4<64, STAGE, RECS>), grid(RECS), dim3(256), 0, st, a);                       \
  } while (0)
    if ((int64_t)((recs + 7) / 8) * a.nkv * a.nseq <= 2048) QPH_COPY(4);
    else if (!a.seqs) QPH_COPY(8);
    else QPH_COPY(32);
#undef QPH_COPY
  } else {
    const dim3 grid((unsigned)(((int64_t)a.n * a.nkv * a.hd / 8 + 255) / 256), 2, a.nseq);
    if (STAGE != 2 && !a.seqs) hipLaunchKernelGGL((k_copy16<STAGE, STAGE != 2>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_copy16<STAGE, false>), grid, dim3(256), 0, st, a);
  }
}
hipError_t launch_kv_copy(int kind, const KvCopyArgs &a, hipStream_t st) {
  if (!a.work) {
    launch_copy<0>(kind, a, st);
    return hipGetLastError();
  }
  launch_copy<1>(kind, a, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  launch_copy<2>(kind, a, st);
  return hipGetLastError();
}

}  // namespace qph
