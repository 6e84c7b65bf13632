// Key / value caches of several sequences, in fp16 or in 4 bits: writing rows, reading them back, and the attention of new
// tokens over them, all positions or a sliding window with a few first positions that stay visible.
//
// The 4-bit cache.  Each 32 dims of one position's K (V) row share an fp16 scale s: a = max |x|, s = fp16(bf16(min(a, 65504)
// / 7)), code = clamp(rint(x / s), -7, 7) + 8.  s has 8 significant bits and code - 8 three, so every value (code - 8) s is an
// fp16 number: the matrix cores' operands, the rows read back and an fp16 snapshot are exact, and a row read back and
// written again gives the same values, as long as s is 7 x 2^-24 or more: the largest code is then 7, and 7 s / 7 is s again.  (Groups
// whose largest is below 2.4e-6 have scales of a few of fp16's least steps; a largest of 10.7 of them gets s = 2 and code 5, which
// written again is s = 1 and, clamped, 7.)  Rounding s to 8 bits costs at most 2^-9 of it, the codes' step is 2^-3.  A group that holds
// a NaN or an infinity has a NaN scale and reads back as NaN.
//
// One record of 9 HD bytes holds 8 positions of one (sequence, kv head); records follow each other in position order:
//   [0, 4 HD)         K codes: position i at i HD / 2, a row's 32-bit word w = dims 8 w ..: dim 8 w + 2 e + o at bits 16 o + 4 e
//   [4 HD, 8 HD)      V codes: dim d's word (d % 16) (HD / 16) + d / 16: position 2 e + o at bits 16 o + 4 e
//   [8 HD, 8.5 HD)    K scales [8 positions][HD / 32]
//   [8.5 HD, 9 HD)    V scales [HD / 32][8 positions]
// K words run along the dims and V words along the positions because the matrix cores sum K q over dims and P V over
// positions: a lane's word is its fragment, four (mask, or, subtract, multiply) pairs away, with no transposition and no LDS
// on the decode path.  A single stream of records per head keeps a tile of 32 positions in 4.5 KiB of consecutive bytes.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <type_traits>

#include "kvrec.hpp"
#include "launch.hpp"

namespace qph {

namespace {
// ------------------------------------------------------------------ writing and reading
// One wave per record's K, one per its V: lane = position lane / 8 of the record, dims EL (lane % 8) ..  Positions outside the
// call's keep their codes and scales: their K rows and scales are not stored, and the V words, which hold all 8
// positions, are read and merged where the call covers a part only (no other workgroup of the launch has the record).
// 2048 positions of 8 heads of 128 dims, fp16 rows: 4.5 us, a launch (2.4) and 10.8 MB at the copy rate (2.2).
template <int HD, int T>
__global__ __launch_bounds__(128) void k_kv4_write(KvIoArgs a) {
  constexpr int EL = HD / 8;   // elements of a lane
  __shared__ __align__(16) uint8_t codes[kRec][HD];
  const int b = blockIdx.z, g = blockIdx.y, lane = threadIdx.x & 63, vside = threadIdx.x >> 6;
  const int P0 = a.pos[b], cnt = tokens_of(a.lens, b, a.n);
  if (P0 < 0 || cnt <= 0) return;
  const int64_t rec = P0 / kRec + (int64_t)blockIdx.x;
  const int64_t last = min((int64_t)P0 + cnt, a.ctx);   // one past the last position written
  if (rec * kRec >= last) return;
  const int row = lane >> 3, part = lane & 7;
  const int64_t p = rec * kRec + row;
  const bool mine = p >= P0 && p < last;
  const KvRows &r = vside ? a.v : a.k;
  store_record<HD, T>([&](float *x) { load_elems<T, EL>(r, b * r.seq + (p - P0) * r.tok + g * r.head + EL * part, x); },
                      [&]() { return (uint8_t *)a.cache + (((int64_t)b * a.nkv + g) * a.nrec + rec) * (9 * HD); }, mine, vside, row, part, rec * kRec, P0, last, codes);
}

// One token a sequence: a wave has one row of K or V, HD / 64 dims a lane.  Lanes of a K word meet by DPP; a V word is read (as soon as
// the position is known, beside the row) and its one code replaced.  In k_kv4_write such a row would keep 8 lanes of 64 busy: 4.9 us
// against 2.9 for 8 heads of 128 dims, of which 2.4 are the launch (bound by latency: position, word, store)
template <int HD, int T>
__global__ __launch_bounds__(128) void k_kv4_write1(KvIoArgs a) {
  constexpr int EL = HD / 64;
  const int b = blockIdx.z, g = blockIdx.y, lane = threadIdx.x & 63, vside = threadIdx.x >> 6;
  const KvRows &r = vside ? a.v : a.k;
  const int64_t at = b * r.seq + g * r.head + EL * lane;
  float x[EL];
#pragma unroll
  for (int i = 0; i < EL; i++) {
    if constexpr (T == RT_F32) x[i] = ((const float *)r.p)[at + i];
    else { const uint16_t h = ((const uint16_t *)r.p)[at + i]; x[i] = T == RT_F16 ? half_bits_to_float(h) : bf16_to_f(h); }
  }
  const int p = a.pos[b];
  if (p < 0 || p >= a.ctx || tokens_of(a.lens, b, a.n) <= 0) return;
  uint8_t *o = (uint8_t *)a.cache + (((int64_t)b * a.nkv + g) * a.nrec + p / kRec) * (9 * HD);
  store_one<HD, T>(o, p % kRec, x, vside, lane);
}

// The same lanes as k_kv4_write's.  A lane takes its position's code out of each of its dims' V words, which 8 lanes read from L1: 4.7 us for
// 2048 positions of 8 heads of 128 dims, a launch and 10.8 MB at the copy rate (single tokens 2.8)
template <int HD, int T>
__global__ __launch_bounds__(128) void k_kv4_read(KvIoArgs a) {
  constexpr int EL = HD / 8, GL = 32 / EL;
  const int b = blockIdx.z, g = blockIdx.y, lane = threadIdx.x & 63, vside = threadIdx.x >> 6;
  const int P0 = a.pos[b], cnt = tokens_of(a.lens, b, a.n);
  if (P0 < 0 || cnt <= 0) return;
  const int64_t rec = P0 / kRec + (int64_t)blockIdx.x;
  const int row = lane >> 3, part = lane & 7;
  const int64_t p = rec * kRec + row;
  if (p < P0 || p >= min((int64_t)P0 + cnt, a.ctx)) return;
  const uint8_t *o = (const uint8_t *)a.cache + (((int64_t)b * a.nkv + g) * a.nrec + rec) * (9 * HD);
  float x[EL];
  if (!vside) {
    const uint16_t s = *(const uint16_t *)(o + 8 * HD + 2 * (row * (HD / 32) + part / GL));
#pragma unroll
    for (int i = 0; i < EL / 8; i++) {
      const h8 v = values(*(const uint32_t *)(o + row * (HD / 2) + part * (EL / 2) + 4 * i), s);
#pragma unroll
      for (int j = 0; j < 8; j++) x[8 * i + j] = (float)v[j];
    }
  } else {
    const float s = half_bits_to_float(*(const uint16_t *)(o + 8 * HD + HD / 2 + 2 * (part / GL * kRec + row)));
#pragma unroll
    for (int i = 0; i < EL; i++) {
      const int d = EL * part + i;
      const uint32_t w = ((const uint32_t *)(o + 4 * HD))[d % 16 * (HD / 16) + d / 16];
      x[i] = ((int)(w >> (16 * (row & 1) + 4 * (row >> 1)) & 15) - 8) * s;
    }
  }
  const KvRows &r = vside ? a.v : a.k;
  store_elems<T, EL>(r, b * r.seq + (p - P0) * r.tok + g * r.head + EL * part, x);
}

// the fp16 cache's: a copy with a conversion, 8 dims of one position's K or V a thread.  Bound by memory: 16 sequences
// of 16384 positions, 8 heads of 128 dims, 347 us either way (6.2 TB/s read and written; fp32 rows 5.9); 2048 positions by the launch (4 to 6 us)
template <bool WRITE, int T>
__global__ __launch_bounds__(256) void k_kv16_io(KvIoArgs a) {
  const int b = blockIdx.z, per = a.nkv * a.hd / 8;
  const int P0 = a.pos[b], cnt = tokens_of(a.lens, b, a.n);
  if (P0 < 0) return;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, t = i / per, p = P0 + t;
  if (t >= cnt || p >= a.ctx) return;
  const int g = (int)(i % per) / (a.hd / 8), d = 8 * ((int)(i % per) % (a.hd / 8));
  const KvRows &r = blockIdx.y ? a.v : a.k;
  uint16_t *c = (uint16_t *)(blockIdx.y ? a.cache_v : a.cache) + b * a.cseq + p * a.crow + g * a.hd + d;
  const int64_t at = b * r.seq + t * r.tok + g * r.head + d;
  float x[8];
  u32x4 w;
  if (WRITE) {
    load_elems<T, 8>(r, at, x);
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = float_to_half_bits(x[2 * j]) | (uint32_t)float_to_half_bits(x[2 * j + 1]) << 16;
    *(u32x4 *)c = w;
  } else {
    w = *(const u32x4 *)c;
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = half_bits_to_float((uint16_t)(w[j / 2] >> 16 * (j & 1)));
    store_elems<T, 8>(r, at, x);
  }
}

// ------------------------------------------------------------------ what a workgroup of the attention reads
// Columns: a kv head's (token, query head) pairs, the head fastest; a workgroup has a.cols of them, a chunk of sequence b.  The
// records any of its columns may see: the SR first ones (positions below sinks), then from the window's first on; virtual
// record v is v, or v + skip from SR on.
struct Span {
  int P0, cnt;      // the sequence's first new position and its tokens that count
  int PA, PB;       // positions of the workgroup's first and last token
  int ws;           // first position of PA's window
  int SR, skip, NR; // virtual records
  int nt, S;        // tiles, splits in use
  bool any;
};
// The columns of a chunk: a.cols from chunk * a.cols on, or, paired (many tokens, no window), half of them from the front and half from
// the back.  In a prompt a workgroup's time goes with its last position, and pairs take more alike: 2048 tokens of 32 heads 65 -> 55 us (fp32
// 105 -> 88).  Behind a long past there is nothing to even out, and pairs change nothing: 77 tokens of 28 heads at 16000 44 us either way, with 4, 5
// and 8 of a workgroup's waves at work, by the columns that its halves have
__device__ __forceinline__ int chunk_half(const KvAttnArgs &a, int chunk, int h) {   // the first column of half h
  return (a.paired ? (h ? 2 * a.nchunk - 1 - chunk : chunk) : 2 * chunk + h) << a.half_log2;
}
__device__ __forceinline__ int chunk_of(const KvAttnArgs &a, int col) {
  const int u = col >> a.half_log2;
  return a.paired ? min(u, 2 * a.nchunk - 1 - u) : u >> 1;
}
// col / rep (kv_attn_plan's reciprocal): the compiler's divisions, 64-bit ones above all, were a third of a short call's instructions
__device__ __forceinline__ int token_of(const KvAttnArgs &a, int col) {
  return a.rep == 1 ? col : (int)(__umulhi((uint32_t)col, a.rep_mul) >> a.rep_shift);
}
__device__ __forceinline__ int last_token(const KvAttnArgs &a, int first) { return token_of(a, first + (1 << a.half_log2) - 1); }   // of a half
__device__ __forceinline__ Span span_of(const KvAttnArgs &a, int b, int chunk) {
  Span s;
  s.P0 = a.pos[b]; s.cnt = tokens_of(a.lens, b, a.n);
  const int ta = token_of(a, chunk_half(a, chunk, 0)), tb = last_token(a, chunk_half(a, chunk, 1));
  s.any = s.P0 >= 0 && ta < s.cnt && (int64_t)s.P0 + ta < a.ctx;
  s.PA = s.P0 + ta;
  // paired, the back half may lie behind the sequence's tokens while the front half does not reach them
  int te = min(tb, s.cnt - 1);
  if (a.paired && token_of(a, chunk_half(a, chunk, 1)) >= s.cnt) te = min(last_token(a, chunk_half(a, chunk, 0)), s.cnt - 1);
  s.PB = (int)min((int64_t)s.P0 + te, a.ctx - 1);
  s.ws = a.window > 0 ? max(0, s.PA - a.window + 1) : 0;
  const int r0 = s.ws / kRec;
  s.SR = min((int)(((uint32_t)a.sinks + kRec - 1) / kRec), r0);
  s.skip = r0 - s.SR;
  s.NR = s.PB / kRec + 1 - s.skip;
  s.nt = (s.NR + (1 << a.tile_log2) - 1) >> a.tile_log2;
  s.S = s.nt <= a.one_tiles ? 1 : min(a.nsplit, (s.nt + (1 << a.min_log2) - 1) >> a.min_log2);
  return s;
}
// The span of a pass over a common prefix: every column sees all of its positions.  Its columns are (sequence, token, query head), the tokens of all
// sequences counted through, and b is 0
// (through the scalar cache: a vector load of it would be waited for together with those before it)
typedef const int __attribute__((address_space(4))) scalar_int;
__device__ __forceinline__ int prefix_length(const KvPrefix &p) { return p.len ? (int)min((int64_t)max(*(const scalar_int *)(uintptr_t)p.len, 0), p.ctx) : (int)p.ctx; }
__device__ __forceinline__ int splits_of(int nt, int one_tiles, int nsplit, int min_log2) { return nt <= one_tiles ? (int)(nt > 0) : min(nsplit, (nt + (1 << min_log2) - 1) >> min_log2); }
__device__ __forceinline__ Span prefix_span_of(const KvPreArgs &a) {
  Span s;
  const int L = prefix_length(a.prefix);
  s.P0 = 0; s.cnt = a.n; s.any = L > 0;
  s.PA = s.PB = L - 1;
  s.ws = s.SR = s.skip = 0;
  s.NR = (L + kRec - 1) / kRec;
  s.nt = (s.NR + (1 << a.tile_log2) - 1) >> a.tile_log2;
  s.S = splits_of(s.nt, a.one_tiles, a.nsplit, a.min_log2);
  return s;
}
__device__ __forceinline__ int prefix_splits(const KvJoin &p) {
  const int nr = (prefix_length(p.prefix) + kRec - 1) / kRec;
  return splits_of((nr + (1 << p.tile_log2) - 1) >> p.tile_log2, p.one_tiles, p.nsplit, p.min_log2);
}
// a token counted through all sequences, as its sequence's
struct SeqTok { int b, t; };
__device__ __forceinline__ SeqTok seq_tok(const KvPreArgs &a, int tok) {
  const int b = a.prefix.n == 1 ? tok : tok / a.prefix.n;
  return {b, tok - b * a.prefix.n};
}
template <bool PRE> using Args = std::conditional_t<PRE, KvPreArgs, KvAttnArgs>;   // of the kernels below
__device__ __forceinline__ bool takes_part(const KvPreArgs &a, SeqTok x) {
  const int P0 = a.pos[x.b];
  return (P0 >= 0) & (x.t < tokens_of(a.lens, x.b, a.prefix.n)) & ((int64_t)P0 + x.t < a.prefix.own_ctx);
}
// the partial sums of a row: the own positions' first, a prefix's last.  JOIN: of a pass whose sums, one split's too, are joined with another pass's
template <bool JOIN>
__host__ __device__ __forceinline__ int slots_of(const KvAttnArgs &a) { return JOIN ? -a.one_tiles : a.nsplit; }
// the first tile of share i of S (the product fits: nt <= 2^25, i <= 64)
__device__ __forceinline__ int share(const Span &s, int i) { return s.S == 1 ? i * s.nt : (int)((uint32_t)i * (uint32_t)s.nt / (uint32_t)s.S); }
__device__ __forceinline__ int record(const Span &s, int v) { return v < s.SR ? v : v + s.skip; }
// whether the token at P, whose window starts behind lo, sees position p (no short cuts: these are lanes' values)
__device__ __forceinline__ int behind(const KvAttnArgs &a, int P) { return a.window > 0 ? P - a.window : -1; }
__device__ __forceinline__ bool sees(const KvAttnArgs &a, int P, int lo, int p) { return (p <= P) & ((p > lo) | (p < a.sinks)); }
// bits of the positions p0 + j, j < 8, that some token of the workgroup sees
__device__ __forceinline__ uint32_t seen_bits(const KvAttnArgs &a, const Span &s, int v, int p0) {
  uint32_t on = 0;
#pragma unroll
  for (int j = 0; j < kRec; j++) on |= (uint32_t)((p0 + j <= s.PB) & ((p0 + j >= s.ws) | (p0 + j < a.sinks))) << j;
  return v < s.NR ? on : 0;
}

// fp16 queries are the matrix cores' operands as they are.  Others enter as fp16, each row scaled by the power of two that brings its largest magnitude into [1, 2), or [2, 4)
// from 2^127 on, where that power is no normal number: bf16 values keep every bit that is not 2^-25 below that (fp32 ones go in two halves, hi + lo, and keep 22 bits).  The power
// returns with the softmax scale, in fp32.
__device__ __forceinline__ float row_power(float mx) {   // 2^-e, 2^-126 at the least; 1 for rows that are zero or not finite
  const uint32_t e = __builtin_bit_cast(uint32_t, mx) >> 23;
  return e == 0 || e == 255 ? 1.f : __builtin_bit_cast(float, (254u - min(e, 253u)) << 23);
}
// Probabilities are held as 2^(x - m + kPBias), where m is a column's maximum as it was when it was last looked for: when there was none,
// and whenever a lane's weights of a tile add up to more than kRoom.  They stay in fp16's range, what lies 2^-32 below m is
// still there, and the sum they are divided by is scaled alike.
constexpr float kPBias = 8.f, kRoom = 32768.f;
// The least and the largest softmax factor of a row: with 0 a masked score would be -inf x 0, with inf a score of 0 would be NaN.  The scores
// that the least takes, up to 2^25, stay below 2^-100
constexpr float kTinyF = 0x1p-126f, kMostF = 0x1.fffffep127f;

// ------------------------------------------------------------------ few tokens
// Grid (split, kv head and column chunk, sequence), 8 waves, each streaming its own tiles of 32 positions (4 records) with
// the next tile's loads in flight.
//   scores  S^T[p][c] = K[p] . q[c] on v_mfma_f32_16x16x32_f16, A = K rows, B = q^T with 16 columns.  Row r of tile half mt is
//           position 8 (r / 4) + 4 mt + r % 4, so the C layout leaves lane group lg = lane / 16 the 8 positions of record lg.
//   values  O^T[d][c] += V^T[d][p] P^T[p][c]: those 8 probabilities are the lane's B fragment as they are, and the A
//           fragment is dim 16 t + lane % 16 of record lg: one word of V codes.
// Why 16 columns and, for 4-bit, no LDS: the heads of a kv group leave much of a product's columns empty, but the cache is read once for
// all of them, and that is what the time goes with: a batch of 32 sequences of up to 8K positions (8 kv heads of 128 dims, 4 heads
// each) 43 us, 4.85 TB/s where a large copy reaches 4.99.  One sequence of 16K is latency (position, first codes, a tile a wave, the
// waves' sums): 6.4 us for 1.9 of bytes.  fp16 V goes through LDS, since the product wants it transposed.
// Splits (kv_attn_plan): up to 1024 positions a sequence is one workgroup's, whose waves meet in LDS, since the merge is a launch of 3.9 us
// (332 positions: 9.4 -> 5.7 us); above, two workgroups a CU, of at least 256 positions each.  A window makes them fewer alike
// TWO (fp32 queries): 8 columns, with the queries' hi halves in columns 0 .. 7 and their lo halves in 8 .. 15 of the same
// product, and P's likewise: 22 bits for the price of 11 where no more than 8 columns are needed.
constexpr int kFewWaves = 8, kFewTile = 32, kFewOcc = 4;   // waves of a workgroup, positions of a tile, waves of a SIMD

template <int HD, int KIND>
struct Tile;
template <int HD>
struct Tile<HD, MK_Q4> {   // a lane's words of a tile: two K row pieces, its V dims of one record
  static constexpr int KW = HD / 32, VW = HD / 16;
  uint32_t k[2][KW], v[VW];
  uint16_t ks[2];
  u32x4 vs[HD / 32];
};
template <int HD>
struct Tile<HD, MK_F32> { u32x4 k[2][HD / 32]; };   // an fp16 cache's K; its V goes to LDS
// a workgroup's part of the cache: its kv head's records, or its rows
struct Head { const uint8_t *rec; const uint16_t *k, *v; };
template <int HD, int KIND>
__device__ __forceinline__ Head head_of(const KvAttnArgs &a, int b, int g) {
  Head h{};
  if constexpr (KIND == MK_Q4) h.rec = (const uint8_t *)a.cache + ((int64_t)b * a.nkv + g) * a.nrec * (9 * HD);
  else { h.k = (const uint16_t *)a.cache + b * a.cseq + g * HD; h.v = (const uint16_t *)a.cache_v + b * a.cseq + g * HD; }
  return h;
}
// records and positions past the span's are the last one's (masked, and in the allocation)
template <typename A>   // (A: ctx, crow)
__device__ __forceinline__ int64_t row_of(const A &a, const Span &s, int v, int j) {
  return min((int64_t)kRec * record(s, min(v, s.NR - 1)) + j, a.ctx - 1) * a.crow;
}
// whether records v .. v + n - 1 are there and follow each other
__device__ __forceinline__ bool run_of(const Span &s, int v, int n) { return v + n <= s.NR && (s.skip == 0 || v >= s.SR || v + n <= s.SR); }
// a 4-bit tile's loads: a scalar base and offsets that a lane keeps where its records follow each other (all tiles but a few)
template <int HD>
__device__ __forceinline__ const uint8_t *tile_base(const Head &h, const Span &s, int tile, bool run, int r) {   // r: the lane's record of the tile
  return h.rec + (run ? (int64_t)record(s, 4 * tile) : (int64_t)record(s, min(4 * tile + r, s.NR - 1)) - r) * (9 * HD);
}
template <int HD, int KIND, typename A>
__device__ __forceinline__ void load_k(const A &a, const Head &h, const Span &s, int tile, int lane, Tile<HD, KIND> &t) {
  const int lr = lane & 15, lg = lane >> 4;
  if constexpr (KIND == MK_Q4) {
    const uint32_t ko = (lr >> 2) * (9 * HD) + (lr & 3) * (HD / 2) + lg * (HD / 8), so = (lr >> 2) * (9 * HD) + 8 * HD + 2 * ((lr & 3) * (HD / 32) + lg * HD / 128);
    auto get = [&](const uint8_t *r) {
#pragma unroll
      for (int mt = 0; mt < 2; mt++) {
        const uint8_t *kp = r + (ko + mt * 2 * HD);
        if constexpr (HD == 128) { const u32x4 x = *(const u32x4 *)kp; t.k[mt][0] = x[0]; t.k[mt][1] = x[1]; t.k[mt][2] = x[2]; t.k[mt][3] = x[3]; }
        else { const u32x2 x = *(const u32x2 *)kp; t.k[mt][0] = x[0]; t.k[mt][1] = x[1]; }
        t.ks[mt] = *(const uint16_t *)(r + (so + mt * (HD / 4)));
      }
    };
    if (run_of(s, 4 * tile, 4)) get(tile_base<HD>(h, s, tile, true, 0));
    else get(tile_base<HD>(h, s, tile, false, lr >> 2));
  } else {
#pragma unroll
    for (int mt = 0; mt < 2; mt++) {
      const uint16_t *r = h.k + row_of(a, s, 4 * tile + (lr >> 2), 4 * mt + (lr & 3)) + 8 * lg;
#pragma unroll
      for (int k = 0; k < HD / 32; k++) t.k[mt][k] = *(const u32x4 *)(r + 32 * k);
    }
  }
}
// 16-byte segment c of V row x sits at c ^ vsw(x): the 8 rows that the 32 lanes of a transpose read address (0 .. 3 or 4 .. 7 of two
// records) cover all banks
template <int HD>
__device__ __forceinline__ int vsw(int x) { return HD == 128 ? 2 * ((x & 3) | (x >> 1 & 4)) : 2 * ((x >> 1 & 1) | (x >> 2 & 2)); }
template <int HD, int KIND, typename A>
__device__ __forceinline__ void load_v(const A &a, const Head &h, const Span &s, int tile, int lane, Tile<HD, KIND> &t, uint16_t *buf) {
  const int lr = lane & 15, lg = lane >> 4;
  if constexpr (KIND == MK_Q4) {
    const uint32_t vo = lg * (9 * HD) + 4 * HD + lr * (HD / 4), so = lg * (9 * HD) + 8 * HD + HD / 2;
    auto get = [&](const uint8_t *r) {
#pragma unroll
      for (int i = 0; i < HD / 64; i++) {
        const u32x4 x = *(const u32x4 *)(r + (vo + 16 * i));
#pragma unroll
        for (int j = 0; j < 4; j++) t.v[4 * i + j] = x[j];
      }
#pragma unroll
      for (int i = 0; i < HD / 32; i++) t.vs[i] = *(const u32x4 *)(r + (so + 16 * i));
    };
    if (run_of(s, 4 * tile, 4)) get(tile_base<HD>(h, s, tile, true, 0));
    else get(tile_base<HD>(h, s, tile, false, lg));
  } else {
    constexpr int SEG = HD / 8, RPI = 64 / SEG;   // 16-byte segments of a row, rows of a 1 KiB load
#pragma unroll
    for (int q = 0; q < kFewTile / RPI; q++) {
      const int x = q * RPI + lane / SEG;
      dma16(h.v + row_of(a, s, 4 * tile + x / kRec, x % kRec) + 8 * (lane % SEG ^ vsw<HD>(x)), buf + q * RPI * HD);
    }
  }
}

// bits of the elements of v that are NaN or infinite
__device__ __forceinline__ uint32_t not_finite(u32x4 w) {
  uint32_t bad = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) bad |= ((w[i] & 0x7c00u) == 0x7c00u ? 1u << 2 * i : 0u) | ((w[i] & 0x7c000000u) == 0x7c000000u ? 2u << 2 * i : 0u);
  return bad;
}
// v with the elements of clear bits of `on` zeroed
__device__ __forceinline__ h8 only(h8 v, uint32_t on) {
  u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
  for (int i = 0; i < 4; i++) w[i] &= (on >> 2 * i & 1 ? 0xffffu : 0u) | (on >> (2 * i + 1) & 1 ? 0xffff0000u : 0u);
  return __builtin_bit_cast(h8, w);
}
// Where some columns see a position and others don't, its V enters the product without its NaN and infinite values, which
// would reach every column through 0 x NaN.  They are then added to the columns that see the position, read again from
// memory: o's dims d .. d + 3 (4-bit: a group's scale is what can be NaN)
template <int HD, int KIND, typename V>
__device__ __forceinline__ void add_bad(const uint8_t *rec, const uint16_t *row, int p, int d, bool sees, V &o, int i0) {
  if constexpr (KIND == MK_Q4) {
    const uint16_t s = *(const uint16_t *)(rec + 8 * HD + HD / 2 + 16 * (d / 32) + 2 * (p % kRec));
    if (sees && (s & 0x7c00) == 0x7c00) {
#pragma unroll
      for (int i = 0; i < 4; i++) o[i0 + i] += __builtin_nanf("");
    }
  } else {
    const u32x2 w = *(const u32x2 *)(row + d);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint16_t h = (uint16_t)(w[i / 2] >> 16 * (i & 1));
      if (sees && (h & 0x7c00) == 0x7c00) o[i0 + i] += half_bits_to_float(h);
    }
  }
}

template <int HD, int KIND, int T>
constexpr int few_lds() {   // bytes: V's tiles, then the waves' sums
  constexpr int tiles = KIND == MK_Q4 ? 0 : kFewWaves * kFewTile * HD * 2, out = kFewWaves * (T == RT_F32 ? 8 : 16) * (HD + 4) * 4;
  return tiles > out ? tiles : out;
}
template <int T> using few_cols = float[kFewWaves][T == RT_F32 ? 8 : 16];   // the waves' maxima, sums
#define KV_OWN 0
#define KV_SPAN(t) s
#define KV_HEAD(t) h
#define KV_MEM(t) a
#define KV_TILE(t) (t)
#define KV_P(t) P
template <int HD, int KIND, int T, bool PRE = false, bool JOIN = false, bool ALL = false>   // (of the body)
__global__ __launch_bounds__(kFewWaves * 64, kFewOcc) void k_kv_few(Args<PRE> a) {
  __shared__ __align__(16) uint8_t sm[few_lds<HD, KIND, T>()];
  __shared__ few_cols<T> wm, wl;
  const int split = blockIdx.x, gc = blockIdx.y, b = blockIdx.z;
#include "kv_few.inc"
}
// LDS of functions within one kernel: the same for the same arguments
template <typename X, int I = 0>
__device__ __forceinline__ X &lds() {
  __shared__ __align__(16) X x;
  return x;
}
// the same within a kernel that has other work beside it (PRE: over a common prefix; below) and LDS bytes for either.  (The arguments by value and LDS by its
// name: by reference that kernel spills)
template <int HD, int KIND, int T, bool PRE, int LDS, bool JOIN = true, bool ALL = false>
__device__ __forceinline__ void few_tokens(Args<PRE> a, int split, int gc, int b) {
  auto &sm = lds<uint8_t[LDS]>();
  auto &wm = lds<few_cols<T>, 0>(), &wl = lds<few_cols<T>, 1>();
  if constexpr (PRE) a.window = a.sinks = a.paired = 0;
#include "kv_few.inc"
}

#undef KV_OWN
#undef KV_SPAN
#undef KV_HEAD
#undef KV_MEM
#undef KV_TILE
#undef KV_P
// A sequence's columns over a common prefix's tiles and then its own, without sums to be joined: a launch and their way through memory are saved, and the prefix is read for each
// sequence anew (kv_prefix_plan).  4 samples behind 700 positions 9.5 -> 8.9 us, 53 sequences of 3 tokens behind 37 13.2 -> 5.6
#define KV_OWN own
#define KV_SPAN(t) ((t) < own ? pspan : s)
#define KV_HEAD(t) ((t) < own ? phead : h)
#define KV_MEM(t) ((t) < own ? mp : mo)
#define KV_TILE(t) ((t) < own ? (t) : (t) - own)
#define KV_P(t) ((t) < own ? live ? pspan.PB : -1 : P)
struct KvMem { int64_t ctx, crow; };
template <int HD, int KIND, int T, bool PRE = false, bool JOIN = false, bool ALL = true>
__global__ __launch_bounds__(kFewWaves * 64, kFewOcc) void k_kv_few_all(Args<PRE> a, KvPreArgs pre) {
  __shared__ __align__(16) uint8_t sm[few_lds<HD, KIND, T>()];
  __shared__ few_cols<T> wm, wl;
  a.window = a.sinks = a.paired = 0;
  const Span pspan = prefix_span_of(pre);
  const int own = pspan.nt;   // the first of the own tiles
  const KvMem mp{pre.ctx, pre.crow}, mo{a.ctx, a.crow};
  const int split = 0, gc = blockIdx.y, b = blockIdx.z;
  const Head phead = head_of<HD, KIND>(pre, 0, a.nchunk == 1 ? gc : gc / (uint32_t)a.nchunk);
#include "kv_few.inc"
}
#undef KV_OWN
#undef KV_SPAN
#undef KV_HEAD
#undef KV_MEM
#undef KV_TILE
#undef KV_P

// The splits' sums of one row a workgroup: 256 threads, HD / 4 of them side by side over the dims, the others over the
// splits.  M = max m, L = sum l 2^(m - M), out = sum o 2^(m - M) / L.  Bound by latency: 3.9 us for 28 rows of 64 splits, 2.4 of them the
// launch.  (All loads asked for before M is known: no faster)
template <int HD, int T>
__global__ __launch_bounds__(256) void k_kv_merge(KvAttnArgs a) {
  constexpr int CT = HD / 4, SL = 256 / CT;
  __shared__ f32x4 oo[SL][CT];
  const int head = blockIdx.x, tok = blockIdx.y, b = blockIdx.z, g = token_of(a, head);
  const int col = tok * a.rep + head - g * a.rep;
  const Span s = span_of(a, b, chunk_of(a, col));
  if (!s.any || s.S == 1 || tok >= s.cnt || (int64_t)s.P0 + tok >= a.ctx) return;
  const int64_t row = ((int64_t)b * a.n + tok) * a.heads + head;
  const float2 *ml = (const float2 *)(a.part + (int64_t)a.nseq * a.n * a.heads * a.nsplit * HD) + row * a.nsplit;
  const float *po = a.part + row * a.nsplit * HD;
  const int ct = threadIdx.x % CT, sl = threadIdx.x / CT, lane = threadIdx.x & 63;
  // every wave forms M and L itself: one split a lane (at most 64)
  const float2 x = lane < s.S ? ml[lane] : make_float2(-INFINITY, 0.f);
  const float M = wave_max(x.x), Mz = M == -INFINITY ? 0.f : M;
  const float L = wave_sum(x.y * __builtin_amdgcn_exp2f(x.x - Mz));
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = sl; i < s.S; i += SL) y += *(const f32x4 *)(po + (int64_t)i * HD + 4 * ct) * __builtin_amdgcn_exp2f(ml[i].x - Mz);
  oo[sl][ct] = y;
  __syncthreads();
  if (sl) return;
#pragma unroll
  for (int i = 1; i < SL; i++) y += oo[i][ct];
  const float inv = 1.f / L;
  float r[4];
#pragma unroll
  for (int i = 0; i < 4; i++) r[i] = y[i] * inv;
  store_elems<T, 4>(a.out, b * a.out.seq + (int64_t)tok * a.out.tok + (int64_t)head * a.out.head + 4 * ct, r);
}

// The same with a row on HD / 4 lanes and 256 / (HD / 4) rows a workgroup, each thread over all splits in order: for many rows, where a
// workgroup each would come in rounds of 4 us (2048 at a time)
template <int HD, int T>
__global__ __launch_bounds__(256) void k_kv_merge_rows(KvAttnArgs a) {
  constexpr int CT = HD / 4;
  const int b = blockIdx.z, ct = threadIdx.x % CT, i = blockIdx.x * (256 / CT) + threadIdx.x / CT;
  if (i >= a.n * a.heads) return;
  const int tok = i / a.heads, head = i - tok * a.heads, g = token_of(a, head), col = tok * a.rep + head - g * a.rep;
  const Span s = span_of(a, b, chunk_of(a, col));
  if (!s.any || s.S == 1 || tok >= s.cnt || (int64_t)s.P0 + tok >= a.ctx) return;
  const int64_t row = ((int64_t)b * a.n + tok) * a.heads + head;
  const float2 *ml = (const float2 *)(a.part + (int64_t)a.nseq * a.n * a.heads * a.nsplit * HD) + row * a.nsplit;
  const float *po = a.part + row * a.nsplit * HD + 4 * ct;
  float M = -INFINITY, L = 0.f;
#pragma unroll 8
  for (int k = 0; k < s.S; k++) M = fmaxf(M, ml[k].x);
  const float Mz = M == -INFINITY ? 0.f : M;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int k = 0; k < s.S; k++) {
    const float2 x = ml[k];
    const float w = __builtin_amdgcn_exp2f(x.x - Mz);
    L += x.y * w;
    y += *(const f32x4 *)(po + (int64_t)k * HD) * w;
  }
  const float inv = 1.f / L;
  float o[4];
#pragma unroll
  for (int k = 0; k < 4; k++) o[k] = y[k] * inv;
  store_elems<T, 4>(a.out, b * a.out.seq + (int64_t)tok * a.out.tok + (int64_t)head * a.out.head + 4 * ct, o);
}

// A sequence's own splits and the common prefix's.  As the two above; every token that takes part has a row of partial sums, and the own part holds at
// least its own position
template <int HD, int T>
__global__ __launch_bounds__(256) void k_kv_join(KvAttnArgs a, KvJoin p) {
  constexpr int CT = HD / 4, SL = 256 / CT;
  __shared__ f32x4 oo[SL][CT];
  const int head = blockIdx.x, tok = blockIdx.y, b = blockIdx.z, g = token_of(a, head);
  const int col = tok * a.rep + head - g * a.rep;
  const Span s = span_of(a, b, chunk_of(a, col));
  if (!s.any || tok >= s.cnt || (int64_t)s.P0 + tok >= a.ctx) return;
  const int S0 = prefix_splits(p);
  const int64_t row = ((int64_t)b * a.n + tok) * a.heads + head;
  const float2 *ml = (const float2 *)(a.part + (int64_t)a.nseq * a.n * a.heads * slots_of<true>(a) * HD) + row * slots_of<true>(a);
  const float *po = a.part + row * slots_of<true>(a) * HD;
  const int ct = threadIdx.x % CT, sl = threadIdx.x / CT, lane = threadIdx.x & 63;
  const float2 none = make_float2(-INFINITY, 0.f), x = lane < s.S ? ml[lane] : none, x0 = lane < S0 ? ml[a.nsplit + lane] : none;
  const float M = wave_max(fmaxf(x.x, x0.x)), Mz = M == -INFINITY ? 0.f : M;
  const float L = wave_sum(x.y * __builtin_amdgcn_exp2f(x.x - Mz) + x0.y * __builtin_amdgcn_exp2f(x0.x - Mz));
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = sl; i < s.S + S0; i += SL) {
    const int k = i < s.S ? i : a.nsplit + i - s.S;
    y += *(const f32x4 *)(po + (int64_t)k * HD + 4 * ct) * __builtin_amdgcn_exp2f(ml[k].x - Mz);
  }
  oo[sl][ct] = y;
  __syncthreads();
  if (sl) return;
#pragma unroll
  for (int i = 1; i < SL; i++) y += oo[i][ct];
  const float inv = 1.f / L;
  float r[4];
#pragma unroll
  for (int i = 0; i < 4; i++) r[i] = y[i] * inv;
  store_elems<T, 4>(a.out, b * a.out.seq + (int64_t)tok * a.out.tok + (int64_t)head * a.out.head + 4 * ct, r);
}
template <int HD, int T>
__global__ __launch_bounds__(256) void k_kv_join_rows(KvAttnArgs a, KvJoin p) {
  constexpr int CT = HD / 4;
  const int b = blockIdx.z, ct = threadIdx.x % CT, i = (blockIdx.y * gridDim.x + blockIdx.x) * (256 / CT) + threadIdx.x / CT;   // (at most 2^30 rows)
  if (i >= a.n * a.heads) return;
  const int tok = i / a.heads, head = i - tok * a.heads, g = token_of(a, head), col = tok * a.rep + head - g * a.rep;
  const Span s = span_of(a, b, chunk_of(a, col));
  if (!s.any || tok >= s.cnt || (int64_t)s.P0 + tok >= a.ctx) return;
  const int S0 = prefix_splits(p);
  const int64_t row = ((int64_t)b * a.n + tok) * a.heads + head;
  const float2 *ml = (const float2 *)(a.part + (int64_t)a.nseq * a.n * a.heads * slots_of<true>(a) * HD) + row * slots_of<true>(a);
  const float *po = a.part + row * slots_of<true>(a) * HD + 4 * ct;
  float M = -INFINITY, L = 0.f;
#pragma unroll 8
  for (int k = 0; k < s.S + S0; k++) M = fmaxf(M, ml[k < s.S ? k : a.nsplit + k - s.S].x);
  const float Mz = M == -INFINITY ? 0.f : M;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int j = 0; j < s.S + S0; j++) {
    const int k = j < s.S ? j : a.nsplit + j - s.S;
    const float2 x = ml[k];
    const float w = __builtin_amdgcn_exp2f(x.x - Mz);
    L += x.y * w;
    y += *(const f32x4 *)(po + (int64_t)k * HD) * w;
  }
  const float inv = 1.f / L;
  float o[4];
#pragma unroll
  for (int k = 0; k < 4; k++) o[k] = y[k] * inv;
  store_elems<T, 4>(a.out, b * a.out.seq + (int64_t)tok * a.out.tok + (int64_t)head * a.out.head + 4 * ct, o);
}

// ------------------------------------------------------------------ many tokens
// 8 waves of 32 columns; the workgroup's 256 columns share blocks of 64 positions (8 records) in LDS, three buffers: while
// one is computed, the block after next is expanded, and the codes of the one behind that are on their way to registers.
//   scores  S^T[p][c] on v_mfma_f32_32x32x16_f16, A = K rows from LDS.  Row r of a 32-position tile is position 16 (r / 16) +
//           8 (r / 4 % 2) + 4 (r / 8 % 2) + r % 4: the C layout then leaves lane half h = lane / 32 the 8 positions of records
//           2 u + h, u = 0, 1, in order, which is the B fragment of the value product's 16-position step u.
//   values  O^T[d][c] += V^T[d][p] P^T[p][c]: 4-bit: V^T lies in LDS as the words expand, 8 positions of a dim together, one
//           16-byte read a fragment; fp16: V lies as stored and two transpose reads fetch one.
// TWO (fp32 queries): hi and lo halves of the queries and probabilities as products of their own.
// A step of 64 positions takes a wave 32 products (1024 cycles of its SIMD's matrix core, two waves a SIMD), some 130 vector instructions and,
// for 4-bit, 60 that expand; the 8 waves read 256 KiB of LDS, 2048 cycles at its 128 bytes a cycle.  The three overlap in part only:
// 2048 tokens of 32 heads over a 4-bit cache 56 to 64 us by machine (620 TFLOP/s of the 1149 that a large fp16 product reaches), 4096
// tokens with a window of 1024 in fp16 95 to 102 us; fp32 rows, with twice the products, 88 and 150 (over an fp16 cache the 128-dim kernel has all
// 256 registers and spills 6).  256 columns a workgroup, since what a block costs to expand and its LDS writes are
// shared by them: with 128 columns and two workgroups a CU the 4-bit prompt took 77 us for 64, the fp16 one 97 for 100, and 64
// tokens each of 32 sequences 6 % more
constexpr int kManyWaves = 8, kManyBlk = 64, kManyCols = 32 * kManyWaves;

template <int HD>
constexpr int many_kst() { return HD + 8; }   // halves of a K row in LDS: an odd number of 16-byte columns
template <int HD, int KIND>
constexpr int many_vst() { return KIND == MK_Q4 ? kManyBlk + 8 : HD + 32; }   // of a V^T row (dims), or a V row (positions): 4 rows of 64 bytes apart
template <int HD, int KIND>
constexpr int many_vn() { return (KIND == MK_Q4 ? HD : kManyBlk) * many_vst<HD, KIND>(); }
template <int HD, int KIND>
constexpr int many_lds() { return 3 * (kManyBlk * many_kst<HD>() + many_vn<HD, KIND>()); }
using many_bad = uint32_t[4][2];   // positions of block kb left to add_bad, at (kb - kb0) % 4: set in step kb - 2 or before the first, read in kb, cleared in kb + 1
template <int HD, int KIND, int T, bool PRE = false, bool JOIN = false>   // (of the body)
__global__ __launch_bounds__(kManyWaves * 64) void k_kv_many(Args<PRE> a) {
  __shared__ __align__(16) uint16_t blocks[many_lds<HD, KIND>()];
  __shared__ many_bad badp;
  const int b = blockIdx.z, g = blockIdx.x, cs = blockIdx.y;
#include "kv_many.inc"
}
template <int HD, int KIND, int T, bool PRE, int LDS, bool JOIN = true>
__device__ __forceinline__ void many_tokens(Args<PRE> a, int g, int cs, int b) {
  uint16_t *blocks = (uint16_t *)lds<uint8_t[LDS]>();
  auto &badp = lds<many_bad>();
  if constexpr (PRE) a.window = a.sinks = a.paired = 0;
#include "kv_many.inc"
}

// ------------------------------------------------------------------ a common prefix
// The sequences' own positions, the prefix as if all sequences' tokens were one sequence's, and what joins their sums (k_kv_join, k_kv_join_rows).  The prefix's
// workgroups come first and the own ones after them in one launch: they fill what the prefix's leave idle, and a launch and the first kernel's last
// workgroups are saved.  4 samples behind 700 positions 17.2 -> 10.2 us with the joining, 83 sequences behind 4380 33 -> 25, 681 tokens of 2 behind 105 45 -> 35, 8 x up to 128 behind
// 12001 211 -> 208.5
template <int HD, int KIND, int T>
__global__ __launch_bounds__(kFewWaves * 64, kFewOcc) void k_kv_both_few(KvAttnArgs a, KvPreArgs p) {
  constexpr int LDS = few_lds<HD, KIND, T>();
  const uint32_t pre = (uint32_t)p.nsplit * p.nkv * p.nchunk;
  if (blockIdx.x < pre) {
    const uint32_t gc = blockIdx.x / (uint32_t)p.nsplit;
    few_tokens<HD, KIND, T, true, LDS>(p, blockIdx.x - gc * p.nsplit, gc, 0);
  } else {
    const uint32_t i = blockIdx.x - pre, r = i / (uint32_t)a.nsplit, per = (uint32_t)a.nkv * a.nchunk, b = r / per;
    few_tokens<HD, KIND, T, false, LDS>(a, i - r * a.nsplit, r - b * per, b);
  }
}
// many columns behind the prefix; OWN: of the sequences themselves too
constexpr int kWideLog2 = 20;   // workgroups side by side: past them the grid has rows (a dimension's threads are counted in 32 bits)
template <int HD, int KIND, int T, bool OWN>
__global__ __launch_bounds__(kManyWaves * 64) void k_kv_both_many(KvAttnArgs a, KvPreArgs p) {
  static_assert(kManyWaves == kFewWaves, "one launch of both");
  constexpr int LDS = OWN || 2 * many_lds<HD, KIND>() > few_lds<HD, KIND, T>() ? 2 * many_lds<HD, KIND>() : few_lds<HD, KIND, T>();
  const uint32_t id = blockIdx.y << kWideLog2 | blockIdx.x, pre = (uint32_t)p.nkv * p.nchunk * p.nsplit, i = id - pre;
  if (id < pre) {
    const uint32_t cs = id / (uint32_t)p.nkv;
    many_tokens<HD, KIND, T, true, LDS>(p, id - cs * p.nkv, cs, 0);
  } else if constexpr (OWN) {
    const uint32_t r = i / (uint32_t)a.nkv, per = (uint32_t)a.nchunk * a.nsplit, b = r / per;
    if (b >= (uint32_t)a.nseq) return;
    many_tokens<HD, KIND, T, false, LDS>(a, i - r * a.nkv, r - b * per, b);
  } else {
    const uint32_t r = i / (uint32_t)a.nsplit, per = (uint32_t)a.nkv * a.nchunk, b = r / per;
    if (b >= (uint32_t)a.nseq) return;
    few_tokens<HD, KIND, T, false, LDS>(a, i - r * a.nsplit, r - b * per, b);
  }
}

// ------------------------------------------------------------------ launches
// KERNEL<HD, T> by head dim and rows' type
#define QPH_KVN(KERNEL, hd, type, grid, threads, ...)                                                                   \
  do {                                                                                                                  \
    const dim3 g_ = (grid), t_(threads);                                                                                \
    if ((hd) == 128) {                                                                                                  \
      if ((type) == RT_F32) hipLaunchKernelGGL((KERNEL<128, RT_F32>), g_, t_, 0, st, __VA_ARGS__);                      \
      else if ((type) == RT_F16) hipLaunchKernelGGL((KERNEL<128, RT_F16>), g_, t_, 0, st, __VA_ARGS__);                 \
      else hipLaunchKernelGGL((KERNEL<128, RT_BF16>), g_, t_, 0, st, __VA_ARGS__);                                      \
    } else {                                                                                                            \
      if ((type) == RT_F32) hipLaunchKernelGGL((KERNEL<64, RT_F32>), g_, t_, 0, st, __VA_ARGS__);                       \
      else if ((type) == RT_F16) hipLaunchKernelGGL((KERNEL<64, RT_F16>), g_, t_, 0, st, __VA_ARGS__);                  \
      else hipLaunchKernelGGL((KERNEL<64, RT_BF16>), g_, t_, 0, st, __VA_ARGS__);                                       \
    }                                                                                                                   \
  } while (0)
#define QPH_KV(KERNEL, hd, type, grid, threads, a) QPH_KVN(KERNEL, hd, type, grid, threads, a)
template <bool WRITE>
void launch_io16(const KvIoArgs &a, hipStream_t st) {
  const dim3 grid((unsigned)(((int64_t)a.n * a.nkv * a.hd / 8 + 255) / 256), 2, a.nseq), thr(256);
  if (a.k.type == RT_F32) hipLaunchKernelGGL((k_kv16_io<WRITE, RT_F32>), grid, thr, 0, st, a);
  else if (a.k.type == RT_F16) hipLaunchKernelGGL((k_kv16_io<WRITE, RT_F16>), grid, thr, 0, st, a);
  else hipLaunchKernelGGL((k_kv16_io<WRITE, RT_BF16>), grid, thr, 0, st, a);
}
}  // namespace

hipError_t launch_kv_write(int kind, const KvIoArgs &a, hipStream_t st) {
  if (kind == MK_Q4 && a.n == 1) QPH_KV(k_kv4_write1, a.hd, a.k.type, dim3(1, a.nkv, a.nseq), 128, a);
  else if (kind == MK_Q4) QPH_KV(k_kv4_write, a.hd, a.k.type, dim3((unsigned)(((int64_t)a.n + 7) / 8 + 1), a.nkv, a.nseq), 128, a);
  else launch_io16<true>(a, st);
  return hipGetLastError();
}
hipError_t launch_kv_read(int kind, const KvIoArgs &a, hipStream_t st) {
  if (kind == MK_Q4) QPH_KV(k_kv4_read, a.hd, a.k.type, dim3((unsigned)(((int64_t)a.n + 7) / 8 + 1), a.nkv, a.nseq), 128, a);
  else launch_io16<false>(a, st);
  return hipGetLastError();
}

int kv_few() {
  const char *e = getenv("QPH_KV_FEW");
  return e && *e ? std::max(0, atoi(e)) : -1;
}
// parted: the sums are joined with others' in any case
size_t kv_attn_plan(KvAttnArgs &a, bool parted) {
  const int cus = 256;
  const bool two = a.q.type == RT_F32;
  const int64_t cols = (int64_t)a.n * a.rep;
  const int few = two ? 8 : 16;
  // positions that a workgroup of c columns can have to read, at most
  auto reach = [&](int c) { return a.window > 0 ? std::min<int64_t>(a.ctx, (int64_t)a.window + a.sinks + (c + a.rep - 1) / a.rep + 3 * kRec) : a.ctx; };
  // k_kv_few's time goes with its chunks of 8 or 16 columns times the positions, each chunk reading them anew; k_kv_many's with the positions
  // alone up to 256 columns, and it takes some 6 us longer to start.  Chunks up to which the first is faster, from both kernels' times at
  // 12 to 640 columns, 1 and 8 sequences of 256 to 16384 positions, 8 kv heads of 128 dims (472 calls; the rule's choice is 1 % slower
  // than the better kernel's in the mean, a limit of 64 columns was 19 %).  4-bit: 64 columns over 8 x 4096 positions 36 us few, 37
  // many; 128 over 8 x 16384 176 and 112; 128 over 8 x 1024 18 and 35.  fp16: the same 92 and 38, 624 and 133, 44 and 31.
  // Other shapes take the same constants.  8 to 512 columns over 512, 4096 and 16384 positions, 1 and 8 sequences, 42 calls each: fp32 rows 0.9 %
  // (4-bit) and 1.8 % (fp16) slower than the better kernel's in the mean, heads of 64 dims 1.9 and 1.7, two of them with fp32 rows 1.9 and 5.3 (the
  // worst: 256 columns over 8 x 512 fp16 positions, 22 us many for 11 few)
  const int64_t chunks = (cols + few - 1) / few, positions = (int64_t)a.nseq * a.nkv * reach(few);
  const int64_t most = a.kind == MK_Q4 ? 4 + (384 << 10) / positions : 1 + (192 << 10) / positions;
  a.many = (a.few >= 0 ? cols > a.few : chunks > std::min<int64_t>(most, 128)) || chunks * a.nkv > 65535;   // (the last: the grid)
  a.cols = a.many ? kManyCols : few;
  a.half_log2 = a.many ? 7 : two ? 2 : 3;
  a.tile_log2 = a.many ? 3 : 2;   // records of a tile
  // tiles of a split, at least (parted, where the sums are joined in any case: with 8, 4 samples behind 700 positions 7.2 us for 6.4)
  a.min_log2 = a.many || parted ? 2 : 3;
  a.one_tiles = parted ? -1 : a.many ? 4 : 4 * kFewWaves;
  const int tile = kRec << a.tile_log2;
  // floor(col / rep) = floor(col mul / 2^(32 + shift)) for col < 2^30: mul = ceil(2^(32 + shift) / rep) with 2^shift < rep <= 2^(shift + 1)
  a.rep_shift = 0;
  while (2 << a.rep_shift < a.rep) a.rep_shift++;
  a.rep_mul = a.rep == 1 ? 0 : (uint32_t)(((1ull << (32 + a.rep_shift)) + a.rep - 1) / a.rep);
  a.nchunk = (int)((cols + a.cols - 1) / a.cols);
  a.paired = a.many && a.window == 0;
  const int64_t tiles = (reach(a.cols) + tile - 1) / tile, groups = (int64_t)a.nkv * a.nchunk * a.nseq;
  const int64_t want = (a.many ? 1 : 2) * (int64_t)cus / std::max<int64_t>(groups, 1);
  a.nsplit = tiles <= a.one_tiles ? 1 : (int)std::max<int64_t>(1, std::min({want, (tiles >> a.min_log2) + 1, (int64_t)64}));
  if (a.n > 65535 || a.nchunk * a.nsplit > 65535) a.nsplit = 1;   // grid limits
  return a.nsplit > 1 ? (size_t)a.nseq * a.n * a.heads * a.nsplit * (a.hd + 2) * 4 : 0;
}

template <int HD, int T> static constexpr auto k_few4 = k_kv_few<HD, MK_Q4, T>;
template <int HD, int T> static constexpr auto k_few16 = k_kv_few<HD, MK_F32, T>;
template <int HD, int T> static constexpr auto k_many4 = k_kv_many<HD, MK_Q4, T>;
template <int HD, int T> static constexpr auto k_many16 = k_kv_many<HD, MK_F32, T>;
// rows from which the splits are merged by k_kv_merge_rows: at 2048 the two are even, 6144 rows 44 -> 39 us with the attention, 16384 50 -> 34
constexpr int kMergeRows = 4096;
hipError_t launch_kv_attn(const KvAttnArgs &a, hipStream_t st) {
  if (a.many) {
    const dim3 grid(a.nkv, a.nchunk * a.nsplit, a.nseq);
    if (a.kind == MK_Q4) QPH_KV(k_many4, a.hd, a.q.type, grid, kManyWaves * 64, a);
    else QPH_KV(k_many16, a.hd, a.q.type, grid, kManyWaves * 64, a);
  } else {
    const dim3 grid(a.nsplit, a.nkv * a.nchunk, a.nseq);
    if (a.kind == MK_Q4) QPH_KV(k_few4, a.hd, a.q.type, grid, kFewWaves * 64, a);
    else QPH_KV(k_few16, a.hd, a.q.type, grid, kFewWaves * 64, a);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.nsplit == 1) return e;
  if ((int64_t)a.nseq * a.n * a.heads >= kMergeRows) QPH_KV(k_kv_merge_rows, a.hd, a.q.type, dim3((a.n * a.heads + 1024 / a.hd - 1) / (1024 / a.hd), 1, a.nseq), 256, a);   // (at most 32768 rows a sequence: groups <= 256)
  else QPH_KV(k_kv_merge, a.hd, a.q.type, dim3(a.heads, a.n, a.nseq), 256, a);
  return hipGetLastError();
}

// ------------------------------------------------------------------ a common prefix
// `a` is the own part's, planned; the prefix's plan goes by the columns of all sequences
// The prefix's columns are few up to one round of k_kv_few's workgroups (480 of them and 504 own ones 16.1 us, 17.7 by k_kv_many; 632 and 672 19.2 and 14.7, 872 and 888 33.8 and 26.0).
// Own tokens of few columns beside many behind the prefix.  k_kv_few has two workgroups a CU in a launch of its own, one in that of both, which it starts with the prefix's.  From
// several rounds on either way is slow: where a sequence's columns are several of k_kv_few's chunks, k_kv_many takes them past 512 workgroups (1014 of them 54 us for 36, 2584 43 for 20,
// 10848 229 for 103; 444 18.0 for 20.0, 475 22.7 for 26.0).  A single chunk would leave it 16 columns of 256: those have a launch of their own
// past 1024 (656 of them 33 us together, 45.5 apart; 920 81 and 84; 2048 103 and 85, 8000 158 and 93)
static int64_t few_blocks(const KvAttnArgs &a) { return (int64_t)a.nsplit * a.nkv * a.nchunk * a.nseq; }
static bool few_apart(const KvAttnArgs &a) { return few_blocks(a) > 1024; }
size_t kv_prefix_plan(KvAttnArgs &a, KvPreArgs &p) {
  kv_attn_plan(a, true);
  kv_attn_plan(p, true);
  if (!p.many && (a.many || few_blocks(p) > 512)) { p.few = 0; kv_attn_plan(p, true); }   // (few columns of either: one launch of k_kv_few's workgroups, two a CU)
  if (p.many && !a.many && a.nchunk > 1 && few_blocks(a) > 512) { a.few = 0; kv_attn_plan(a, true); }
  // Few positions of both: each workgroup takes all that its columns see, and nothing is left to be joined.  24 tiles of both 22.5 us for 19.0, 11 10.5 for 7.9, 4 8.1 for 4.5; with 128 dims
  // 27 9.9 for 12.9 and 30 9.5 for 10.6, with 64 30 8.5 for 7.9 and 43 9.2 for 11.7.  Like all of the plan it goes by the caches' room, since the host does not know what they hold: 53 sequences of 3 tokens
  // at 50 behind 37 5.6 us with caches as long as that, 11.1 where the own ones have room for 4096 positions
  const int64_t tiles = (p.ctx + kFewTile - 1) / kFewTile + (a.ctx + kFewTile - 1) / kFewTile;
  if (!p.many && tiles <= (a.hd == 64 ? 4 : 3) * kFewWaves && few_blocks(a) / a.nsplit <= 512) {
    p.nsplit = 0;   // (says so to the launch)
    return 0;
  }
  p.paired = 0;   // (every column sees all: nothing to even out)
  if (p.many && !a.many && !few_apart(a)) a.nsplit = std::max(1, a.nsplit / 2);   // (one workgroup a CU beside the others: 32 sequences behind 8190 positions 38.4 us for 35.2)
  a.one_tiles = p.one_tiles = -(a.nsplit + p.nsplit);
  return (size_t)a.nseq * a.n * a.heads * slots_of<true>(a) * (a.hd + 2) * 4;
}
template <int HD, int T> static constexpr auto k_all4 = k_kv_few_all<HD, MK_Q4, T>;
template <int HD, int T> static constexpr auto k_all16 = k_kv_few_all<HD, MK_F32, T>;
template <int HD, int T> static constexpr auto k_own4 = k_kv_few<HD, MK_Q4, T, false, true>;
template <int HD, int T> static constexpr auto k_own16 = k_kv_few<HD, MK_F32, T, false, true>;
template <int HD, int T> static constexpr auto k_few_few4 = k_kv_both_few<HD, MK_Q4, T>;
template <int HD, int T> static constexpr auto k_few_few16 = k_kv_both_few<HD, MK_F32, T>;
template <int HD, int T> static constexpr auto k_many_few4 = k_kv_both_many<HD, MK_Q4, T, false>;
template <int HD, int T> static constexpr auto k_many_few16 = k_kv_both_many<HD, MK_F32, T, false>;
template <int HD, int T> static constexpr auto k_many_many4 = k_kv_both_many<HD, MK_Q4, T, true>;
template <int HD, int T> static constexpr auto k_many_many16 = k_kv_both_many<HD, MK_F32, T, true>;
hipError_t launch_kv_prefix(const KvAttnArgs &a, const KvPreArgs &p, hipStream_t st) {
  hipError_t e;
  if (p.nsplit == 0) {
    const dim3 grid(1, a.nkv * a.nchunk, a.nseq);
    if (p.kind == MK_Q4) QPH_KVN(k_all4, p.hd, p.q.type, grid, kFewWaves * 64, a, p);
    else QPH_KVN(k_all16, p.hd, p.q.type, grid, kFewWaves * 64, a, p);
    return hipGetLastError();
  }
  const bool q4 = p.kind == MK_Q4, apart = p.many && !a.many && few_apart(a);
  const int64_t all = (int64_t)p.nsplit * p.nkv * p.nchunk + (apart ? 0 : few_blocks(a)), width = std::min(all, (int64_t)1 << kWideLog2);
  KvAttnArgs own = a;
  if (apart) {
    own.nseq = 0;   // (none in the launch below)
    const dim3 grid(a.nsplit, a.nkv * a.nchunk, a.nseq);
    if (q4) QPH_KV(k_own4, a.hd, a.q.type, grid, kFewWaves * 64, a);
    else QPH_KV(k_own16, a.hd, a.q.type, grid, kFewWaves * 64, a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  const dim3 both((unsigned)width, (unsigned)((all + width - 1) / width));
  if (!p.many) {   // (at most 65535 workgroups of the prefix, whose chunks have 8 columns at least: 2^21 of all)
    if (q4) QPH_KVN(k_few_few4, p.hd, p.q.type, dim3((unsigned)all), kFewWaves * 64, a, p);
    else QPH_KVN(k_few_few16, p.hd, p.q.type, dim3((unsigned)all), kFewWaves * 64, a, p);
  } else if (!a.many) {
    if (q4) QPH_KVN(k_many_few4, p.hd, p.q.type, both, kManyWaves * 64, own, p);
    else QPH_KVN(k_many_few16, p.hd, p.q.type, both, kManyWaves * 64, own, p);
  } else {
    if (q4) QPH_KVN(k_many_many4, p.hd, p.q.type, both, kManyWaves * 64, own, p);
    else QPH_KVN(k_many_many16, p.hd, p.q.type, both, kManyWaves * 64, own, p);
  }
  if ((e = hipGetLastError()) != hipSuccess) return e;
  const KvJoin j{p.prefix, p.tile_log2, p.min_log2, p.one_tiles, p.nsplit};
  const unsigned blocks = (unsigned)(((int64_t)a.n * a.heads + 1024 / a.hd - 1) / (1024 / a.hd)), wide = std::min(blocks, 65536u);   // (a grid's threads are counted in 32 bits for each dimension)
  if ((int64_t)a.nseq * a.n * a.heads >= kMergeRows || a.n > 65535) QPH_KVN(k_kv_join_rows, a.hd, a.q.type, dim3(wide, (blocks + wide - 1) / wide, a.nseq), 256, a, j);
  else QPH_KVN(k_kv_join, a.hd, a.q.type, dim3(a.heads, a.n, a.nseq), 256, a, j);
  return hipGetLastError();
}

}  // namespace qph
