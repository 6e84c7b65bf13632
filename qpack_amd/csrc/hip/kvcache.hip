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

#include "launch.hpp"

namespace qph {

namespace {
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s4 lds_s4;

constexpr int kRec = kKvRec;   // positions of a record

__device__ __forceinline__ float bf16_to_f(uint16_t h) { return __builtin_bit_cast(float, (uint32_t)h << 16); }
// round to nearest even; NaN stays NaN
__device__ __forceinline__ uint16_t f_to_bf16(float f) {
  const uint32_t u = __builtin_bit_cast(uint32_t, f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)(u >> 16 | 0x40);
  return (uint16_t)((u + 0x7fff + (u >> 16 & 1)) >> 16);
}

// N (a multiple of 8) consecutive elements of type T (RowType) from element `at` of rows.  The loads and stores are 16 (8) bytes at any alignment of
// the type, which the memory pipeline takes as they are: a second, element by element, path made the kernels twice as
// long, and their first pass through the instruction cache is what a short call waits for
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));
template <int T, int N>
__device__ __forceinline__ void load_elems(const KvRows &r, int64_t at, float *x) {
  if constexpr (T == RT_F32) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const u32x4 v = *(const u32x4_any *)((const float *)r.p + at + i);
#pragma unroll
      for (int j = 0; j < 4; j++) { const uint32_t w = v[j]; x[i + j] = __builtin_bit_cast(float, w); }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 8) {
      const u32x4 v = *(const u32x4_any *)((const uint16_t *)r.p + at + i);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const uint16_t h = (uint16_t)(v[j / 2] >> 16 * (j & 1));
        x[i + j] = T == RT_F16 ? half_bits_to_float(h) : bf16_to_f(h);
      }
    }
  }
}
// N a multiple of 4
template <int T, int N>
__device__ __forceinline__ void store_elems(const KvRows &r, int64_t at, const float *x) {
  auto e = [](float f) { return (uint32_t)(T == RT_F16 ? float_to_half_bits(f) : f_to_bf16(f)); };
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    if constexpr (T == RT_F32) {
      *(u32x4_any *)((float *)r.p + at + i) = (u32x4){__builtin_bit_cast(uint32_t, x[i]), __builtin_bit_cast(uint32_t, x[i + 1]), __builtin_bit_cast(uint32_t, x[i + 2]),
                                                      __builtin_bit_cast(uint32_t, x[i + 3])};
    } else {
      *(u32x2_any *)((uint16_t *)r.p + at + i) = (u32x2){e(x[i]) | e(x[i + 1]) << 16, e(x[i + 2]) | e(x[i + 3]) << 16};
    }
  }
}

// 8 fp16 elements as the matrix cores take them
__device__ __forceinline__ h8 load_halves(const KvRows &r, int64_t at) {
  const u32x4 v = *(const u32x4_any *)((const uint16_t *)r.p + at);
  return __builtin_bit_cast(h8, v);
}

// bit position of element i (0 .. 7) of a word of codes
__host__ __device__ constexpr int nib(int i) { return 16 * (i & 1) + 4 * (i >> 1); }

// a word's 8 values in element order.  Codes 0 .. 15 in the low mantissa bits of fp16 1024 (or, four bits higher, 16 times
// them, brought back by an exact fma): c - 8 exact, times the elements' scales exact
__device__ __forceinline__ uint32_t vreg(uint32_t c) { asm("" : "+v"(c)); return c; }   // an instruction reads one scalar: v_and_or_b32 wants the other constant in a vector register
__device__ __forceinline__ h2 code_pair(uint32_t w, int e) {
  const h2 k1032 = {(_Float16)1032.f, (_Float16)1032.f}, k16 = {(_Float16)0.0625f, (_Float16)0.0625f}, k72 = {(_Float16)-72.f, (_Float16)-72.f};
  if (e & 1) {
    const h2 x = __builtin_bit_cast(h2, ((e > 1 ? w >> 8 : w) & 0x00f000f0u) | vreg(0x64006400u));
    return __builtin_elementwise_fma(x, k16, k72);
  }
  const h2 x = __builtin_bit_cast(h2, ((e > 1 ? w >> 8 : w) & 0x000f000fu) | vreg(0x64006400u));
  return x - k1032;
}
// scales of the four element pairs: one for all (K: a group of dims), or the positions' own (V)
__device__ __forceinline__ h8 values(uint32_t w, h2 s0, h2 s1, h2 s2, h2 s3) {
  const h2 a = code_pair(w, 0) * s0, b = code_pair(w, 1) * s1, c = code_pair(w, 2) * s2, d = code_pair(w, 3) * s3;
  return (h8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ h8 values(uint32_t w, uint16_t s) {
  const h2 x = __builtin_bit_cast(h2, (uint32_t)s * 0x10001u);
  return values(w, x, x, x, x);
}
__device__ __forceinline__ h8 values(uint32_t w, u32x4 s) {
  const uint32_t s0 = s[0], s1 = s[1], s2 = s[2], s3 = s[3];   // (a bit cast of a vector's element takes the first one)
  return values(w, __builtin_bit_cast(h2, s0), __builtin_bit_cast(h2, s1), __builtin_bit_cast(h2, s2), __builtin_bit_cast(h2, s3));
}

__device__ __forceinline__ int tokens_of(const int *lens, int b, int n) { return lens ? min(max(lens[b], 0), n) : n; }

// ------------------------------------------------------------------ writing and reading
// the scale of a group from the bits of its largest magnitude
__device__ __forceinline__ uint16_t group_scale(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return 0x7e00;
  const float a = fminf(__builtin_bit_cast(float, amax_bits), 65504.f);
  return float_to_half_bits(bf16_to_f(f_to_bf16(a / 7.f)));
}
// clamp(rint(x / s), -7, 7) + 8, ties to even, of the real quotient: the product with 1 / s is off by one step at most, and
// only next to a border; e = x - r s is exact (r s has 11 bits, e is a multiple of x's last place below 2^24 of them).
// 16-bit rows: x has 11 bits at most and s 8, so x / s is a border (half an odd number) or 2^-12 away from all of them.  Rounded to a
// multiple of 2^-16 first (by adding 192), the product, which is off by less than 2^-20, is on the right side or on the border itself; a
// second sum rounds it to a whole number in the float's low bits.  Four instructions for fifteen: 2048
// positions of 8 heads of 128 dims 7.1 -> 4.5 us
template <int T>
__device__ __forceinline__ uint32_t code_of(float x, float s, float inv) {
  const float y = __builtin_amdgcn_fmed3f(x, -7.f * s, 7.f * s);
  if constexpr (T != RT_F32) {
    const float t = __builtin_fmaf(y, inv, 192.f) + (12582912.f + 8.f - 192.f);
    return __builtin_bit_cast(uint32_t, t) & 15;
  }
  float r = __builtin_rintf(y * inv);
  const float e = 2.f * __builtin_fmaf(-r, s, y);
  const bool odd = ((int)r & 1) != 0;
  if (e > s || (e == s && odd)) r += 1.f;
  else if (e < -s || (e == -s && odd)) r -= 1.f;
  return (uint32_t)((int)r + 8);
}

// One wave per record's K, one per its V: lane = position lane / 8 of the record, dims EL (lane % 8) ..  Positions outside the
// call's keep their codes and scales: their K rows and scales are not stored, and the V words, which hold all 8
// positions, are read and merged where the call covers a part only (no other workgroup of the launch has the record).
// 2048 positions of 8 heads of 128 dims, fp16 rows: 4.5 us, a launch (2.4) and 10.8 MB at the copy rate (2.2).
template <int HD, int T>
__global__ __launch_bounds__(128) void k_kv4_write(KvIoArgs a) {
  constexpr int EL = HD / 8, GL = 32 / EL;   // elements of a lane; lanes of a group
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
  float x[EL];
  uint32_t mx = 0;
  if (mine) {
    load_elems<T, EL>(r, b * r.seq + (p - P0) * r.tok + g * r.head + EL * part, x);
#pragma unroll
    for (int i = 0; i < EL; i++) mx = max(mx, __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu);
  }
  mx = max(mx, (uint32_t)dpp_i<kDppQuadXor1>((int)mx));
  if (GL == 4) mx = max(mx, (uint32_t)dpp_i<kDppQuadXor2>((int)mx));
  const uint16_t sb = group_scale(mx);
  const float s = half_bits_to_float(sb);
  uint32_t c[EL];
  if (s > 0.f) {
    const float inv = 1.f / s;
#pragma unroll
    for (int i = 0; i < EL; i++) c[i] = mine ? code_of<T>(x[i], s, inv) : 8;
  } else {
#pragma unroll
    for (int i = 0; i < EL; i++) c[i] = 8;
  }
  uint8_t *o = (uint8_t *)a.cache + (((int64_t)b * a.nkv + g) * a.nrec + rec) * (9 * HD);
  if (!vside) {
    if (!mine) return;
    uint32_t w[EL / 8];
#pragma unroll
    for (int i = 0; i < EL / 8; i++) {
      w[i] = 0;
#pragma unroll
      for (int j = 0; j < 8; j++) w[i] |= c[8 * i + j] << nib(j);
      *(uint32_t *)(o + row * (HD / 2) + part * (EL / 2) + 4 * i) = w[i];
    }
    if (part % GL == 0) *(uint16_t *)(o + 8 * HD + 2 * (row * (HD / 32) + part / GL)) = sb;
    return;
  }
  if (mine && part % GL == 0) *(uint16_t *)(o + 8 * HD + HD / 2 + 2 * (part / GL * kRec + row)) = sb;
#pragma unroll
  for (int i = 0; i < EL; i += 4) *(uint32_t *)&codes[row][EL * part + i] = c[i] | c[i + 1] << 8 | c[i + 2] << 16 | c[i + 3] << 24;
  // the V wave alone reads what it wrote
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  uint32_t keep = 0;   // bits of the positions that the call does not write
#pragma unroll
  for (int i = 0; i < kRec; i++)
    if (!(rec * kRec + i >= P0 && rec * kRec + i < last)) keep |= 15u << nib(i);
#pragma unroll
  for (int k = 0; k < HD / 64; k++) {
    const int idx = lane * (HD / 64) + k, d = idx % (HD / 16) * 16 + idx / (HD / 16);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < kRec; i++) w |= (uint32_t)codes[i][d] << nib(i);
    uint32_t *dst = (uint32_t *)(o + 4 * HD) + idx;
    if (keep) w = (w & ~keep) | (*dst & keep);
    *dst = w;
  }
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
  const int row = p % kRec;
  uint32_t *vw[EL], old[EL];
  if (vside) {
#pragma unroll
    for (int i = 0; i < EL; i++) {
      const int d = EL * lane + i;
      vw[i] = (uint32_t *)(o + 4 * HD) + d % 16 * (HD / 16) + d / 16;
      old[i] = *vw[i];
    }
  }
  uint32_t mx = 0;
#pragma unroll
  for (int i = 0; i < EL; i++) mx = max(mx, __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu);
  mx = max(mx, (uint32_t)dpp_i<kDppQuadXor1>((int)mx));
  mx = max(mx, (uint32_t)dpp_i<kDppQuadXor2>((int)mx));
  mx = max(mx, (uint32_t)dpp_i<kDppHalfMirror>((int)mx));
  mx = max(mx, (uint32_t)dpp_i<kDppMirror>((int)mx));
  if (EL == 1) {   // 32 dims are 32 lanes (a maximum of the bits: NaN's are the largest)
    float u, v;
    swap16(__builtin_bit_cast(float, mx), u, v);
    mx = max(__builtin_bit_cast(uint32_t, u), __builtin_bit_cast(uint32_t, v));
  }
  const uint16_t sb = group_scale(mx);
  const float s = half_bits_to_float(sb), inv = 1.f / s;
  uint32_t c[EL];
#pragma unroll
  for (int i = 0; i < EL; i++) c[i] = s > 0.f ? code_of<T>(x[i], s, inv) : 8;
  if (vside) {
    const int sh = 16 * (row & 1) + 4 * (row >> 1);
#pragma unroll
    for (int i = 0; i < EL; i++) *vw[i] = (old[i] & ~(15u << sh)) | c[i] << sh;
    if (lane % (32 / EL) == 0) *(uint16_t *)(o + 8 * HD + HD / 2 + 2 * (lane / (32 / EL) * kRec + row)) = sb;
    return;
  }
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < EL; i++) { const int j = (EL * lane + i) & 7; w |= c[i] << (16 * (j & 1) + 4 * (j >> 1)); }
  w |= (uint32_t)dpp_i<kDppQuadXor1>((int)w);
  w |= (uint32_t)dpp_i<kDppQuadXor2>((int)w);
  if (EL == 1) w |= (uint32_t)dpp_i<kDppHalfMirror>((int)w);
  if (lane % (8 / EL) == 0) *(uint32_t *)(o + row * (HD / 2) + EL * lane / 2) = w;
  if (lane % (32 / EL) == 0) *(uint16_t *)(o + 8 * HD + 2 * (row * (HD / 32) + lane / (32 / EL))) = sb;
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
__device__ __forceinline__ int64_t row_of(const KvAttnArgs &a, const Span &s, int v, int j) {
  return min((int64_t)kRec * record(s, min(v, s.NR - 1)) + j, a.ctx - 1) * a.crow;
}
// whether records v .. v + n - 1 are there and follow each other
__device__ __forceinline__ bool run_of(const Span &s, int v, int n) { return v + n <= s.NR && (s.skip == 0 || v >= s.SR || v + n <= s.SR); }
// a 4-bit tile's loads: a scalar base and offsets that a lane keeps where its records follow each other (all tiles but a few)
template <int HD>
__device__ __forceinline__ const uint8_t *tile_base(const Head &h, const Span &s, int tile, bool run, int r) {   // r: the lane's record of the tile
  return h.rec + (run ? (int64_t)record(s, 4 * tile) : (int64_t)record(s, min(4 * tile + r, s.NR - 1)) - r) * (9 * HD);
}
template <int HD, int KIND>
__device__ __forceinline__ void load_k(const KvAttnArgs &a, const Head &h, const Span &s, int tile, int lane, Tile<HD, KIND> &t) {
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
template <int HD, int KIND>
__device__ __forceinline__ void load_v(const KvAttnArgs &a, const Head &h, const Span &s, int tile, int lane, Tile<HD, KIND> &t, uint16_t *buf) {
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
__global__ __launch_bounds__(kFewWaves * 64, kFewOcc) void k_kv_few(KvAttnArgs a) {
  constexpr bool TWO = T == RT_F32;
  constexpr int NW = kFewWaves, KS = HD / 32, DT = HD / 16, NC = TWO ? 8 : 16, QS = HD + 4;
  constexpr int kTileBytes = KIND == MK_Q4 ? 0 : NW * kFewTile * HD * 2, kOutBytes = NW * NC * QS * 4;
  __shared__ __align__(16) uint8_t sm[kTileBytes > kOutBytes ? kTileBytes : kOutBytes];
  __shared__ float wm[NW][NC], wl[NW][NC];
  const int b = blockIdx.z, g = a.nchunk == 1 ? blockIdx.y : blockIdx.y / (uint32_t)a.nchunk, chunk = blockIdx.y - g * a.nchunk, c0 = chunk * NC, split = blockIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
  // columns past the call's last are that one again: another row may be another workgroup's, whose results may be on their way into it (out may
  // be q).  (Zeros without a load, or the first column's row: 0.3 us of a short call)
  const int col = min(c0 + (TWO ? lr & 7 : lr), a.n * a.rep - 1), tok = token_of(a, col), hr = col - tok * a.rep;
  // the column's query: dims HD / 4 lg + 8 k + j (4-bit: a lane's words are consecutive) or 32 k + 8 lg + j.  Asked for before
  // the sequence's position is known
  h8 q[KS];
  float x[KS][8];
  {
    const int64_t at = b * a.q.seq + (int64_t)tok * a.q.tok + (int64_t)(g * a.rep + hr) * a.q.head;
#pragma unroll
    for (int k = 0; k < KS; k++) {
      const int64_t d = at + (KIND == MK_Q4 ? HD / 4 * lg + 8 * k : 32 * k + 8 * lg);
      if constexpr (T == RT_F16) q[k] = load_halves(a.q, d);
      else load_elems<T, 8>(a.q, d, x[k]);
    }
  }
  const Span s = span_of(a, b, chunk);
  if (!s.any || split >= s.S) return;
  const bool live = tok < s.cnt && (int64_t)s.P0 + tok < a.ctx;
  const int P = live ? s.P0 + tok : -1;
  const int lo = behind(a, P);
  const int t0 = share(s, split), t1 = share(s, split + 1);
  const Head h = head_of<HD, KIND>(a, b, g);
  uint16_t *vbuf = (uint16_t *)sm + wave * kFewTile * HD;
  Tile<HD, KIND> cur;
  if (t0 + wave < t1) { load_v<HD, KIND>(a, h, s, t0 + wave, lane, cur, vbuf); load_k<HD, KIND>(a, h, s, t0 + wave, lane, cur); }
  float f = a.scale2;   // softmax scale in base 2, times the row's power
  if constexpr (T != RT_F16) {
    float mx = 0.f;
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
      for (int j = 0; j < 8; j++) mx = fmaxf(mx, fabsf(x[k][j]));
    mx = pair_max32(pair_max16(mx));
    const float p2 = row_power(mx);
    f = fminf(fmaxf(f / p2, kTinyF), kMostF);
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float y = x[k][j] * p2;
        const _Float16 hi = (_Float16)y;
        q[k][j] = TWO && lr >= 8 ? (_Float16)(y - (float)hi) : hi;
      }
  }
  f32x4 o[DT];
#pragma unroll
  for (int d = 0; d < DT; d++) o[d] = (f32x4){0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f, sub = kPBias;
  // the next tile's K is asked for once this one's is used, its V likewise: either is on its way during the other's product
  for (int tile = t0 + wave; tile < t1; tile += NW) {
    const int v = 4 * tile + lg, p0 = kRec * record(s, min(v, s.NR - 1)), Pin = v < s.NR ? P : -1;
    // whether some column does not see all of the tile: its first and last position bound the others
    const int pf = kRec * record(s, 4 * tile), pl = kRec * record(s, min(4 * tile + 3, s.NR - 1)) + kRec - 1;
    const bool edge = 4 * tile + 4 > s.NR || pl > s.PA || (a.window > 0 && pf <= s.PB - a.window && pl >= a.sinks);
    f32x4 sc[2];
#pragma unroll
    for (int mt = 0; mt < 2; mt++) {
      sc[mt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KS; k++) {
        h8 kf;
        if constexpr (KIND == MK_Q4) kf = values(cur.k[mt][k], cur.ks[mt]);
        else kf = __builtin_bit_cast(h8, cur.k[mt][k]);
        sc[mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[k], sc[mt], 0, 0, 0);
      }
    }
    if constexpr (KIND == MK_Q4) { if (tile + NW < t1) load_k<HD, KIND>(a, h, s, tile + NW, lane, cur); }
    float y[8];
    uint32_t on = 255;   // positions that a column of the workgroup sees
#pragma unroll
    for (int j = 0; j < 8; j++) {
      y[j] = sc[j >> 2][j & 3];
      if (TWO) y[j] += xchg8_f(y[j]);
    }
    if (edge) {
      on = seen_bits(a, s, v, p0);
#pragma unroll
      for (int j = 0; j < 8; j++) y[j] = sees(a, Pin, lo, p0 + j) ? y[j] : -INFINITY;
    }
    h8 ph;
    auto weights = [&]() {   // y -> ph and their sum over the lane's positions
      float rs = 0.f;
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float w0 = __builtin_amdgcn_exp2f(__builtin_fmaf(y[j], f, sub)), w1 = __builtin_amdgcn_exp2f(__builtin_fmaf(y[j + 1], f, sub));
        h2 hi = {(_Float16)w0, (_Float16)w1};
        if constexpr (TWO) {
          rs += w0; rs += w1;
          if (lr >= 8) hi = (h2){(_Float16)(w0 - (float)hi[0]), (_Float16)(w1 - (float)hi[1])};
        } else {
          rs = __builtin_amdgcn_fdot2(hi, (h2){(_Float16)1.f, (_Float16)1.f}, rs, false);   // the sum of what the product takes
        }
        ph[j] = hi[0]; ph[j + 1] = hi[1];
      }
      return rs;
    };
    float rs = weights();
    // The maximum is looked for only where a token's weights say that it has outgrown m, or where there is none yet.  (What rows that
    // take no part hold decides nothing: the columns of a wave look for theirs together, which shows in their last bits)
    if (__any((int)live & (int)(!(rs <= kRoom) | (m == -INFINITY)))) {
      if constexpr (TWO && KIND != MK_Q4) {
        // An infinite K (4-bit scales make it NaN): the score is what the hi half says, whose infinity the lo half's 0 x inf, or infinity of
        // the other sign, would turn into NaN.  The tile's K is still there (the products again: their results kept would spill)
        if (__any(!(rs == rs))) {
#pragma unroll
          for (int mt = 0; mt < 2; mt++) {
            f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KS; k++) t = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, cur.k[mt][k]), q[k], t, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const float other = xchg8_f(t[i]), hi = lr < 8 ? t[i] : other;
              if (y[4 * mt + i] != y[4 * mt + i] && fabsf(hi) == INFINITY) y[4 * mt + i] = hi;   // (masked ones are -inf)
            }
          }
        }
      }
      float bm = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; j++) bm = fmaxf(bm, y[j]);
      bm = pair_max32(pair_max16(bm)) * f;   // f > 0
      const float mn = fmaxf(m, bm), corr = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= corr;
#pragma unroll
      for (int d = 0; d < DT; d++) o[d] *= corr;
      sub = kPBias - (m == -INFINITY ? 0.f : m);
      rs = weights();
    }
    l += rs;
    // what no column sees may hold anything: zeroed (4-bit: its scales), since 0 x NaN is not 0; what only some see, without its
    // NaN and infinite values
    uint32_t bad = 0;
    auto clean = [&](u32x4 w) {
      uint32_t keep = on;
      if (s.PA != s.PB) { const uint32_t n = not_finite(w) & on; bad |= n; keep &= ~n; }
      return __builtin_bit_cast(u32x4, only(__builtin_bit_cast(h8, w), keep));
    };
    if constexpr (KIND == MK_Q4) {
      if (edge) {
#pragma unroll
        for (int i = 0; i < HD / 32; i++) cur.vs[i] = clean(cur.vs[i]);
      }
#pragma unroll
      for (int d = 0; d < DT; d++) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(values(cur.v[d], cur.vs[d / 2]), ph, o[d], 0, 0, 0);
    } else {
      // V's tile in LDS (a wait written out, since the compiler does not see what the loads write)
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (tile + NW < t1) load_k<HD, KIND>(a, h, s, tile + NW, lane, cur);
      // ds_read_b64_tr_b16 hands lane i of 16 the element i % 4 of what lanes 4 j + i / 4 address, as its element j
      const int xr = 8 * lg + (lr >> 2), dq = 4 * (lr & 3);
#pragma unroll
      for (int d = 0; d < DT; d++) {
        const int seg = (16 * d + dq) >> 3, in8 = dq & 4;
        const s4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(vbuf + xr * HD + 8 * (seg ^ vsw<HD>(xr)) + in8));
        const s4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(vbuf + (xr + 4) * HD + 8 * (seg ^ vsw<HD>(xr + 4)) + in8));
        u32x4 w = __builtin_bit_cast(u32x4, (s8)__builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
        if (edge) w = clean(w);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, w), ph, o[d], 0, 0, 0);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the tile is read before the next one's loads write it
    }
    if (tile + NW < t1) load_v<HD, KIND>(a, h, s, tile + NW, lane, cur, vbuf);
    if (__any(bad != 0)) {
#pragma unroll 1
      for (int i = 0; i < kFewTile; i++) {   // record i / 8 is lane group i / 8's
        if (!(__ballot(bad >> (i % kRec) & 1) >> 16 * (i / kRec) & 0xffff)) continue;
        const int r = record(s, 4 * tile + i / kRec), p = kRec * r + i % kRec;
        const bool sp = sees(a, P, lo, p) & (!TWO | (lr < 8));
#pragma unroll
        for (int d = 0; d < DT; d++) add_bad<HD, KIND>(h.rec + (int64_t)r * (9 * HD), h.v + (int64_t)p * a.crow, p, 16 * d + 4 * lg, sp, o[d], 0);
      }
    }
  }
  l = pair_sum32(pair_sum16(l));
  // the waves' sums meet in LDS
  if (KIND != MK_Q4) __syncthreads();   // no wave's V tile is in use
  float *ored = (float *)sm;
#pragma unroll
  for (int d = 0; d < DT; d++) {
    f32x4 y = o[d];
    if (TWO) {
#pragma unroll
      for (int i = 0; i < 4; i++) {   // an infinite V: as the scores, hi's sum where only lo's makes it NaN
        const float both = y[i] + xchg8_f(y[i]);
        y[i] = KIND != MK_Q4 && both != both && fabsf(y[i]) == INFINITY ? y[i] : both;
      }
    }
    if (lr < NC) *(f32x4 *)(ored + (wave * NC + lr) * QS + 16 * d + 4 * lg) = y;
  }
  if (lg == 0 && lr < NC) { wm[wave][lr] = m; wl[wave][lr] = l; }
  __syncthreads();
  const int e = threadIdx.x, c = e / (HD / 4), d = 4 * (e % (HD / 4));
  if (c >= NC) return;
  const int cc = c0 + c, tk = token_of(a, cc);
  if (tk >= s.cnt || (int64_t)s.P0 + tk >= a.ctx) return;
  float M = -INFINITY, L = 0.f;
#pragma unroll
  for (int w = 0; w < NW; w++) M = fmaxf(M, wm[w][c]);
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  const float Mz = M == -INFINITY ? 0.f : M;
#pragma unroll
  for (int w = 0; w < NW; w++) {
    const float k = __builtin_amdgcn_exp2f(wm[w][c] - Mz);
    L += wl[w][c] * k;
    y += *(const f32x4 *)(ored + (w * NC + c) * QS + d) * k;
  }
  const int head = g * a.rep + cc - tk * a.rep;
  if (s.S == 1) {
    const float inv = 1.f / L;   // a visible position's score is -inf only where the plain softmax gives NaN too: 0 x inf
    float r[4];
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = y[i] * inv;
    store_elems<T, 4>(a.out, b * a.out.seq + (int64_t)tk * a.out.tok + (int64_t)head * a.out.head + d, r);
    return;
  }
  const int64_t row = ((int64_t)b * a.n + tk) * a.heads + head, at = row * a.nsplit + split;
  *(f32x4 *)(a.part + at * HD + d) = y;
  if (d == 0) *(float2 *)(a.part + (int64_t)a.nseq * a.n * a.heads * a.nsplit * HD + 2 * at) = make_float2(M, L);
}

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
// 256 registers and spills 4).  256 columns a workgroup, since what a block costs to expand and its LDS writes are
// shared by them: with 128 columns and two workgroups a CU the 4-bit prompt took 77 us for 64, the fp16 one 97 for 100, and 64
// tokens each of 32 sequences 6 % more
constexpr int kManyWaves = 8, kManyBlk = 64, kManyCols = 32 * kManyWaves;

template <int HD, int KIND, int T>
__global__ __launch_bounds__(kManyWaves * 64) void k_kv_many(KvAttnArgs a) {
  constexpr bool TWO = T == RT_F32;
  constexpr int NT = kManyWaves * 64, KQ = HD / 16, OT = HD / 32, BR = kManyBlk / kRec;
  constexpr int KST = HD + 8;                                   // halves of a K row in LDS: an odd number of 16-byte columns
  constexpr int VST = KIND == MK_Q4 ? kManyBlk + 8 : HD + 32;   // of a V^T row (dims), or a V row (positions): 4 rows of 64 bytes apart
  constexpr int VN = KIND == MK_Q4 ? HD * VST : kManyBlk * VST;
  __shared__ __align__(16) uint16_t blocks[3 * (kManyBlk * KST + VN)];
  auto k_of = [&](int kb) { return blocks + kb % 3 * (kManyBlk * KST); };
  auto v_of = [&](int kb) { return blocks + 3 * (kManyBlk * KST) + kb % 3 * VN; };
  __shared__ uint32_t badp[4][2];   // positions of block kb left to add_bad, at (kb - kb0) % 4: set in step kb - 2 or before the first, read in kb, cleared in kb + 1
  const int b = blockIdx.z, g = blockIdx.x, rest = a.nsplit == 1 ? blockIdx.y : blockIdx.y / (uint32_t)a.nsplit, split = blockIdx.y - rest * a.nsplit;
  const int chunk = a.nchunk - 1 - rest;   // without pairs: the last columns, with the most to read, first
  const Span s = span_of(a, b, chunk);
  if (!s.any || split >= s.S) return;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, ln = lane & 31, hf = lane >> 5;
  // waves w and w + 4 share a SIMD: one of the front half, one of the back half
  const int cw = chunk_half(a, chunk, wave / (kManyWaves / 2)) + 32 * (wave % (kManyWaves / 2));
  // (columns past the last read its query, as in k_kv_few; a wave without any other takes no block and uses none of it)
  const int col = min(cw + ln, a.n * a.rep - 1), tok = token_of(a, col), head = g * a.rep + col - tok * a.rep;
  const bool live = col == cw + ln && tok < s.cnt && (int64_t)s.P0 + tok < a.ctx;
  const int P = live ? s.P0 + tok : -1;
  const int lo = behind(a, P);
  // first and last position of the wave's own columns, and of the halves'
  const int wa = token_of(a, cw);
  const bool wlive = wa < s.cnt && (int64_t)s.P0 + wa < a.ctx;
  auto position = [&](int t) { return (int)min((int64_t)s.P0 + min(t, s.cnt - 1), a.ctx - 1); };
  const int PA = s.P0 + wa, PB = position(token_of(a, cw + 31));
  const int A0 = s.PA, B0 = position(last_token(a, chunk_half(a, chunk, 0))), A1 = s.P0 + token_of(a, chunk_half(a, chunk, 1));
  const int kb0 = share(s, split), kb1 = share(s, split + 1);
  const Head hd = head_of<HD, KIND>(a, b, g);

  // ---- a block's codes (or fp16 pieces): memory -> registers -> LDS
  // 4-bit: a thread has W words of a K row, and W of a record's V: dims 16 (W vt + i) + vr of record vl, so that the 16 lanes of a
  // group write V^T rows next to each other.  fp16: pieces tid + NT i
  constexpr int W = HD / 64, NP = KIND == MK_Q4 ? 1 : kManyBlk * HD / 8 / NT;
  typedef uint32_t words __attribute__((ext_vector_type(W)));
  struct Stage { words kq, vq; uint16_t ksc; u32x4 vsc, kp[NP], vp[NP]; };
  const int krow = tid >> 3, kw = tid & 7, vl = tid >> 6, vr = tid & 15, vt = tid >> 4 & 3;
  const uint32_t ko = krow / kRec * (9 * HD) + krow % kRec * (HD / 2) + 4 * W * kw, kso = krow / kRec * (9 * HD) + 8 * HD + 2 * (krow % kRec * (HD / 32) + W * kw / 4);
  const uint32_t vo = vl * (9 * HD) + 4 * HD + vr * (HD / 4) + 4 * W * vt, vso = vl * (9 * HD) + 8 * HD + HD / 2 + 16 * (W * vt / 2);
  int64_t po[NP];
#pragma unroll
  for (int i = 0; i < NP; i++) po[i] = (int64_t)((tid + NT * i) / (HD / 8)) * a.crow + 8 * ((tid + NT * i) % (HD / 8));
  auto fetch = [&](int kb, Stage &g) {
    const int v0 = BR * kb;
    if constexpr (KIND == MK_Q4) {
      if (run_of(s, v0, BR)) {
        const uint8_t *r = hd.rec + (int64_t)record(s, v0) * (9 * HD);
        g.kq = *(const words *)(r + ko); g.ksc = *(const uint16_t *)(r + kso);
        g.vq = *(const words *)(r + vo); g.vsc = *(const u32x4 *)(r + vso);
      } else {
        const uint8_t *r = hd.rec + ((int64_t)record(s, min(v0 + krow / kRec, s.NR - 1)) - krow / kRec) * (9 * HD);
        const uint8_t *rv = hd.rec + ((int64_t)record(s, min(v0 + vl, s.NR - 1)) - vl) * (9 * HD);
        g.kq = *(const words *)(r + ko); g.ksc = *(const uint16_t *)(r + kso);
        g.vq = *(const words *)(rv + vo); g.vsc = *(const u32x4 *)(rv + vso);
      }
    } else {
      const int64_t p0 = (int64_t)kRec * record(s, v0);
      const bool run = run_of(s, v0, BR) && p0 + kManyBlk <= a.ctx;
      const uint16_t *k0 = hd.k + p0 * a.crow, *v00 = hd.v + p0 * a.crow;
#pragma unroll
      for (int i = 0; i < NP; i++) {
        const int c = tid + NT * i, x = c / (HD / 8), sg = c % (HD / 8);
        if (run) { g.kp[i] = *(const u32x4 *)(k0 + po[i]); g.vp[i] = *(const u32x4 *)(v00 + po[i]); }
        else {
          const int64_t at = row_of(a, s, v0 + x / kRec, x % kRec) + 8 * sg;
          g.kp[i] = *(const u32x4 *)(hd.k + at);
          g.vp[i] = *(const u32x4 *)(hd.v + at);
        }
      }
    }
  };
  // Blocks by number.  A block from the window's on holds positions 64 kb + 8 skip ..; those before it (the first positions that stay
  // visible) count as seen in part.  Of tokens A .. B: from whole(A) on A does not see all of a block, before left(B) B does not,
  // ends(B) is the last that B sees some of.  (Comparisons with these few numbers: worked out anew for every block, they were a
  // third of the loop's instructions, and a wave issues one in about ten cycles)
  const int NRb = s.NR / BR, R0 = s.skip ? (s.SR + BR - 1) / BR : 0, off = kRec * s.skip;
  auto whole = [&](int A) { return min((A + 1 - off) >> 6, NRb); };
  auto left = [&](int B) { return a.window > 0 ? max((B - a.window - off) >> 6, -1) + 1 : 0; };
  auto ends = [&](int B) { return (B - off) >> 6; };
  static_assert(kManyBlk == 64, "the shifts above");
  const int wK = whole(PA), wY = max(left(PB), R0), wE = wlive ? ends(PB) : -1;          // the wave's
  const int gK0 = whole(A0), gE0 = ends(B0), gK1 = whole(A1), gY = max(left(s.PB), R0);   // the workgroup's halves'
  auto partial = [&](int kb) { return (kb >= wK) | (kb < wY); };
  // the same of the waves that take the block: a wave does not take a block behind its last position
  auto partial_any = [&](int kb) { return ((kb >= gK0) & (kb <= gE0)) | (kb >= gK1) | (kb < gY); };
  // what no column sees zeroed, and what only some see without its NaN and infinite values (4-bit: by the scales)
  auto clean = [&](int kb, Stage &g) {
    if constexpr (KIND == MK_Q4) {
      const int v = BR * kb + vl;
      const uint32_t on = seen_bits(a, s, v, kRec * record(s, min(v, s.NR - 1))), bad = on & not_finite(g.vsc);
      if (bad) atomicOr(&badp[(kb - kb0) % 4][vl / 4], bad << 8 * (vl % 4));
      g.vsc = __builtin_bit_cast(u32x4, only(__builtin_bit_cast(h8, g.vsc), on & ~bad));
    } else {
#pragma unroll
      for (int i = 0; i < NP; i++) {
        const int x = (tid + NT * i) / (HD / 8), v = BR * kb + x / kRec;
        const uint32_t on = seen_bits(a, s, v, kRec * record(s, min(v, s.NR - 1))) >> x % kRec & 1 ? 255u : 0u, bad = on & not_finite(g.vp[i]);
        if (bad) atomicOr(&badp[(kb - kb0) % 4][x / 32], 1u << x % 32);
        g.vp[i] = __builtin_bit_cast(u32x4, only(__builtin_bit_cast(h8, g.vp[i]), on & ~bad));
      }
    }
  };
  auto expand = [&](int kb, Stage &g) {
    uint16_t *kd = k_of(kb), *vd = v_of(kb);
    if constexpr (KIND == MK_Q4) {
#pragma unroll
      for (int i = 0; i < W; i++) {
        *(h8 *)(kd + krow * KST + 8 * (W * kw + i)) = values(g.kq[i], g.ksc);
        *(h8 *)(vd + (16 * (W * vt + i) + vr) * VST + kRec * vl) = values(g.vq[i], g.vsc);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NP; i++) {
        const int c = tid + NT * i, x = c / (HD / 8), sg = c % (HD / 8);
        *(u32x4 *)(kd + x * KST + 8 * sg) = g.kp[i];
        *(u32x4 *)(vd + x * VST + 8 * sg) = g.vp[i];
      }
    }
  };
  if (tid < 8) badp[tid / 2][tid % 2] = 0;
  h8 q[KQ], ql[TWO ? KQ : 1];
  float f = a.scale2;
  Stage st;
  {  // the first two blocks, asked for together
    Stage st1;
    fetch(kb0, st);
    if (kb0 + 1 < kb1) fetch(kb0 + 1, st1);
    // ---- queries
    {
      const int64_t at = b * a.q.seq + (int64_t)tok * a.q.tok + (int64_t)head * a.q.head + 8 * hf;
      float x[KQ][8], mx = 0.f;
#pragma unroll
      for (int k = 0; k < KQ; k++) {
        if constexpr (T == RT_F16) q[k] = load_halves(a.q, at + 16 * k);
        else {
          load_elems<T, 8>(a.q, at + 16 * k, x[k]);
#pragma unroll
          for (int j = 0; j < 8; j++) mx = fmaxf(mx, fabsf(x[k][j]));
        }
      }
      if constexpr (T != RT_F16) {
        mx = pair_max32(mx);
        const float p2 = row_power(mx);
        f = fminf(fmaxf(f / p2, kTinyF), kMostF);
#pragma unroll
        for (int k = 0; k < KQ; k++)
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const float y = x[k][j] * p2;
            const _Float16 h = (_Float16)y;
            q[k][j] = h;
            if constexpr (TWO) ql[k][j] = (_Float16)(y - (float)h);
          }
      }
    }
    __syncthreads();   // badp
    if (partial_any(kb0)) clean(kb0, st);
    expand(kb0, st);
    if (kb0 + 1 < kb1) {
      if (partial_any(kb0 + 1)) clean(kb0 + 1, st1);
      expand(kb0 + 1, st1);
    }
  }
  if (kb0 + 2 < kb1) fetch(kb0 + 2, st);
  __syncthreads();
  f32x16 o[OT];
#pragma unroll
  for (int t = 0; t < OT; t++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[t][i] = 0.f;
  float m = -INFINITY, l = 0.f;
  // LDS row of the lane's K row
  const int kr = (ln & 16) | (ln & 4) << 1 | (ln & 8) >> 1 | (ln & 3);
  auto vfrag = [&](const uint16_t *v, int t, int u) {
    if constexpr (KIND == MK_Q4) return *(const h8 *)(v + (32 * t + ln) * VST + 16 * u + 8 * hf);
    else {
      const int r = lane & 15, x = 16 * u + 8 * hf + (r >> 2), d = 32 * t + (ln & 16) + 4 * (r & 3);
      const s4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(v + x * VST + d));
      const s4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(v + (x + 4) * VST + d));
      return __builtin_bit_cast(h8, (s8)__builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  };
  h8 ph[4], pl[TWO ? 4 : 1];
  f32x16 sc[2];
  auto dots = [&](int kb) {   // K q of a block
    const uint16_t *kl = k_of(kb);
#pragma unroll
    for (int mt = 0; mt < 2; mt++) {
#pragma unroll
      for (int i = 0; i < 16; i++) sc[mt][i] = 0.f;
#pragma unroll
      for (int k = 0; k < KQ; k++) {
        const h8 kf = *(const h8 *)(kl + (32 * mt + kr) * KST + 16 * k + 8 * hf);
        sc[mt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, q[k], sc[mt], 0, 0, 0);
        if constexpr (TWO) sc[mt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, ql[k], sc[mt], 0, 0, 0);
      }
    }
  };
  float sub = kPBias;
  auto weights = [&]() {   // sc -> ph, pl and their sum over the lane's positions
    float rs = 0.f;
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u >> 1][8 * (u & 1) + j], f, sub));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u >> 1][8 * (u & 1) + j + 1], f, sub));
        const h2 h = {(_Float16)p0, (_Float16)p1};
        ph[u][j] = h[0]; ph[u][j + 1] = h[1];
        if constexpr (TWO) {
          rs += p0; rs += p1;
          pl[u][j] = (_Float16)(p0 - (float)h[0]); pl[u][j + 1] = (_Float16)(p1 - (float)h[1]);
        } else {
          rs = __builtin_amdgcn_fdot2(h, (h2){(_Float16)1.f, (_Float16)1.f}, rs, false);   // the sum of what the product takes
        }
      }
    return rs;
  };
  auto product = [&](int kb) {
    const uint16_t *vb = v_of(kb);
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
      for (int t = 0; t < OT; t++) {
        const h8 x = vfrag(vb, t, u);
        o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, ph[u], o[t], 0, 0, 0);
        if constexpr (TWO) o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, pl[u], o[t], 0, 0, 0);
      }
  };
  auto fix = [&](int kb) {
#pragma unroll 1
      for (int w = 0; w < 2; w++) {
        uint32_t bad = __builtin_amdgcn_readfirstlane(badp[(kb - kb0) % 4][w]);
        while (bad) {
          const int x = 32 * w + __builtin_ctz(bad), r = record(s, BR * kb + x / kRec), p = kRec * r + x % kRec;
          const bool sp = sees(a, P, lo, p);
          bad &= bad - 1;
#pragma unroll
          for (int t = 0; t < OT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) add_bad<HD, KIND>(hd.rec + (int64_t)r * (9 * HD), hd.v + (int64_t)p * a.crow, p, 32 * t + 8 * i + 4 * hf, sp, o[t], 4 * i);
        }
      }
  };
  auto first = [&](int kb) { return kRec * record(s, BR * kb); };
  auto last = [&](int kb) { return kRec * record(s, min(BR * kb + BR - 1, s.NR - 1)) + kRec - 1; };
  // Step kb: K q, the weights, then P V beside the expansion of block kb + 2 (whose codes were asked for a step ago); kb + 3 is asked for.
  // Two blocks ahead, not one: 4 % less time
  for (int kb = kb0; kb < kb1; kb++) {
    if (kb + 2 < kb1 && partial_any(kb + 2)) clean(kb + 2, st);
    // one of the wave's columns sees some of the block?  (Read through the lane: left to itself the compiler splits the loop at wE and
    // keeps two copies of o, 58 registers more)
    const int before = (int)(a.window > 0) & (int)(kb < wY) & (int)(last(kb) <= PA - a.window) & (int)(first(kb) >= a.sinks);
    if (__builtin_amdgcn_readfirstlane((int)(kb <= wE) & (before ^ 1))) {
      dots(kb);
      if (partial(kb)) {
#pragma unroll
        for (int u = 0; u < 4; u++) {
          const int v = BR * kb + 2 * u + hf, p0 = kRec * record(s, min(v, s.NR - 1)), Pin = v < s.NR ? P : -1;
#pragma unroll
          for (int j = 0; j < 8; j++) sc[u >> 1][8 * (u & 1) + j] = sees(a, Pin, lo, p0 + j) ? sc[u >> 1][8 * (u & 1) + j] : -INFINITY;
        }
      }
      float rs = weights();
      // as in k_kv_few, by the tokens' columns alone
      if (__any((int)live & (int)(!(rs <= kRoom) | (m == -INFINITY)))) {
        if constexpr (TWO && KIND != MK_Q4) {
          // An infinite K, as in k_kv_few: where the sum is NaN (the masked are -inf) and hi's product alone infinite, that is the score
          if (__any(!(rs == rs))) {
            const uint16_t *kl = k_of(kb);
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
              f32x16 t;
#pragma unroll
              for (int i = 0; i < 16; i++) t[i] = 0.f;
#pragma unroll
              for (int k = 0; k < KQ; k++) t = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const h8 *)(kl + (32 * mt + kr) * KST + 16 * k + 8 * hf), q[k], t, 0, 0, 0);
#pragma unroll
              for (int i = 0; i < 16; i++)
                if (sc[mt][i] != sc[mt][i] && fabsf(t[i]) == INFINITY) sc[mt][i] = t[i];
            }
          }
        }
        float bm = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
          for (int i = 0; i < 16; i++) bm = fmaxf(bm, sc[mt][i]);
        bm = pair_max32(bm) * f;   // f > 0
        const float mn = fmaxf(m, bm), corr = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= corr;
#pragma unroll
        for (int t = 0; t < OT; t++) o[t] *= corr;
        sub = kPBias - (m == -INFINITY ? 0.f : m);
        rs = weights();
      }
      l += rs;
      product(kb);
      expand(kb + 2, st);   // (past the last block: what the registers hold, to a place that is not read again)
      if (partial_any(kb)) fix(kb);   // (also for the columns of a wave that see all of it)
    } else {
      expand(kb + 2, st);
    }
    if (kb + 3 < kb1) fetch(kb + 3, st);
    if (tid < 2) badp[(kb - kb0 + 3) % 4][tid] = 0;
    __syncthreads();
  }
  l = pair_sum32(l);
  if constexpr (TWO && KIND != MK_Q4) {
    // An infinite V: the lo halves (0, or of either sign) turn the sum into NaN.  Such sums are what the values say that are not finite and
    // that the column sees, read again.  (Where l is NaN a score was, and the row is)
    bool nan = false;
#pragma unroll
    for (int t = 0; t < OT; t++)
#pragma unroll
      for (int i = 0; i < 16; i++) nan |= o[t][i] != o[t][i];
    if (__any((int)live & (int)nan & (int)(l == l))) {
#pragma unroll
      for (int t = 0; t < OT; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[t][i] = o[t][i] != o[t][i] ? 0.f : o[t][i];
#pragma unroll 1
      for (int64_t i = (int64_t)kManyBlk * kb0; i < min((int64_t)kManyBlk * kb1, (int64_t)kRec * s.NR); i++) {
        const int p = kRec * record(s, (int)(i / kRec)) + (int)(i % kRec);
        const bool sp = sees(a, P, lo, p);
        if (!__any(sp)) continue;   // (also the positions past ctx)
#pragma unroll
        for (int t = 0; t < OT; t++)
#pragma unroll
          for (int j = 0; j < 4; j++) add_bad<HD, KIND>(nullptr, hd.v + (int64_t)p * a.crow, p, 32 * t + 8 * j + 4 * hf, sp, o[t], 4 * j);
      }
    }
  }
  if constexpr (T != RT_F32) {
    if (s.S == 1) {
      // A lane has 4 dims here and there of its column; by way of the wave's own part of LDS the rows leave in 16-byte pieces
      // next to each other (4096 tokens with 32 heads: 105 -> 101 us)
      constexpr int RS = HD + 8;
      static_assert(kManyWaves * 32 * RS <= 3 * (kManyBlk * KST + VN), "the columns fit where the blocks were");
      uint16_t *ow = blocks + wave * 32 * RS;
      const float inv = 1.f / l;
      const KvRows lds{ow + ln * RS, T, 0, 0, 0};
#pragma unroll
      for (int t = 0; t < OT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float r[4] = {o[t][4 * i] * inv, o[t][4 * i + 1] * inv, o[t][4 * i + 2] * inv, o[t][4 * i + 3] * inv};
          store_elems<T, 4>(lds, 32 * t + 8 * i + 4 * hf, r);
        }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      constexpr int LR = HD / 8, RI = 64 / LR;   // lanes of a row, rows at a time
#pragma unroll
      for (int i = 0; i < 32 / RI; i++) {
        const int c = RI * i + lane / LR, cc = cw + c, tk = token_of(a, cc);
        if (tk < s.cnt && (int64_t)s.P0 + tk < a.ctx) {
          const int64_t at = b * a.out.seq + (int64_t)tk * a.out.tok + (int64_t)(g * a.rep + cc - tk * a.rep) * a.out.head + 8 * (lane % LR);
          *(u32x4_any *)((uint16_t *)a.out.p + at) = *(const u32x4 *)(ow + c * RS + 8 * (lane % LR));
        }
      }
      return;
    }
  }
  if (!live) return;
  if (s.S == 1) {
    const float inv = 1.f / l;
    const int64_t at = b * a.out.seq + (int64_t)tok * a.out.tok + (int64_t)head * a.out.head;
#pragma unroll
    for (int t = 0; t < OT; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float r[4] = {o[t][4 * i] * inv, o[t][4 * i + 1] * inv, o[t][4 * i + 2] * inv, o[t][4 * i + 3] * inv};
        store_elems<T, 4>(a.out, at + 32 * t + 8 * i + 4 * hf, r);
      }
    return;
  }
  const int64_t row = ((int64_t)b * a.n + tok) * a.heads + head, at = row * a.nsplit + split;
#pragma unroll
  for (int t = 0; t < OT; t++)
#pragma unroll
    for (int i = 0; i < 4; i++)
      *(f32x4 *)(a.part + at * HD + 32 * t + 8 * i + 4 * hf) = (f32x4){o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]};
  if (hf == 0) *(float2 *)(a.part + (int64_t)a.nseq * a.n * a.heads * a.nsplit * HD + 2 * at) = make_float2(m, l);
}

// ------------------------------------------------------------------ launches
// KERNEL<HD, T> by head dim and rows' type
#define QPH_KV(KERNEL, hd, type, grid, threads, a)                                                                      \
  do {                                                                                                                  \
    const dim3 g_ = (grid), t_(threads);                                                                                \
    if ((hd) == 128) {                                                                                                  \
      if ((type) == RT_F32) hipLaunchKernelGGL((KERNEL<128, RT_F32>), g_, t_, 0, st, a);                                \
      else if ((type) == RT_F16) hipLaunchKernelGGL((KERNEL<128, RT_F16>), g_, t_, 0, st, a);                           \
      else hipLaunchKernelGGL((KERNEL<128, RT_BF16>), g_, t_, 0, st, a);                                                \
    } else {                                                                                                            \
      if ((type) == RT_F32) hipLaunchKernelGGL((KERNEL<64, RT_F32>), g_, t_, 0, st, a);                                 \
      else if ((type) == RT_F16) hipLaunchKernelGGL((KERNEL<64, RT_F16>), g_, t_, 0, st, a);                            \
      else hipLaunchKernelGGL((KERNEL<64, RT_BF16>), g_, t_, 0, st, a);                                                 \
    }                                                                                                                   \
  } while (0)
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
size_t kv_attn_plan(KvAttnArgs &a) {
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
  a.min_log2 = a.many ? 2 : 3;    // tiles of a split, at least
  a.one_tiles = a.many ? 4 : 4 * kFewWaves;
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

}  // namespace qph
