// The key / value caches' elements: rows of tokens, the 4-bit cache's codes and scales (the format: kvcache.hip).  For the kernels of kvcache.hip and kvstep.hip.
#pragma once
#include <hip/hip_runtime.h>

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

// bits of the V codes of a record's positions p0 .. that lie outside from .. to - 1
__device__ __forceinline__ uint32_t kept_bits(int64_t p0, int64_t from, int64_t to) {
  uint32_t keep = 0;
#pragma unroll
  for (int i = 0; i < kRec; i++)
    if (!(p0 + i >= from && p0 + i < to)) keep |= 15u << nib(i);
  return keep;
}
// A wave's K (V) rows of a record: lane = position row = lane / 8, dims HD / 8 part .. by load(x), part = lane % 8, where the position is `mine`.  Others keep their codes
// and scales: their K rows and scales are not stored, and V words, which hold all 8 positions, are merged: the record's positions are p0 .., the call's
// from .. to - 1.  codes: LDS, the V wave's
template <int HD, int T, typename Load, typename Record>
__device__ __forceinline__ void store_record(Load load, Record record, bool mine, bool vside, int row, int part, int64_t p0, int64_t from, int64_t to, uint8_t (*codes)[HD]) {
  constexpr int EL = HD / 8, GL = 32 / EL;   // elements of a lane; lanes of a group
  float x[EL];
  uint32_t mx = 0;
  if (mine) {
    load(x);
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
  uint8_t *o = record();
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
  const int lane = 8 * row + part;
  const uint32_t keep = kept_bits(p0, from, to);
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
// A wave's one row of K (V) at position `row` of the record at o: lane's dims HD / 64 lane .. in x.  Lanes of a K word meet by DPP; a V word is read and its one
// code replaced
template <int HD, int T>
__device__ __forceinline__ void store_one(uint8_t *o, int row, const float *x, bool vside, int lane) {
  constexpr int EL = HD / 64;
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
}  // namespace

}  // namespace qph
