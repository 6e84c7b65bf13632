// Log probabilities of given tokens, with the entropy, the tokens' ranks and the most probable alternatives, in one pass over the logits.
//
// A row x of V logits, any reference m: s = sum e^(x - m), t = sum (x - m) e^(x - m);
//   log p_i = x_i - m - ln s,   entropy = -sum p ln p = ln s - t / s
// m is a wave's: a maximum as it was when a logit last passed it by more than kRoom, so that the sums are scaled again a few times a row and not at
// every step.  x - m is one rounding off and e^(x - m) its own size times 2^-24 and two of the exponential's last places; sums are fp32, a thread's own,
// then added as a tree.
//
// The alternatives: a wave keeps the K <= 64 first of what it has seen in order, one a lane, and inserts what precedes the last of them.  Its indices
// rise, so that among equal values the list's own come first and a comparison of values decides.  Of a random row few logits pass: K ln(V / 512) a wave
// or so; the first 64 lanes' worth is cut down first, to what reaches the K-th largest of the lanes' maxima.
//
// A workgroup of 4 waves has a row, or a share of one where there are few; shares leave sums and lists that k_logprobs_merge joins.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

#include "kvrec.hpp"
#include "launch.hpp"

namespace qph {

namespace {
constexpr int kLpWaves = 4;
constexpr float kLpRoom = 6.f, kLog2e = 1.44269504088896341f;

// values' order as whole numbers' (-0 as 0); kNone precedes none of them
constexpr int kNone = INT_MIN;
__device__ __forceinline__ int order_of(float x) {
  const int b = __builtin_bit_cast(int, x + 0.f);
  return b ^ (b >> 31 & 0x7fffffff);
}
__device__ __forceinline__ float value_of(int o) { return __builtin_bit_cast(float, o ^ (o >> 31 & 0x7fffffff)); }
__device__ __forceinline__ bool before(int o, int i, int o2, int i2) { return o > o2 || (o == o2 && i < i2); }

template <int T>
constexpr int lp_elems() { return T == RT_F32 ? 4 : 8; }   // of 16 bytes
template <int T>
__device__ __forceinline__ float lp_elem(u32x4 w, int i) {
  if constexpr (T == RT_F32) { const uint32_t u = w[i]; return __builtin_bit_cast(float, u); }
  else {
    const uint32_t u = w[i / 2];
    if constexpr (T == RT_F16) return half_bits_to_float((uint16_t)(u >> 16 * (i & 1)));
    return __builtin_bit_cast(float, i & 1 ? u & 0xffff0000u : u << 16);
  }
}
template <int T>
__device__ __forceinline__ float lp_load(const void *p, int64_t i) {
  if constexpr (T == RT_F32) return ((const float *)p)[i];
  else { const uint16_t h = ((const uint16_t *)p)[i]; return T == RT_F16 ? half_bits_to_float(h) : bf16_to_f(h); }
}
// what a share of a row comes to
struct LpSum { float m, s, t; int ahead; };
__device__ __forceinline__ float ref(float m) { return m == -INFINITY ? 0.f : m; }
// a difference as a factor: past -kFar its exponential is 0, and products with it stay finite (a mask of a type's lowest value is a finite logit)
constexpr float kFar = 1e20f;
__device__ __forceinline__ float near(float d) { return fmaxf(d, -kFar); }
// b's sums brought to a's reference and added: e^(x - m') = e^(x - m) e^(m - m'), x - m' = (x - m) + (m - m')
__device__ __forceinline__ void join(LpSum &a, const LpSum &b) {
  const float m = fmaxf(a.m, b.m), z = ref(m);
  const float da = a.m == -INFINITY ? 0.f : near(a.m - z), db = b.m == -INFINITY ? 0.f : near(b.m - z);   // (without a reference all is 0 or NaN)
  const float ca = __builtin_amdgcn_exp2f(da * kLog2e), cb = __builtin_amdgcn_exp2f(db * kLog2e);
  a.t = (a.t + a.s * da) * ca + (b.t + b.s * db) * cb;
  a.s = a.s * ca + b.s * cb;
  a.m = m;
  a.ahead += b.ahead;
}
// a list's entry into the outputs
__device__ __forceinline__ void put_top(const LogprobArgs &a, int64_t row, int k, int o, int i, float m, float ls) {
  a.top_index[row * a.top + k] = o == kNone ? -1 : i;
  a.top_logp[row * a.top + k] = o == kNone ? __builtin_nanf("") : value_of(o) - ref(m) - ls;
}
__device__ __forceinline__ void put(const LogprobArgs &a, int64_t row, const LpSum &s, float ls, float xt, bool has) {
  if (a.logp) a.logp[row] = has ? xt - ref(s.m) - ls : __builtin_nanf("");
  if (a.rank) a.rank[row] = has ? s.ahead : -1;
  if (a.entropy) a.entropy[row] = ls - s.t / s.s;
}

// a wave's list: lane i < K has the i-th
struct LpList { int o = kNone, i = 0; };
__device__ __forceinline__ void insert(LpList &l, int lane, int o, int i) {
  const int p = __popcll(__ballot(l.o >= o));   // (kNone below all)
  const int so = __builtin_amdgcn_update_dpp(0, l.o, 0x138, 0xf, 0xf, false), si = __builtin_amdgcn_update_dpp(0, l.i, 0x138, 0xf, 0xf, false);   // wave_shr:1
  l.o = lane < p ? l.o : lane == p ? o : so;
  l.i = lane < p ? l.i : lane == p ? i : si;
}

template <int T, bool TOP>
__global__ __launch_bounds__(kLpWaves * 64) void k_logprobs(LogprobArgs a) {
  constexpr int VE = lp_elems<T>(), GE = 64 * VE, U = 4;   // elements of a lane's load, of a wave's; loads on their way
  __shared__ LpSum sums[kLpWaves];
  __shared__ int lo[kLpWaves * kLpTop], li[kLpWaves * kLpTop];
  const int64_t row = blockIdx.x / (uint32_t)a.splits;
  const int split = blockIdx.x - (int)row * a.splits;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int from = split * a.share, to = min(a.vocab, from + a.share);
  const int esize = T == RT_F32 ? 4 : 2;
  const uint8_t *x0 = (const uint8_t *)a.x + row * a.ld * esize;
  const int token = a.tokens ? a.tokens[row] : -1;
  const bool has = token >= 0 && token < a.vocab;
  const float xt = has ? lp_load<T>(x0, token) : INFINITY;
  LpSum s{-INFINITY, 0.f, 0.f, 0};
  LpList list;
  float last = 0.f;   // value of the list's K-th
  bool first = true;
  auto load = [&](int at) -> u32x4 {   // a lane's elements from at on
    if (at + VE <= to) return *(const u32x4_any *)(x0 + (int64_t)at * esize);
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (T == RT_F32) w[i] = at + i < to ? ((const uint32_t *)x0)[at + i] : 0xff800000u;
      else {
        const uint32_t none = T == RT_F16 ? 0xfc00u : 0xff80u;
        const uint32_t u0 = at + 2 * i < to ? ((const uint16_t *)x0)[at + 2 * i] : none, u1 = at + 2 * i + 1 < to ? ((const uint16_t *)x0)[at + 2 * i + 1] : none;
        w[i] = u0 | u1 << 16;
      }
    }
    return w;
  };
  auto take = [&](u32x4 w, int base) {   // a wave's elements base .., those past `to` -inf
    const int at = base + VE * lane;
    float x[VE], bm = -INFINITY;
#pragma unroll
    for (int i = 0; i < VE; i++) { x[i] = lp_elem<T>(w, i); bm = fmaxf(bm, x[i]); }
    if (__any(bm > s.m + kLpRoom)) {   // (always while there is none)
      const float m = wave_max(bm);
      if (m > s.m) {
        const float d = s.m == -INFINITY ? 0.f : near(s.m - m), c = __builtin_amdgcn_exp2f(d * kLog2e);
        s.t = (s.t + s.s * d) * c;
        s.s *= c;
        s.m = m;
      }
    }
    const float z = ref(s.m);
#pragma unroll
    for (int i = 0; i < VE; i++) {
      const float d = x[i] - z, e = __builtin_amdgcn_exp2f(d * kLog2e);
      s.s += e;
      s.t = __builtin_fmaf(e, near(d), s.t);   // (0 x inf; a NaN is in s)
    }
    if (base + GE <= token) {
#pragma unroll
      for (int i = 0; i < VE; i++) s.ahead += x[i] >= xt;
    } else if (base > token) {
#pragma unroll
      for (int i = 0; i < VE; i++) s.ahead += x[i] > xt;
    } else {
#pragma unroll
      for (int i = 0; i < VE; i++) s.ahead += (x[i] > xt) | ((x[i] == xt) & (at + i < token));
    }
    if constexpr (TOP) {
      if (first) {
        // the K-th largest of the lanes' first ones bounds the K-th largest of all from below
        first = false;
        int o[VE], mo = kNone;
#pragma unroll
        for (int i = 0; i < VE; i++) { o[i] = at + i < to ? order_of(x[i]) : kNone; mo = max(mo, o[i]); }
        int n = 0;
#pragma unroll 8
        for (int l = 0; l < 64; l++) {
          const int other = __builtin_amdgcn_readlane(mo, l);
          n += other > mo || (other == mo && l < lane);
        }
        const int bound = __builtin_amdgcn_readlane(mo, __builtin_ctzll(__ballot(n == a.top - 1)));
        uint64_t lanes = __ballot(mo >= bound && mo != kNone);
        while (lanes) {
          const int l = __builtin_ctzll(lanes);
          lanes &= lanes - 1;
#pragma unroll
          for (int i = 0; i < VE; i++) {
            const int v = __builtin_amdgcn_readlane(o[i], l);
            if (v >= bound && v != kNone) insert(list, lane, v, base + VE * l + i);
          }
        }
      } else {
        uint64_t lanes = __ballot(bm > last);
        if (!lanes) return;
        while (lanes) {
          const int l = __builtin_ctzll(lanes);
          lanes &= lanes - 1;
          int lo = __builtin_amdgcn_readlane(list.o, a.top - 1);
#pragma unroll
          for (int i = 0; i < VE; i++) {
            const int v = order_of(__builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x[i]), l)));
            if (v > lo) { insert(list, lane, v, base + VE * l + i); lo = __builtin_amdgcn_readlane(list.o, a.top - 1); }
          }
        }
      }
      last = value_of(__builtin_amdgcn_readlane(list.o, a.top - 1));
    }
  };
  u32x4 w[U];
  int base = from + GE * wave;
  constexpr int STEP = GE * kLpWaves;
#pragma unroll
  for (int u = 0; u < U; u++) if (base + u * STEP < to) w[u] = load(base + u * STEP + VE * lane);
  while (base < to) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (base < to) {
        const u32x4 now = w[u];
        if (base + U * STEP < to) w[u] = load(base + U * STEP + VE * lane);
        take(now, base);
      }
      base += STEP;
    }
  }
  // lanes share the reference; then the waves
  s.s = wave_sum(s.s); s.t = wave_sum(s.t);
  s.ahead = sum32_i(s.ahead);
  s.ahead += __shfl_xor(s.ahead, 32);
  if (lane == 0) sums[wave] = s;
  if constexpr (TOP) {
    if (lane < a.top) { lo[wave * a.top + lane] = list.o; li[wave * a.top + lane] = list.i; }
  }
  __syncthreads();
  LpSum all = sums[0];
#pragma unroll
  for (int i = 1; i < kLpWaves; i++) join(all, sums[i]);
  const float ls = logf(all.s);
  const int64_t part = row * a.splits + split;
  if (threadIdx.x == 0) {
    if (a.splits == 1) put(a, row, all, ls, xt, has);
    else ((LpSum *)a.work)[part] = all;
  }
  if constexpr (TOP) {
    // an entry's place among all is the number before it (those of kNone are alike, in the lists' order)
    const int e = threadIdx.x;
    if (e < kLpWaves * a.top) {
      const int o = lo[e], i = o == kNone ? INT_MAX : li[e];
      int n = 0;
      for (int j = 0; j < kLpWaves * a.top; j++) {
        const int oj = lo[j], ij = oj == kNone ? INT_MAX : li[j];
        n += before(oj, ij, o, i) || (oj == kNone && o == kNone && j < e);
      }
      if (n < a.top) {
        if (a.splits == 1) put_top(a, row, n, o, i, all.m, ls);
        else ((int2 *)((LpSum *)a.work + a.rows * a.splits))[part * a.top + n] = make_int2(o, i);
      }
    }
  }
}

// The shares of a row: a workgroup joins their sums and picks the first K of their lists
template <int T>
__global__ __launch_bounds__(256) void k_logprobs_merge(LogprobArgs a) {
  constexpr int kMost = kLpSplits * kLpTop;
  __shared__ LpSum all;
  __shared__ int heads[kLpSplits], bound, count;
  __shared__ int co[kMost], ci[kMost];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, S = a.splits;
  const LpSum *sums = (const LpSum *)a.work + row * S;
  const int2 *lists = (const int2 *)((const LpSum *)a.work + a.rows * S) + row * S * a.top;
  if (tid < S && a.top) heads[tid] = lists[tid * a.top].x;
  if (tid == 0) { count = 0; bound = kNone; }
  if (tid < 64) {
    LpSum s = tid < S ? sums[tid] : LpSum{-INFINITY, 0.f, 0.f, 0};
#pragma unroll
    for (int d = 32; d; d >>= 1) join(s, LpSum{__shfl_xor(s.m, d), __shfl_xor(s.s, d), __shfl_xor(s.t, d), __shfl_xor(s.ahead, d)});
    if (tid == 0) all = s;
  }
  __syncthreads();
  const float ls = logf(all.s);
  if (tid == 0) {
    const int token = a.tokens ? a.tokens[row] : -1;
    const bool has = token >= 0 && token < a.vocab;
    put(a, row, all, ls, has ? lp_load<T>((const uint8_t *)a.x + row * a.ld * (T == RT_F32 ? 4 : 2), token) : 0.f, has);
  }
  if (!a.top) return;
  // what lies behind the K-th of the lists' first entries is not among the first K
  if (tid < S && S >= a.top) {
    int n = 0;
    for (int j = 0; j < S; j++) n += heads[j] > heads[tid] || (heads[j] == heads[tid] && j < tid);
    if (n == a.top - 1) bound = heads[tid];
  }
  __syncthreads();
  for (int e = tid; e < S * a.top; e += 256) {
    const int2 x = lists[e];
    if (x.x >= bound && x.x != kNone) { const int c = atomicAdd(&count, 1); co[c] = x.x; ci[c] = x.y; }
  }
  __syncthreads();
  for (int e = tid; e < max(count, a.top); e += 256) {
    if (e >= count) { put_top(a, row, e, kNone, 0, all.m, ls); continue; }   // fewer than K (a vocabulary of NaN)
    int n = 0;
    for (int j = 0; j < count; j++) n += before(co[j], ci[j], co[e], ci[e]);
    if (n < a.top) put_top(a, row, n, co[e], ci[e], all.m, ls);
  }
}
}  // namespace

size_t logprobs_plan(LogprobArgs &a) {
  // A workgroup's pass over its share is a chain of loads: rows are shared out until there are four workgroups a CU, in
  // pieces of a wave's load for each of its waves
  const int unit = kLpWaves * 64 * (a.type == RT_F32 ? 4 : 8);
  const int units = (a.vocab + unit - 1) / unit;
  const int want = (int)std::min<int64_t>(std::max<int64_t>(1024 / a.rows, 1), std::min(units, kLpSplits));
  const int each = (units + want - 1) / want;
  a.share = (int)std::min<int64_t>((int64_t)each * unit, INT_MAX);
  a.splits = (units + each - 1) / each;
  return a.splits == 1 ? 0 : (size_t)a.rows * a.splits * (sizeof(LpSum) + 8 * a.top);
}
hipError_t launch_logprobs(const LogprobArgs &a, hipStream_t st) {
  const dim3 grid((unsigned)(a.rows * a.splits)), thr(kLpWaves * 64);
#define QPH_LP(T)                                                                          \
  do {                                                                                     \
    if (a.top) hipLaunchKernelGGL((k_logprobs<T, true>), grid, thr, 0, st, a);             \
    else hipLaunchKernelGGL((k_logprobs<T, false>), grid, thr, 0, st, a);                  \
    const hipError_t e = hipGetLastError();                                                \
    if (e != hipSuccess || a.splits == 1) return e;                                        \
    hipLaunchKernelGGL((k_logprobs_merge<T>), dim3((unsigned)a.rows), dim3(256), 0, st, a);\
  } while (0)
  if (a.type == RT_F32) QPH_LP(RT_F32);
  else if (a.type == RT_F16) QPH_LP(RT_F16);
  else QPH_LP(RT_BF16);
#undef QPH_LP
  return hipGetLastError();
}

}  // namespace qph
