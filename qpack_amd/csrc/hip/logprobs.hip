// Log probabilities of given tokens, with the entropy, the tokens' ranks and the most probable alternatives, in one pass over the logits.
//
// A row x of V logits, any reference m: s = sum e^(x - m), t = sum (x - m) e^(x - m);
//   log p_i = x_i - m - ln s,   entropy = -sum p ln p = ln s - t / s
// m is a wave's: a maximum as it was when a logit last passed it by more than kRoom, so that the sums are scaled again a few times a row and not at
// every step.  x - m is one rounding off and e^(x - m) its own size times 2^-24 and two of the exponential's last places; sums are fp32, a thread's own,
// then added as a tree.
//
// The alternatives: a wave keeps in LDS what of its logits may be among the K <= 64 first, and a bound that K of them reach.  Indices rise, so that only a
// logit above the bound can get past those that are there; all lanes that have one leave it by a ballot and a count of the lanes before them.  The first
// bound is what K of the lanes' maxima of two loads reach; past some 32 entries more than needed it is raised, by bisection over the values' order with a ballot and
// a count for each entry of a lane.  Where too many are equal, the lower indices stay.  (Kept in order in registers and inserted one by one, a chain of some
// hundred dependent instructions each, 20 alternatives of one row took 24 us, and of 1024 rows in bf16 129.  The first bound from all values of the load, 8 ballots and
// counts a step: 64 rows of 151936 14.1 us for 13.0)
//
// A workgroup of 4 waves has a row, or a share of one where there are few; shares leave sums and lists that k_logprobs_merge joins.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <type_traits>

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
// a logit's place among the others as one number: what is ahead is larger
__device__ __forceinline__ int64_t key_of(int o, int i) { return (int64_t)o << 32 | (uint32_t)~i; }
__device__ __forceinline__ int order_in(int64_t k) { return (int)(k >> 32); }
__device__ __forceinline__ int index_in(int64_t k) { return ~(int)k; }
constexpr int64_t kNoKey = INT64_MIN;   // kNone's

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
// an element by a scalar load (16 bits: of the 4 bytes that it lies in)
typedef const int __attribute__((address_space(4))) scalar_int;
template <int T>
__device__ __forceinline__ float lp_scalar(const void *p, int64_t i) {
  const uintptr_t at = (uintptr_t)p + i * (T == RT_F32 ? 4 : 2);
  const uint32_t w = *(const scalar_int *)(at & ~(uintptr_t)3);
  if constexpr (T == RT_F32) return __builtin_bit_cast(float, w);
  const uint16_t h = (uint16_t)(w >> (at & 2 ? 16 : 0));
  return T == RT_F16 ? half_bits_to_float(h) : bf16_to_f(h);
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
__device__ __forceinline__ void put_top(const LogprobArgs &a, int64_t row, int k, int64_t key, float m, float ls) {
  const int o = order_in(key);
  a.top_index[row * a.top + k] = o == kNone ? -1 : index_in(key);
  a.top_logp[row * a.top + k] = o == kNone ? __builtin_nanf("") : value_of(o) - ref(m) - ls;
}
__device__ __forceinline__ void put(const LogprobArgs &a, int64_t row, const LpSum &s, float ls, float xt, bool has) {
  if (a.logp) a.logp[row] = has ? xt - ref(s.m) - ls : __builtin_nanf("");
  if (a.rank) a.rank[row] = has ? s.ahead : -1;
  if (a.entropy) a.entropy[row] = ls - s.t / s.s;
}

constexpr int kLpKeep = 128;   // entries that a wave goes on with, at most
__device__ __forceinline__ void wave_sync() {   // what lanes left in LDS is there for the others of the wave
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
__device__ __forceinline__ int lanes_before(uint64_t m) { return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0)); }
// The lanes' M values each.  lo is raised towards hi as long as more than `most` of them, n, reach it and K do; K reach it at the start
template <int M>
__device__ __forceinline__ int raised(const int (&o)[M], int lo, int hi, int K, int most, int &n) {
  lo = __builtin_amdgcn_readfirstlane(lo); hi = __builtin_amdgcn_readfirstlane(hi);   // (the wave's: scalar arithmetic)
  int mid = hi;   // (what a single alternative needs)
  while (n > most && lo < hi) {
    int c = 0;
#pragma unroll
    for (int k = 0; k < M; k++) c += __popcll(__ballot(o[k] >= mid));
    if (c >= K) { lo = mid; n = c; }
    else hi = mid - 1;
    mid = lo + (int)(((uint32_t)hi - (uint32_t)lo + 1) >> 1);   // above lo, up to hi
  }
  return lo;
}
// the key that K to `most` (at least K) of the entries reach, kNoKey: none; their orders lie between lo, which K reach, and hi
template <int M>
__device__ __forceinline__ int64_t bound_of(const int64_t (&x)[M], int lo, int hi, int K, int most) {
  int n = 0, o[M];
#pragma unroll
  for (int k = 0; k < M; k++) { o[k] = order_in(x[k]); n += __popcll(__ballot(o[k] >= lo)); }
  lo = raised<M>(o, lo, hi, K, most, n);
  int low = 0;   // (of the key: every index)
  if (n > most) {   // too many are equal: their indices, without the sign that the order has
    int above = 0, t[M];
#pragma unroll
    for (int k = 0; k < M; k++) { above += __popcll(__ballot(o[k] > lo)); t[k] = o[k] == lo ? (int)x[k] : kNone; }
    n -= above;
    low = raised<M>(t, kNone + 1, -1, K - above, K - above, n);
  }
  return (int64_t)lo << 32 | (uint32_t)low;
}
// a wave's n <= 64 M entries cut down to K .. most; the order of the last, which was `lo`
template <int M>
__device__ __forceinline__ int cut(int64_t *buf, int &n, int lo, int K, int most, int lane) {
  int64_t x[M];
  int hi = kNone;
#pragma unroll
  for (int k = 0; k < M; k++) {
    x[k] = 64 * k + lane < n ? buf[64 * k + lane] : kNoKey;
    hi = max(hi, order_in(x[k]));
  }
  hi = order_of(wave_max(value_of(hi)));   // (NaN, which lanes without an entry have here, is no maximum)
  const int64_t b = bound_of<M>(x, max(lo, kNone + 1), hi, K, most);
  int left = 0;
#pragma unroll
  for (int k = 0; k < M; k++) {
    const bool here = x[k] >= b;   // (above kNoKey)
    const uint64_t m = __ballot(here);
    if (here) buf[left + lanes_before(m)] = x[k];
    left += __popcll(m);
  }
  n = left;
  wave_sync();
  return order_in(b);
}
// the number of n entries ahead of x
__device__ __forceinline__ int ahead_of(int64_t x, const int64_t *all, int n) {
  int k = 0;
#pragma unroll 8
  for (int j = 0; j < n; j++) k += all[j] > x;
  return k;
}
// the wave's lanes that have an x to add leave it among the workgroup's
__device__ __forceinline__ void add_to(int64_t *all, int *count, bool has, int64_t x, int lane) {
  const uint64_t m = __ballot(has);
  int at = 0;
  if (lane == 0 && m) at = atomicAdd(count, __popcll(m));
  at = __builtin_amdgcn_readfirstlane(at);
  if (has) all[at + lanes_before(m)] = x;
}

// TINY: vocabularies of less than a lane's load
template <int T, bool TOP, bool TINY = false>
__global__ __launch_bounds__(kLpWaves * 64) void k_logprobs(LogprobArgs a) {
  constexpr int VE = lp_elems<T>(), GE = 64 * VE, U = 2;   // elements of a lane's load, of a wave's; loads on their way (3 and 4: no faster, and longer code)
  __shared__ LpSum sums[kLpWaves];
  constexpr int CAP = kLpKeep + GE;
  __shared__ int64_t entries[TOP ? kLpWaves : 1][TOP ? CAP : 1], joint[TOP ? kLpWaves * kLpKeep : 1];
  __shared__ int count, kept, bounds[kLpWaves];
  const int64_t row = blockIdx.x / (uint32_t)a.splits;
  const int split = blockIdx.x - (int)row * a.splits;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int from = split * a.share, to = min(a.vocab, from + a.share);
  const int esize = T == RT_F32 ? 4 : 2;
  const uint8_t *x0 = (const uint8_t *)a.x + row * a.ld * esize;
  LpSum s{-INFINITY, 0.f, 0.f, 0};
  int64_t *buf = entries[TOP ? wave : 0];
  int held = 0, bound = kNone;   // entries, what the K-th of them reaches
  float last = 0.f;              // that, as a value
  bool first = true, soft = false;   // soft: the next load holds some that reach the bound
  // what a cut leaves, and from how many entries on there is one: a bound near the K-th lets few logits pass, a cut costs as much as some of them
  const int most = a.top + a.top / 4 + 2, full = min(most + 32, kLpKeep);
  if (threadIdx.x == 0) count = 0;
  // A lane's elements from `at` on: where the share ends before, the last ones of it, of which those before `at` don't count.  Every load is made, so that the
  // compiler can count those on their way
  auto start = [&](int at) { return TINY ? at : min(at, to - VE); };
  auto load = [&](int at) -> u32x4 {
    if constexpr (!TINY) return __builtin_nontemporal_load((const u32x4_any *)(x0 + (int64_t)start(at) * esize));   // (read once: 1023 x 128256 fp32 95 -> 85 us)
    u32x4 w = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < VE; i++) {
      if (at + i >= to) continue;
      if constexpr (T == RT_F32) w[i] = ((const uint32_t *)x0)[at + i];
      else w[i / 2] |= (uint32_t)((const uint16_t *)x0)[at + i] << 16 * (i & 1);
    }
    return w;
  };
  u32x4 w[U];
  constexpr int STEP = GE * kLpWaves;
  const int steps = (to - from + STEP - 1) / STEP, base = from + GE * wave;
#pragma unroll
  for (int u = 0; u < U; u++) w[u] = load(base + u * STEP + VE * lane);
  // the token and its logit through the scalar cache: in the vector loads' order they would be waited for one after the other
  const int token = a.tokens ? __builtin_amdgcn_readfirstlane(*(const scalar_int *)(uintptr_t)(a.tokens + row)) : -1;
  const bool has = token >= 0 && token < a.vocab;
  const float xt = has ? lp_scalar<T>(x0, token) : INFINITY;
  auto take = [&](u32x4 w, int base, auto may_be_first, u32x4 next) {   // a wave's elements base ..; next: those STEP further on, of the first
    const int from0 = base + VE * lane, at = start(from0);
    float x[VE], bm = -INFINITY;
#pragma unroll
    for (int i = 0; i < VE; i++) x[i] = lp_elem<T>(w, i);
    uint32_t counts = ~0u;
    if (base + GE > to) {
      counts = 0;
#pragma unroll
      for (int i = 0; i < VE; i++) {
        const bool c = (at + i >= from0) & (at + i < to);
        counts |= (uint32_t)c << i;
        x[i] = c ? x[i] : -INFINITY;
      }
    }
#pragma unroll
    for (int i = 0; i < VE; i++) bm = fmaxf(bm, x[i]);
    if (__any(bm > s.m + kLpRoom)) {   // (always while there is none)
      const float m = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, wave_max(bm))));
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
      for (int i = 0; i < VE; i++) s.ahead += __popcll(__ballot(x[i] >= xt));
    } else if (base > token) {
#pragma unroll
      for (int i = 0; i < VE; i++) s.ahead += __popcll(__ballot(x[i] > xt));
    } else {
#pragma unroll
      for (int i = 0; i < VE; i++) s.ahead += __popcll(__ballot((x[i] > xt) | ((x[i] == xt) & (at + i < token) & (int)(counts >> i & 1))));
    }
    if constexpr (TOP) {
      if (decltype(may_be_first)::value && first) {
        // K of 128 maxima reach the first bound, and few of the other logits: the lanes' of this load and the next one, or of the halves of a last load; 20 of 128 maxima of 8 some 22 of
        // 1024.  (Of the halves always: 5 of 64 x 151936 17.7 us for 17.0, 64 of them 27.6 for 26.0)
        first = false;
        float h[2] = {x[0], x[VE / 2]};
        if (base + STEP + GE <= to) {
          h[0] = bm;
          h[1] = lp_elem<T>(next, 0);
#pragma unroll
          for (int i = 1; i < VE; i++) h[1] = fmaxf(h[1], lp_elem<T>(next, i));
          soft = true;
        } else {
#pragma unroll
          for (int i = 1; i < VE / 2; i++) { h[0] = fmaxf(h[0], x[i]); h[1] = fmaxf(h[1], x[VE / 2 + i]); }
        }
        const int o[2] = {order_of(fmaxf(h[0], -INFINITY)), order_of(fmaxf(h[1], -INFINITY))};   // (of NaN alone)
        int n = 128;
        bound = raised<2>(o, order_of(-wave_max(-fminf(value_of(o[0]), value_of(o[1])))), order_of(wave_max(fmaxf(value_of(o[0]), value_of(o[1])))), a.top, most, n);
        if (bound == order_of(-INFINITY)) {   // what a mask leaves, or a load with few elements: these too, but NaN, which no bound holds back
#pragma unroll
          for (int i = 0; i < VE; i++) {
            const bool here = (int)(x[i] == -INFINITY) & (int)(counts >> i & 1);
            const uint64_t m = __ballot(here);
            if (here) buf[held + lanes_before(m)] = key_of(order_of(x[i]), at + i);
            held += __popcll(m);
          }
        }
        // The value just below the bound: what passes reaches it (-0 has 0's place: below 0 is the largest negative one).  Not any lower, since a cut keeps what reaches the bound: of a
        // load full of logits one step below it none would be left, and the next load's at the bound would not pass
        last = value_of(max(bound - (bound ? 1 : 2), order_of(-INFINITY)));
      }
      if ((held <= full) & !__any(bm > last)) return;
#pragma unroll
      for (int i = 0; i < VE; i++) {
        const uint64_t m = __ballot(x[i] > last);
        if (m) {
          if (x[i] > last) buf[held + lanes_before(m)] = key_of(order_of(x[i]), at + i);
          held += __popcll(m);
        }
      }
      wave_sync();
      if (decltype(may_be_first)::value && soft) soft = false;   // (the next load's that are at the bound have to pass too)
      else last = value_of(bound);
      if (held > full) {
        bound = held > kLpKeep ? cut<CAP / 64>(buf, held, bound, a.top, most, lane) : cut<kLpKeep / 64>(buf, held, bound, a.top, most, lane);
        last = value_of(bound);
      }
    }
  };
  static_assert(U == 2, "the loop below");
  for (int k = 0; k < steps; k += U) {
    const u32x4 x0 = w[0];
    w[0] = load(base + (k + U) * STEP + VE * lane);
    take(x0, base + k * STEP, std::true_type(), w[1]);
    const u32x4 x1 = w[1];
    w[1] = load(base + (k + U + 1) * STEP + VE * lane);
    if (k + 1 < steps) take(x1, base + (k + 1) * STEP, std::false_type(), x1);
  }
  // lanes share the reference; then the waves
  s.s = wave_sum(s.s); s.t = wave_sum(s.t);
  if (lane == 0) sums[wave] = s;
  if constexpr (TOP) {
    wave_sync();
    if (held > most) bound = cut<kLpKeep / 64>(buf, held, bound, a.top, most, lane);
    if (lane == 0) bounds[wave] = bound;
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
    // what reaches every wave's bound is put together; an entry's place is the number of those before it
    int most = bounds[0];
#pragma unroll
    for (int i = 1; i < kLpWaves; i++) most = max(most, bounds[i]);
    for (int e = lane; e - lane < held; e += 64) {
      const int64_t x = e < held ? buf[e] : kNoKey;
      add_to(joint, &count, e < held && order_in(x) >= most, x, lane);
    }
    __syncthreads();
    int n = count;
    if (n > 2 * kLpTop) {   // (where four lists of many are left; count stays, so that all waves come here)
      if (wave == 0) {
        cut<kLpWaves * kLpKeep / 64>(joint, n, most, a.top, kLpTop + 16, lane);
        if (lane == 0) kept = n;
      }
      __syncthreads();
      n = kept;
    }
    auto put_at = [&](int k, int64_t x) {
      if (a.splits == 1) put_top(a, row, k, x, all.m, ls);
      else ((int64_t *)((LpSum *)a.work + a.rows * a.splits))[part * a.top + k] = x;
    };
    for (int e = threadIdx.x; e < max(n, a.top); e += kLpWaves * 64) {
      if (e >= n) { put_at(e, kNoKey); continue; }   // fewer than K (a share of a few logits)
      const int64_t x = joint[e];
      const int k = ahead_of(x, joint, n);
      if (k < a.top) put_at(k, x);
    }
  }
}

// The shares of a row: a workgroup joins their sums and picks the first K of their lists.  Bound by latency: all that can be is asked for before anything is waited
// for (20 of one row: 6.3 -> 5.4 us)
template <int T>
__global__ __launch_bounds__(256) void k_logprobs_merge(LogprobArgs a) {
  constexpr int kMost = kLpSplits * kLpTop, N = 8;   // (63 shares' 20 entries are 5 a thread; past 2048 entries they are loaded in their turn)
  __shared__ LpSum all;
  __shared__ int64_t firsts[kLpSplits + 2 * kLpTop], bound, joint[kMost];
  __shared__ int count;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, S = a.splits, K = a.top;
  const LpSum *sums = (const LpSum *)a.work + row * S;
  const int64_t *lists = (const int64_t *)((const LpSum *)a.work + a.rows * S) + row * S * K;
  // the first d of each list are K at least; what the K-th of them precedes is not among the first K.  (Of no more than K the last is some list's least, which many precede:
  // 64 of 16 x 32000 39 us for 17)
  const int d = K ? min((K + K / 2 + S - 1) / S, K) : 0, F = S * d;
  const int64_t mine = tid < F ? lists[tid / d * K + tid % d] : kNoKey;
  LpSum s = tid < S ? sums[tid] : LpSum{-INFINITY, 0.f, 0.f, 0};
  int64_t x[N];
#pragma unroll
  for (int i = 0; i < N; i++) x[i] = tid + 256 * i < S * K ? lists[tid + 256 * i] : kNoKey;
  const int token = a.tokens ? *(const scalar_int *)(uintptr_t)(a.tokens + row) : -1;
  const bool has = token >= 0 && token < a.vocab;
  const float xt = has ? lp_scalar<T>((const uint8_t *)a.x + row * a.ld * (T == RT_F32 ? 4 : 2), token) : 0.f;
  if (tid < F) firsts[tid] = mine;
  if (tid == 0) { count = 0; bound = kNoKey + 1; }
  if (tid < 64) {
#pragma unroll
    for (int d = 32; d; d >>= 1) join(s, LpSum{__shfl_xor(s.m, d), __shfl_xor(s.s, d), __shfl_xor(s.t, d), __shfl_xor(s.ahead, d)});
    if (tid == 0) all = s;
  }
  __syncthreads();
  const float ls = logf(all.s);
  if (tid == 0) put(a, row, all, ls, xt, has);
  if (!K) return;
  if (order_in(mine) != kNone && ahead_of(mine, firsts, F) == K - 1) bound = mine;
  __syncthreads();
  auto pick = [&](int64_t x) { add_to(joint, &count, order_in(x) != kNone && x >= bound, x, tid & 63); };
#pragma unroll
  for (int i = 0; i < N; i++)
    if (256 * i < S * K) pick(x[i]);
  for (int e = tid + 256 * N; e - tid < S * K; e += 256) pick(e < S * K ? lists[e] : kNoKey);
  __syncthreads();
  const int n = count;
  for (int e = tid; e < max(n, K); e += 256) {
    if (e >= n) { put_top(a, row, e, kNoKey, all.m, ls); continue; }   // fewer than K (a vocabulary of NaN)
    const int64_t x = joint[e];
    const int k = ahead_of(x, joint, n);
    if (k < K) put_top(a, row, k, x, all.m, ls);
  }
}
}  // namespace

size_t logprobs_plan(LogprobArgs &a) {
  // A workgroup's pass over its share is a chain of loads, of its waves' loads side by side (a unit) after one another: rows are shared out until there are four workgroups a CU.  Not
  // rows of few units, since the shares' joining costs as much as some of them (a row of 2000 to 5000 fp32 logits 8.8 us in shares, 5.6 to 7.1 without; 256 rows of 16000
  // 14.3 and 13.2, 64 of them 11.5 and 12.8), and not into shares of one unit where there are more than two a CU then (16 rows of 64000 12.4 us for 11.2)
  const int unit = kLpWaves * 64 * (a.type == RT_F32 ? 4 : 8);
  const int units = (a.vocab + unit - 1) / unit;
  const int least = a.rows * std::min(units, kLpSplits) > 512 ? 2 : 1;
  const int want = units <= 6 + a.rows / 24 ? 1 : (int)std::min<int64_t>(std::max<int64_t>(1024 / a.rows, 1), std::min((units + least - 1) / least, kLpSplits));
  const int each = (units + want - 1) / want;
  a.share = (int)std::min<int64_t>((int64_t)each * unit, INT_MAX);
  a.splits = (units + each - 1) / each;
  return a.splits == 1 ? 0 : (size_t)a.rows * a.splits * (sizeof(LpSum) + 8 * a.top);
}
hipError_t launch_logprobs(const LogprobArgs &a, hipStream_t st) {
  const dim3 grid((unsigned)(a.rows * a.splits)), thr(kLpWaves * 64);
#define QPH_LP(T)                                                                          \
  do {                                                                                     \
    if (a.vocab < lp_elems<T>()) hipLaunchKernelGGL((k_logprobs<T, true, true>), grid, thr, 0, st, a); \
    else if (a.top) hipLaunchKernelGGL((k_logprobs<T, true>), grid, thr, 0, st, a);             \
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
