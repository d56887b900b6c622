// Log probabilities of given tokens, the entropy and the most likely tokens of rows of logits, in one pass over them.
//
//   log p(t) = x_t - m - ln s,   s = sum_j e^(x_j - m),   H = ln s - (1/s) sum_j e^(x_j - m) (x_j - m),   m = max_j x_j;
//   the `top` largest logits (of equal ones the lowest index first) with their log p.
// Every thread keeps a sum and a weighted sum (fp32, base-2 exponents) of its elements, relative to a reference that all
// lanes of its warp share: the largest element of the warp's first groups, and a later one only where that is 4 more, so
// that weights go up to e^4 and few sums are rescaled; warps and CTAs are joined relative to the larger reference, and in
// the end to the row's maximum. A row is cut into groups of 512 consecutive bytes, one load of a warp each, whose largest
// value is kept as an ordered 32-bit key (one redux). The top tokens lie in the `top` groups that come first by (largest
// value, index): each of those holds an element that comes before all of any other group's. So they are found from the keys
// and read once more, whatever the logits look like. (Many equal logits, which the selection has to tell apart by their
// index, cost up to a quarter more over 1024 rows and up to 18 us over a few; warps that have seen nothing but -inf, or a
// reference beyond 1e4, take one element at a time: 1024 rows with five tokens left 100 us, far from 0 120 us.)
//
// Few rows are split over CTAs, each of which leaves its sums and its groups' keys in the workspace; the last of a row's
// CTAs to arrive adds them up in their order (results do not depend on timing). A NaN or +inf logit makes a row's
// probabilities NaN; a row of -inf alone has log p = -inf and entropy 0.
//
// What bounds it: many rows of bf16 the arithmetic (one exponential and 8.5 instructions an element; 1024 rows of 151936
// 54.4 us without top tokens, 5.7 TB/s, 62.2 with one and 75 with twenty: a row's two selections are 2 us each, in which
// its CTA loads nothing), of fp32 HBM (512 rows 49.5 us, 6.3 TB/s); rows that do not fill waves of CTAs the places left
// empty (300, 512 and 740 rows 31, 39 and 54 us with one top token, whose bytes take 14, 24 and 34); few rows the chain of
// round trips (one row 5.8 us without, 9.3 with one and 11.9 with twenty top tokens). Tried: the loads ahead in registers (4%
// longer: they leave no more than four CTAs an SM either way and cost moves), 128 threads a CTA (2% longer, a quarter
// with twenty top tokens), parts of all rows of a last wave (a quarter longer).
#include "internal.h"
#include "common.cuh"

namespace egpt {
namespace lgp {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxTop = 32;
constexpr int kMaxVocab = 1 << 20;
constexpr int kResident = 4;      // CTAs of an SM
constexpr int kAtOnce = 4, kRing = 2;  // groups that a warp loads at once, and how many times that is on its way
constexpr int kRingBytes = kRing * kAtOnce * 512 * kWarps;
constexpr int kSplitRows = 4096;  // arrival counters: more than the CTAs of a GPU
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr uint32_t kNegInf = 0x007fffffu, kInf = 0xff800000u;  // keys of the infinities; above kInf NaN, below kNegInf nothing

struct Params {
  const void *x;
  int64_t ldx;
  const int64_t *tokens;  // nullable
  int m, v, top;
  int whole, splits;  // rows of a CTA each; CTAs of each of the others
  float *logp, *entropy, *top_logp;
  int64_t *top_ids;
  unsigned *cnt;   // arrivals of a split row, zero between calls
  float4 *parts;   // [split rows][splits] maximum, sum, weighted sum, largest key
  uint32_t *keys;  // [split rows][most groups]
  int key_stride;
};

// Keys in the order of the values: -inf < ... < +inf < NaN (0x7fffffff, as a sum gives it), zeros alike.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(__fadd_rn(x, 0.f));
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  if (key == 0xffffffffu) return NAN;
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// A row in 16-byte chunks from the aligned address at or before its start: E elements each, chunk c from element c E - off.
template <typename T>
struct Row {
  static constexpr int E = 16 / (int)sizeof(T);
  const T *x;
  int v, off, groups;
  __device__ Row(const Params &p, int row) {
    x = (const T *)p.x + row * p.ldx;
    v = p.v, off = (int)(((uintptr_t)x & 15u) / sizeof(T));
    groups = (v + off + 32 * E - 1) / (32 * E);
  }
  static __device__ float widen(float t) { return t; }
  static __device__ float widen(uint16_t t) { return bf16_bits_to_f32(t); }
  // Elements of chunk c; outside the row -inf. -> whether any is inside
  __device__ __forceinline__ bool load(int c, float (&y)[E]) const {
    const int i0 = c * E - off;
    if (i0 >= 0 && i0 + E <= v) {
      const uint4 a = *(const uint4 *)(x + i0);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int e = 0; e < E; ++e)
        y[e] = E == 4 ? __uint_as_float(w[e % 4]) : (e % 2 ? bf16_hi(w[(e / 2) % 4]) : bf16_lo(w[(e / 2) % 4]));
      return true;
    }
    bool any = false;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool in = i0 + e >= 0 && i0 + e < v;
      y[e] = in ? widen(x[i0 + e]) : -INFINITY;
      any |= in;
    }
    return any;
  }
};

struct Sums {
  float m, s, w;  // reference (-inf: none yet), sum of 2^exponent(x, m), the same times its exponent
};
// (x - m) log2 e. For m up to 1e4 as x log2 e less m log2 e, rounded: what that is off (residual(m), 5e-4 at most) is the same for
// all x and cancels in the entropy; log p and a change of m put it back. Beyond, where it grows and x log2 e can overflow, as the
// difference times log2 e.
__device__ __forceinline__ bool plain_range(float m) { return fabsf(m) <= 1e4f; }
__device__ __forceinline__ float exponent(float x, float m) {
  return plain_range(m) ? fmaf(x, kLog2e, -__fmul_rn(m, kLog2e)) : (x - m) * kLog2e;
}
__device__ __forceinline__ float residual(float m) {  // m log2 e, rounded, less m log2 e
  return plain_range(m) ? -fmaf(m, kLog2e, -__fmul_rn(m, kLog2e)) : 0.f;
}
__device__ __forceinline__ float log_prob(float x, float m, float log_s) {
  return x - m - fmaf(residual(m), kLn2, log_s);
}
// The exponent that takes sums from one reference to another, from <= to. (2^-1000 is 0, and 0 times it too; of two -inf, whose
// difference is NaN, the sums are 0.)
__device__ __forceinline__ float moved(float from, float to) {
  return fmaxf(fmaf(from - to, kLog2e, residual(from) - residual(to)), -1000.f);
}
__device__ __forceinline__ void rescale(Sums &a, float m) {  // m >= a.m
  const float t = moved(a.m, m), f = apf::ex2(t);
  a.w = f * fmaf(t, a.s, a.w), a.s *= f, a.m = m;
}
// The same for (a, b) and (b, a), to the bit. One exponential: with both sums moved to the maximum one row takes 1.9 us longer.
__device__ __forceinline__ void join(Sums &a, const Sums &b) {
  const bool less = a.m < b.m;
  const Sums lo = less ? a : b, hi = less ? b : a;
  const float t = moved(lo.m, hi.m), f = apf::ex2(t);
  a.s = fmaf(f, lo.s, hi.s), a.w = fmaf(f, fmaf(t, lo.s, lo.w), hi.w), a.m = hi.m;
}
// The sums of N neighbouring lanes in all of them.
template <int N>
__device__ __forceinline__ void join_lanes(Sums &a) {
#pragma unroll
  for (int o = 1; o < N; o <<= 1) {
    Sums b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
    b.w = __shfl_xor_sync(0xffffffffu, a.w, o);
    join(a, b);
  }
}
template <int E>
__device__ __forceinline__ void take(Sums &a, const float (&y)[E], float largest) {
  if (largest > a.m) rescale(a, largest);
  const float m = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float t = fmaxf(exponent(y[e], m), -1000.f);
    const float f = apf::ex2(t);
    a.s += f, a.w = fmaf(f, t, a.w);
  }
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// The largest element of a whole chunk (16 bytes), NaN if there is one.
template <int E>
__device__ __forceinline__ float largest_of(uint4 c) {
  if (E == 8) {
    const uint32_t mx = max2_nan(max2_nan(c.x, c.y), max2_nan(c.z, c.w));
    return max_nan(bf16_lo(mx), bf16_hi(mx));
  }
  return max_nan(max_nan(__uint_as_float(c.x), __uint_as_float(c.y)), max_nan(__uint_as_float(c.z), __uint_as_float(c.w)));
}
// Its elements into sums kept in pairs, relative to m (of the plain range).
template <int E>
__device__ __forceinline__ void take2(uint64_t &s, uint64_t &w, float m, uint4 c) {
  const uint32_t v[4] = {c.x, c.y, c.z, c.w};
  const uint64_t less = f2_pack(-__fmul_rn(m, kLog2e), -__fmul_rn(m, kLog2e)), log2e = f2_pack(kLog2e, kLog2e);
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    // no lower than -1e37 (0xfcf0, as bf16 -9.97e36), whose weight is 0 and exponent finite: -inf would give 0 times infinity
    uint64_t x;
    if (E == 8) {
      const uint32_t t = max2(v[i % 4], 0xfcf0fcf0u);
      x = f2_pack(bf16_lo(t), bf16_hi(t));
    } else {
      x = f2_pack(fmaxf(__uint_as_float(v[(2 * i) % 4]), -1e37f), fmaxf(__uint_as_float(v[(2 * i + 1) % 4]), -1e37f));
    }
    const uint64_t t = f2_fma(x, log2e, less);
    const float2 th = f2_unpack(t);
    const uint64_t f = f2_pack(apf::ex2(th.x), apf::ex2(th.y));
    s = f2_add(s, f), w = f2_fma(f, t, w);
  }
}

constexpr int kMore = 8;        // threads more than asked for that may have a key which passes the selection's first step
constexpr int kKeysEach = 33;   // keys of a thread at most: 2^20 fp32 logits off the 16-byte grid are 8193 groups
struct Smem {
  Sums sums[kWarps];
  uint32_t largest[kWarps];
  uint2 cand[(kMaxTop + kMore) * kKeysEach];  // keys that may be among the first
  uint2 best[kMaxTop];    // the first ones in order: value, ~index
  uint2 range[kWarps];
  int group[kMaxTop];
  int count, last;
  float m, log_s;
  uint32_t keys[1];  // the row's groups (where no other CTA has some), then the elements of the selected ones
};
constexpr int kMostGroups = kMaxVocab / 128 + 1;  // of fp32 logits, in a row off the 16-byte grid
constexpr size_t kMostSmem = kRingBytes + sizeof(Smem) + 4 * kMostGroups;
static_assert(kMostGroups >= kMaxTop * 256 && kMostGroups <= kKeysEach * kThreads && kMostSmem <= 100 * 1024, "sizes");
__device__ __forceinline__ bool before(uint2 a, uint2 b) { return a.x > b.x || (a.x == b.x && a.y > b.y); }

// The `top` first of the keys get(0 .. n - 1) (value, ~index: all different), in order, into sm.best (value 0: fewer than top), n <=
// kKeysEach kThreads. A threshold is found by bisection that the first keys of `top` to top + kMore threads reach, so at most
// kKeysEach keys of each of those do, mostly a few more than top; they are ranked by counting. Every thread calls it.
template <typename F>
__device__ __forceinline__ void select(Smem &sm, int n, int top, F get) {
  constexpr int kHeld = 4;  // keys of a thread in registers
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  uint2 held[kHeld], first = make_uint2(0u, 0u);
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    held[i] = make_uint2(0u, 0u);
    if (t + i * kThreads < n) held[i] = get(t + i * kThreads);
  }
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (before(held[i], first)) first = held[i];
  for (int i = t + kHeld * kThreads; i < n; i += kThreads) {
    const uint2 k = get(i);
    if (before(k, first)) first = k;
  }
  // the least and the largest value of the threads' first keys, between which the threshold's is
  const uint32_t warp_lo = __reduce_min_sync(0xffffffffu, first.x), warp_hi = __reduce_max_sync(0xffffffffu, first.x);
  if (lane == 0) sm.range[warp] = make_uint2(warp_lo, warp_hi);
  if (t == 0) sm.count = 0;
  if (t < kMaxTop) sm.best[t] = make_uint2(0u, 0u);
  uint2 lo = make_uint2(0u, 1u);  // every key reaches it
  if (__syncthreads_count(first.x != 0u) > top + kMore) {
    uint2 hi = make_uint2(0u, 0xffffffffu);
    lo.x = 0xffffffffu;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) lo.x = min(lo.x, sm.range[w].x), hi.x = max(hi.x, sm.range[w].y);
    lo.y = 0u;  // (an index of 0 is no key's; a value of 0 none's either, so that all of them count as reaching it)
    for (;;) {
      // halfway in the values, then in the indices
      uint2 mid = make_uint2(lo.x + (hi.x - lo.x) / 2, 0u);
      if (hi.x - lo.x <= 1u) mid = hi.x == lo.x ? make_uint2(lo.x, lo.y + (hi.y - lo.y) / 2) : make_uint2(hi.x, 0u);
      if (hi.x == lo.x && mid.y == lo.y) mid.y = hi.y;
      const int reach = __syncthreads_count(first.x != 0u && !before(mid, first));
      if (reach >= top) lo = mid;
      else hi = make_uint2(mid.y ? mid.x : mid.x - 1u, mid.y - 1u);
      if (reach >= top && reach <= top + kMore) break;
    }
  }
  auto offer = [&](uint2 k) {
    if (k.x != 0u && !before(lo, k)) sm.cand[atomicAdd(&sm.count, 1)] = k;
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i) offer(held[i]);
  for (int i = t + kHeld * kThreads; i < n; i += kThreads) offer(get(i));
  __syncthreads();
  const int count = sm.count;
  for (int i = t; i < count; i += kThreads) {
    const uint2 k = sm.cand[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < count; ++j) rank += before(sm.cand[j], k);
    if (rank < top) sm.best[rank] = k;
  }
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads, kResident) logprobs_kernel(const Params p) {
  constexpr int E = Row<T>::E, U = kAtOnce;
  extern __shared__ __align__(16) uint8_t smem_raw[];  // the warps' rings, then Smem
  Smem &sm = *(Smem *)(smem_raw + kRingBytes);
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cut = (int)blockIdx.x - p.whole;
  // this CTA's row, its part and the row's parts
  const int at = cut < 0 ? 0 : cut / p.splits, row = cut < 0 ? (int)blockIdx.x : p.whole + at;
  const int split = cut < 0 ? 0 : cut - at * p.splits, splits = cut < 0 ? 1 : p.splits;
  float x_token = 0.f;  // asked for early: the last of the row's CTAs needs it
  int64_t token = -1;
  if (threadIdx.x == 0 && p.tokens) token = p.tokens[row];
  const Row<T> r(p, row);
  const int g0 = (int)((int64_t)r.groups * split / splits), g1 = (int)((int64_t)r.groups * (split + 1) / splits);
  if (token >= 0 && token < p.v) x_token = Row<T>::widen(r.x[token]);
  uint32_t *keys = splits == 1 ? sm.keys : p.keys + (int64_t)at * p.key_stride;
  uint32_t largest = 0u;
  auto note = [&](int g, uint32_t key) {
    key = __reduce_max_sync(0xffffffffu, key);
    if (p.top && lane == 0) keys[g] = key;
    return key;
  };
  // Groups that lie inside the row whole, U loads on their way at once.
  const int whole0 = max(g0, r.off ? 1 : 0), whole1 = min(g1, (r.v + r.off) / (32 * E));
  Sums a = {-INFINITY, 0.f, 0.f};
  uint64_t s2 = 0u, w2 = 0u;
  auto add = [&](int g, const auto &c) {  // groups g, g + kWarps, ...
    constexpr int N = (int)(sizeof(c) / sizeof(c[0]));
    uint32_t most = 0u;
#pragma unroll
    for (int u = 0; u < N; ++u) most = max(most, note(g + u * kWarps, key_of(largest_of<E>(c[u]))));
    largest = max(largest, most);
    const float mx = value_of(most);  // the same in all lanes, as a.m is
    if (!(mx <= a.m + 4.f) || !plain_range(a.m)) {
      const float2 s = f2_unpack(s2), w = f2_unpack(w2);
      a.s += s.x + s.y, a.w += w.x + w.y, s2 = w2 = 0u;
      if (mx > a.m) rescale(a, mx);
      if (!plain_range(a.m)) {  // nothing yet, or far from 0: one element at a time
#pragma unroll 1
        for (int u = 0; u < N; ++u) {
          float y[E];
          r.load((g + u * kWarps) * 32 + lane, y);
          take<E>(a, y, -INFINITY);
        }
        return;
      }
    }
#pragma unroll
    for (int u = 0; u < N; ++u) take2<E>(s2, w2, a.m, c[u]);
  };
  int g = whole0 + warp;
  constexpr int kStep = U * kWarps, kSpan = kStep - kWarps;
  if (g + kSpan < whole1) {  // the next ones on their way while these are added (in shared memory: registers are full)
    uint4 *mine = (uint4 *)smem_raw + warp * (kRing * U * 32) + lane;  // a lane reads what it has copied itself
    int fetch = g;
    auto copy = [&](int slot) {
      if (fetch + kSpan < whole1)
#pragma unroll
        for (int u = 0; u < U; ++u)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(mine + (slot * U + u) * 32)),
                       "l"((const uint4 *)(r.x - r.off) + (fetch + u * kWarps) * 32 + lane)
                       : "memory");
      asm volatile("cp.async.commit_group;" ::: "memory");
      fetch += kStep;
    };
#pragma unroll
    for (int i = 0; i < kRing; ++i) copy(i);
    for (int slot = 0; g + kSpan < whole1; g += kStep) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 1) : "memory");
      uint4 c[U];
#pragma unroll
      for (int u = 0; u < U; ++u) c[u] = mine[(slot * U + u) * 32];
      copy(slot);
      slot = slot + 1 == kRing ? 0 : slot + 1;
      add(g, c);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  for (; g < whole1; g += kWarps) {
    const uint4 c[1] = {__ldg((const uint4 *)(r.x - r.off) + g * 32 + lane)};
    add(g, c);
  }
  const float2 s = f2_unpack(s2), w = f2_unpack(w2);
  a.s += s.x + s.y, a.w += w.x + w.y;
  // the first and the last one otherwise
  const int ends[2] = {r.off ? 0 : -1, r.groups - 1 >= (r.v + r.off) / (32 * E) && (r.groups > 1 || !r.off) ? r.groups - 1 : -1};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (warp != i || ends[i] < g0 || ends[i] >= g1) continue;
    float y[E], mx = -INFINITY;
    const bool any = r.load(ends[i] * 32 + lane, y);
#pragma unroll
    for (int e = 0; e < E; ++e) mx = max_nan(mx, y[e]);
    if (any) take<E>(a, y, mx);
    largest = max(largest, note(ends[i], any ? key_of(mx) : 0u));
  }
  join_lanes<32>(a);
  if (lane == 0) sm.sums[warp] = a, sm.largest[warp] = largest;
  __syncthreads();
  if (warp == 0) {
    a = lane < kWarps ? sm.sums[lane] : Sums{-INFINITY, 0.f, 0.f};
    join_lanes<kWarps>(a);
    largest = __reduce_max_sync(0xffffffffu, lane < kWarps ? sm.largest[lane] : 0u);
  }
  if (splits > 1) {
    if (threadIdx.x == 0) {
      p.parts[(int64_t)at * splits + split] = make_float4(a.m, a.s, a.w, __uint_as_float(largest));
      __threadfence();  // the record and (by the barrier) the keys
      const bool last = atomicAdd(p.cnt + at, 1u) == (unsigned)splits - 1u;
      if (last) {
        __threadfence();
        p.cnt[at] = 0u;
      }
      sm.last = last;
    }
    __syncthreads();
    if (!sm.last) return;
    if (p.top)  // (a thread reads its own ones again)
      for (int i = threadIdx.x; i < r.groups; i += kThreads) sm.keys[i] = __ldcg(keys + i);
    if (warp == 0) {  // the row's parts: a lane takes every 32nd, then the lanes'
      a = {-INFINITY, 0.f, 0.f}, largest = 0u;
      for (int i = lane; i < splits; i += 32) {
        const float4 t = __ldcg(p.parts + (int64_t)at * splits + i);
        join(a, Sums{t.x, t.y, t.z});
        largest = max(largest, __float_as_uint(t.w));
      }
      join_lanes<32>(a);
      largest = __reduce_max_sync(0xffffffffu, largest);
    }
  }
  if (warp == 0) {
    const bool none = largest == kNegInf, bad = largest >= kInf;
    // of a row of -inf alone, log p is that too
    if (!none && !bad) rescale(a, value_of(largest));
    const float m = bad ? NAN : (none ? 0.f : a.m), log_s = none ? 0.f : log2f(a.s) * kLn2;
    if (lane == 0) {
      sm.m = m, sm.log_s = log_s;
      p.entropy[row] = bad ? NAN : (none ? 0.f : fmaxf(0.f, log_s - a.w / a.s * kLn2));
      if (p.tokens) {
        float lp = 0.f;  // -1: no token
        if (token >= 0 && token < p.v) lp = log_prob(x_token, m, log_s);
        else if (token != -1) set_device_error(EGPT_ERR_SHAPE), lp = NAN;
        p.logp[row] = lp;
      }
    }
  }
  if (!p.top) return;
  // ---- the groups with the top tokens, then the first of their elements
  select(sm, r.groups, p.top, [&](int i) { return make_uint2(sm.keys[i], ~(uint32_t)i); });
  const int groups = min(p.top, r.groups);
  if (threadIdx.x < groups) sm.group[threadIdx.x] = (int)~sm.best[threadIdx.x].y;
  uint32_t *elems = sm.keys;  // the groups' own keys are done with
  for (int j = warp; j < groups; j += kWarps) {
    const int c = (int)~sm.best[j].y * 32 + lane;
    float y[E];
    r.load(c, y);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = c * E - r.off + e;
      elems[(j * 32 + lane) * E + e] = i >= 0 && i < r.v ? key_of(y[e]) : 0u;
    }
  }
  __syncthreads();
  select(sm, groups * 32 * E, p.top, [&](int i) {
    return make_uint2(elems[i], ~(uint32_t)(sm.group[i / (32 * E)] * 32 * E + i % (32 * E) - r.off));
  });
  if (threadIdx.x < p.top) {
    const uint2 k = sm.best[threadIdx.x];
    p.top_ids[(int64_t)row * p.top + threadIdx.x] = (int64_t)(~k.y);
    p.top_logp[(int64_t)row * p.top + threadIdx.x] = log_prob(value_of(k.x), sm.m, sm.log_s);
  }
}

static int group_elems(bool f32) { return 512 / (f32 ? 4 : 2); }
// Groups of a row at most (a row may start inside a 16-byte chunk).
static int most_groups(int64_t v, bool f32) { return (int)((v + 16 / (f32 ? 4 : 2) - 1 + group_elems(f32) - 1) / group_elems(f32)); }
// The rows in full waves of CTAs take one each. Those behind them are split where two parts or more of each fit into one wave, with
// 16 groups (two loads a warp) a part at least. More parts than that cost more than the places they fill: a part ends
// with a fence, an arrival and an idle stream (1024 rows of 151936 bf16 logits, 432 of them behind a wave of 592, take 16%
// longer in quarters than whole).
static void cut(int64_t m, int64_t v, bool f32, int &whole, int &splits) {
  const int wave = std::min(num_sms() * kResident, kSplitRows), rest = (int)(m % wave);
  splits = rest ? std::max(1, std::min(wave / rest, most_groups(v, f32) / 16)) : 1;
  whole = splits > 1 ? (int)m - rest : (int)m;
}
static size_t ws_bytes(int64_t m, int64_t v, bool f32) {
  int whole, splits;
  cut(m, v, f32, whole, splits);
  if (splits == 1) return 0;
  return kSplitRows * sizeof(unsigned) +
         (size_t)(m - whole) * (splits * sizeof(float4) + (most_groups(v, f32) + 3) / 4 * 4 * sizeof(uint32_t));
}

}  // namespace lgp
}  // namespace egpt

using namespace egpt;

extern "C" size_t egpt_token_logprobs_ws_bytes(int64_t m, int64_t v) {
  if (m < 1 || v < 1 || v > lgp::kMaxVocab) return 0;
  return std::max(lgp::ws_bytes(m, v, false), lgp::ws_bytes(m, v, true));
}

extern "C" size_t egpt_token_logprobs_max_ws_bytes(int64_t m, int64_t v) {
  size_t most = 0;  // the rows behind the last full wave decide: m of less than two waves have all there are
  for (int64_t rows = 1; rows <= std::min<int64_t>(m, 2 * lgp::kSplitRows); ++rows)
    most = std::max(most, egpt_token_logprobs_ws_bytes(rows, v));
  return most;
}

extern "C" int egpt_token_logprobs(float *logp, float *entropy, int64_t *top_ids, float *top_logp, const void *logits,
                                   int64_t ldx, int dtype, int64_t m, int64_t v, const int64_t *tokens, int top, void *ws,
                                   size_t ws_bytes, unsigned flags, void *stream) {
  clear_error();
  if (!entropy || !logits || (tokens && !logp) || (top > 0 && (!top_ids || !top_logp)))
    return set_error(EGPT_ERR_ARG, "token_logprobs: null pointer");
  if (dtype != EGPT_BF16 && dtype != EGPT_F32) return set_error(EGPT_ERR_DTYPE, "token_logprobs: logits are bf16 or fp32");
  const bool f32 = dtype == EGPT_F32;
  if (m < 1 || m > 65535 || v < 1 || v > lgp::kMaxVocab || ldx < v)
    return set_error(EGPT_ERR_SHAPE, "token_logprobs: bad rows (1 to 65535), vocabulary (1 to 2^20) or leading dimension");
  if (top < 0 || top > lgp::kMaxTop || top > v)
    return set_error(EGPT_ERR_SHAPE, "token_logprobs: top must be in [0, %d] and no more than the vocabulary", lgp::kMaxTop);
  if ((uintptr_t)logits % (f32 ? 4 : 2)) return set_error(EGPT_ERR_ALIGN, "token_logprobs: logits must be aligned to their type");
  lgp::Params p{};
  lgp::cut(m, v, f32, p.whole, p.splits);
  if (p.splits > 1) {
    if (!ws || ws_bytes < lgp::ws_bytes(m, v, f32)) return set_error(EGPT_ERR_WORKSPACE, "token_logprobs: workspace too small");
    if ((uintptr_t)ws % 16) return set_error(EGPT_ERR_ALIGN, "token_logprobs: workspace must be 16-byte aligned");
  }
  p.x = logits, p.ldx = ldx, p.tokens = tokens, p.m = (int)m, p.v = (int)v, p.top = top;
  p.logp = logp, p.entropy = entropy, p.top_logp = top_logp, p.top_ids = top_ids;
  p.cnt = (unsigned *)ws, p.parts = (float4 *)((char *)ws + lgp::kSplitRows * sizeof(unsigned));
  p.keys = (uint32_t *)(p.parts + (m - p.whole) * p.splits), p.key_stride = (lgp::most_groups(v, f32) + 3) / 4 * 4;
  const int words = std::max(lgp::most_groups(v, f32), top * lgp::group_elems(f32));
  const size_t smem = lgp::kRingBytes + sizeof(lgp::Smem) + (top ? words * sizeof(uint32_t) : 0);
  const void *fn = f32 ? (const void *)lgp::logprobs_kernel<float> : (const void *)lgp::logprobs_kernel<uint16_t>;
  static int configured[2][64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[f32][dev]) {
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)lgp::kMostSmem);
    if (e != cudaSuccess) return check_launch(e, "token_logprobs_kernel");
    if (dev >= 0 && dev < 64) configured[f32][dev] = 1;
  }
  return check_launch(launch_kernel(fn, dim3((unsigned)(p.whole + (m - p.whole) * p.splits)), dim3(lgp::kThreads), smem, (cudaStream_t)stream,
                                    (flags & EGPT_FLAG_PDL) != 0, p),
                      "token_logprobs_kernel");
}
