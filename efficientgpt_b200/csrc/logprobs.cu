// Log probabilities of given tokens, the entropy and the most likely tokens of rows of logits, in one pass over them.
//
//   log p(t) = x_t - m - ln s,   s = sum_j e^(x_j - m),   H = ln s - (1/s) sum_j e^(x_j - m) (x_j - m),   m = max_j x_j;
//   the `top` largest logits (of equal ones the lowest index first) with their log p.
// Every thread keeps a running maximum, sum and weighted sum (fp32, base-2 exponents) of its elements, rescaled when the
// maximum moves. A row is cut into groups of 512 consecutive bytes, one load of a warp each, whose largest value is kept
// as an ordered 32-bit key (one redux). The top tokens lie in the `top` groups that come first by (largest value, index):
// each of those holds an element that comes before all of any other group's. So they are found from the keys and
// read once more, whatever the logits look like: sorted, constant or mostly masked ones cost no more than others.
//
// Few rows are split over CTAs, each of which leaves its sums and its groups' keys in the workspace; the last of a row's
// CTAs to arrive adds them up in their order (results do not depend on timing). A NaN or +inf logit makes a row's
// probabilities NaN; a row of -inf alone has log p = -inf and entropy 0.
#include "internal.h"
#include "common.cuh"

namespace egpt {
namespace lgp {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxTop = 32;
constexpr int kMaxVocab = 1 << 20;
constexpr int kSplitRows = 512;   // rows that may be split, and arrival counters
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr uint32_t kNegInf = 0x007fffffu, kInf = 0xff800000u;  // keys of the infinities; above kInf NaN, below kNegInf nothing

struct Params {
  const void *x;
  int64_t ldx;
  const int64_t *tokens;  // nullable
  int m, v, top, splits;
  float *logp, *entropy, *top_logp;
  int64_t *top_ids;
  unsigned *cnt;   // arrivals of a split row, zero between calls
  float4 *parts;   // [m][splits] maximum, sum, weighted sum, largest key
  uint32_t *keys;  // [m][most groups]
  int key_stride;
};

// Keys in the order of the values: -inf < ... < +inf < NaN, zeros alike.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(__fadd_rn(x, 0.f));
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
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
  float m, s, w;  // maximum (-inf: none yet), sum of 2^((x - m) log2 e), the same times its exponent
};
__device__ __forceinline__ void rescale(Sums &a, float m) {  // m >= a.m
  const float t = fmaxf((a.m - m) * kLog2e, -1000.f), f = apf::ex2(t);  // (2^-1000 is 0, and 0 times it too)
  a.w = f * fmaf(t, a.s, a.w), a.s *= f, a.m = m;
}
__device__ __forceinline__ void join(Sums &a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return;
  rescale(a, m), rescale(b, m);
  a.s += b.s, a.w += b.w;
}
// The sums of N neighbouring lanes in all of them, the lower lane's first.
template <int N>
__device__ __forceinline__ void join_lanes(Sums &a) {
#pragma unroll
  for (int o = 1; o < N; o <<= 1) {
    Sums b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
    b.w = __shfl_xor_sync(0xffffffffu, a.w, o);
    if (threadIdx.x & o) {
      const Sums t = a;
      a = b, b = t;
    }
    join(a, b);
  }
}
template <int E>
__device__ __forceinline__ void take(Sums &a, const float (&y)[E], float largest) {
  if (largest > a.m) rescale(a, largest);
  const float m = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float t = fmaxf((y[e] - m) * kLog2e, -1000.f);
    const float f = apf::ex2(t);
    a.s += f, a.w = fmaf(f, t, a.w);
  }
}

// Two fp32 operations an instruction.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 halves(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
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
// A whole chunk (16 bytes) into sums kept in pairs; -> its largest value, NaN if there is one.
struct Sums2 {
  float m;
  uint64_t s, w;
};
template <int E>
__device__ __forceinline__ float take2(Sums2 &a, uint4 c) {
  uint32_t v[4] = {c.x, c.y, c.z, c.w};
  float largest;
  if (E == 8) {
    const uint32_t mx = max2_nan(max2_nan(v[0], v[1]), max2_nan(v[2], v[3]));
    largest = max_nan(bf16_lo(mx), bf16_hi(mx));
  } else {
    largest = max_nan(max_nan(__uint_as_float(v[0]), __uint_as_float(v[1])),
                      max_nan(__uint_as_float(v[2]), __uint_as_float(v[3])));
  }
  if (largest > a.m || !(fabsf(a.m) <= 1e36f)) {
    const float2 s = halves(a.s), w = halves(a.w);
    Sums t = {a.m, s.x + s.y, w.x + w.y};
    if (largest > t.m) rescale(t, largest);
    a.m = t.m;
    if (!(fabsf(t.m) <= 1e36f)) {  // nothing yet, or differences that can overflow: one at a time
      float y[E];
#pragma unroll
      for (int e = 0; e < E; ++e)
        y[e] = E == 4 ? __uint_as_float(v[e % 4]) : (e % 2 ? bf16_hi(v[(e / 2) % 4]) : bf16_lo(v[(e / 2) % 4]));
      take<E>(t, y, largest);
      a.s = pair(t.s, 0.f), a.w = pair(t.w, 0.f);
      return largest;
    }
    a.s = pair(t.s, 0.f), a.w = pair(t.w, 0.f);
  }
  const uint64_t less = pair(-a.m, -a.m), log2e = pair(kLog2e, kLog2e);
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    // no lower than -1e37 (0xfcf0, as bf16 -9.97e36), whose weight is 0 and exponent finite: -inf would give 0 times infinity
    uint64_t x;
    if (E == 8) {
      const uint32_t t = max2(v[i % 4], 0xfcf0fcf0u);
      x = pair(bf16_lo(t), bf16_hi(t));
    } else {
      x = pair(fmaxf(__uint_as_float(v[(2 * i) % 4]), -1e37f), fmaxf(__uint_as_float(v[(2 * i + 1) % 4]), -1e37f));
    }
    const uint64_t t = mul2(add2(x, less), log2e);
    const float2 th = halves(t);
    const uint64_t f = pair(apf::ex2(th.x), apf::ex2(th.y));
    a.s = add2(a.s, f), a.w = fma2(f, t, a.w);
  }
  return largest;
}

constexpr int kFew = 48;        // how many threads at most have a key that passes the selection's first step
constexpr int kKeysEach = 33;   // keys of a thread at most: 2^20 fp32 logits off the 16-byte grid are 8193 groups
struct Smem {
  Sums sums[kWarps];
  uint32_t largest[kWarps];
  uint2 cand[kFew * kKeysEach];  // keys that may be among the first
  uint2 best[kMaxTop];    // the first ones in order: value, ~index
  int group[kMaxTop];
  int count, last;
  float m, log_s;
  uint32_t keys[1];  // the row's groups (where no other CTA has some), then the elements of the selected ones
};
__device__ __forceinline__ bool before(uint2 a, uint2 b) { return a.x > b.x || (a.x == b.x && a.y > b.y); }

// The `top` first of the keys get(0 .. n - 1) (value, ~index: all different), in order, into sm.best (value 0: fewer than top), n <=
// kKeysEach kThreads. A threshold is found by bisection that `top` to kFew threads' first keys reach, so at most kKeysEach
// kFew keys do, mostly a few more than top; those are ranked by counting. Every thread calls it.
template <typename F>
__device__ __forceinline__ void select(Smem &sm, int n, int top, F get) {
  const int t = threadIdx.x;
  uint2 first = make_uint2(0u, 0u);
  for (int i = t; i < n; i += kThreads) {
    const uint2 k = get(i);
    if (before(k, first)) first = k;
  }
  if (t == 0) sm.count = 0;
  if (t < kMaxTop) sm.best[t] = make_uint2(0u, 0u);
  uint2 lo = make_uint2(0u, 1u);  // every key reaches it
  if (__syncthreads_count(before(first, make_uint2(0u, 0u))) > kFew) {
    uint2 hi = make_uint2(0xffffffffu, 0xffffffffu);
    for (;;) {
      // halfway in the values, then in the indices
      uint2 mid = make_uint2(lo.x + (hi.x - lo.x) / 2, 0u);
      if (hi.x - lo.x <= 1u) mid = hi.x == lo.x ? make_uint2(lo.x, lo.y + (hi.y - lo.y) / 2) : make_uint2(hi.x, 0u);
      if (hi.x == lo.x && mid.y == lo.y) mid.y = hi.y;
      const int reach = __syncthreads_count(!before(mid, first));
      if (reach >= top) lo = mid;
      else hi = make_uint2(mid.y ? mid.x : mid.x - 1u, mid.y - 1u);
      if (reach >= top && reach <= kFew) break;
    }
  }
  for (int i = t; i < n; i += kThreads) {
    const uint2 k = get(i);
    if (k.x != 0u && !before(lo, k)) sm.cand[atomicAdd(&sm.count, 1)] = k;
  }
  __syncthreads();
  const int count = sm.count;
  for (int i = t; i < count; i += kThreads) {
    const uint2 k = sm.cand[i];
    int rank = 0;
    for (int j = 0; j < count; ++j) rank += before(sm.cand[j], k);
    if (rank < top) sm.best[rank] = k;
  }
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const Params p) {
  constexpr int E = Row<T>::E, U = 4;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Smem &sm = *(Smem *)smem_raw;
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.y, split = blockIdx.x;
  const Row<T> r(p, row);
  const int g0 = (int)((int64_t)r.groups * split / p.splits), g1 = (int)((int64_t)r.groups * (split + 1) / p.splits);
  uint32_t *keys = p.splits == 1 ? sm.keys : p.keys + (int64_t)row * p.key_stride;
  uint32_t largest = 0u;
  auto note = [&](int g, uint32_t key) {
    key = __reduce_max_sync(0xffffffffu, key);
    largest = max(largest, key);
    if (p.top && lane == 0) keys[g] = key;
  };
  // groups that lie inside the row whole, U loads on their way at once
  const int whole0 = max(g0, r.off ? 1 : 0), whole1 = min(g1, (r.v + r.off) / (32 * E));
  Sums2 a2 = {-INFINITY, 0u, 0u};
  for (int g = whole0 + warp; g < whole1; g += U * kWarps) {
    uint4 c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      c[u] = make_uint4(0u, 0u, 0u, 0u);
      if (g + u * kWarps < whole1) c[u] = __ldg((const uint4 *)(r.x - r.off) + (g + u * kWarps) * 32 + lane);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (g + u * kWarps < whole1) note(g + u * kWarps, key_of(take2<E>(a2, c[u])));
  }
  const float2 s2 = halves(a2.s), w2 = halves(a2.w);
  Sums a = {a2.m, s2.x + s2.y, w2.x + w2.y};
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
    note(ends[i], any ? key_of(mx) : 0u);
  }
  join_lanes<32>(a);
  if (lane == 0) sm.sums[warp] = a, sm.largest[warp] = largest;
  __syncthreads();
  if (warp == 0) {
    a = lane < kWarps ? sm.sums[lane] : Sums{-INFINITY, 0.f, 0.f};
    join_lanes<kWarps>(a);
    largest = __reduce_max_sync(0xffffffffu, lane < kWarps ? sm.largest[lane] : 0u);
  }
  if (p.splits > 1) {
    if (threadIdx.x == 0) {
      p.parts[(int64_t)row * p.splits + split] = make_float4(a.m, a.s, a.w, __uint_as_float(largest));
      __threadfence();  // the record and (by the barrier) the keys
      const bool last = atomicAdd(p.cnt + row, 1u) == (unsigned)p.splits - 1u;
      if (last) {
        __threadfence();
        p.cnt[row] = 0u;
      }
      sm.last = last;
    }
    __syncthreads();
    if (!sm.last) return;
    if (warp == 0) {  // the row's parts: a lane takes every 32nd, then the lanes'
      a = {-INFINITY, 0.f, 0.f}, largest = 0u;
      for (int i = lane; i < p.splits; i += 32) {
        const float4 t = __ldcg(p.parts + (int64_t)row * p.splits + i);
        join(a, Sums{t.x, t.y, t.z});
        largest = max(largest, __float_as_uint(t.w));
      }
      join_lanes<32>(a);
      largest = __reduce_max_sync(0xffffffffu, largest);
    }
  }
  if (warp == 0) {
    const bool none = largest == kNegInf, bad = largest >= kInf;
    // of a row of -inf alone, log p is that too: x - 0 - 0
    const float m = bad ? NAN : (none ? 0.f : a.m), log_s = none ? 0.f : log2f(a.s) * kLn2;
    if (lane == 0) {
      sm.m = m, sm.log_s = log_s;
      p.entropy[row] = bad ? NAN : (none ? 0.f : fmaxf(0.f, log_s - a.w / a.s * kLn2));
      if (p.tokens) {
        const int64_t t = p.tokens[row];
        float lp = 0.f;  // -1: no token
        if (t >= 0 && t < p.v) lp = Row<T>::widen(r.x[t]) - m - log_s;
        else if (t != -1) set_device_error(EGPT_ERR_SHAPE), lp = NAN;
        p.logp[row] = lp;
      }
    }
  }
  if (!p.top) return;
  // ---- the groups with the top tokens, then the first of their elements
  const bool split_keys = p.splits > 1;
  select(sm, r.groups, p.top, [&](int i) { return make_uint2(split_keys ? __ldcg(keys + i) : keys[i], ~(uint32_t)i); });
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
    p.top_logp[(int64_t)row * p.top + threadIdx.x] = value_of(k.x) - sm.m - sm.log_s;
  }
}

static int group_elems(bool f32) { return 512 / (f32 ? 4 : 2); }
// Groups of a row at most (a row may start inside a 16-byte chunk).
static int most_groups(int64_t v, bool f32) { return (int)((v + 16 / (f32 ? 4 : 2) - 1 + group_elems(f32) - 1) / group_elems(f32)); }
// CTAs of a row: about two for every SM, each with 16 groups (two loads a warp) at least; rows alone fill the GPU otherwise.
static int splits_of(int64_t m, int64_t v, bool f32) {
  const int64_t want = std::min<int64_t>(2 * num_sms() / m, most_groups(v, f32) / 16);
  return m > kSplitRows ? 1 : (int)std::max<int64_t>(1, want);
}
static size_t ws_bytes(int64_t m, int64_t v, bool f32) {
  if (splits_of(m, v, f32) == 1) return 0;
  return kSplitRows * sizeof(unsigned) + (size_t)m * (splits_of(m, v, f32) * sizeof(float4) + (most_groups(v, f32) + 3) / 4 * 16);
}

}  // namespace lgp
}  // namespace egpt

using namespace egpt;

extern "C" size_t egpt_token_logprobs_ws_bytes(int64_t m, int64_t v) {
  if (m < 1 || v < 1 || v > lgp::kMaxVocab) return 0;
  return std::max(lgp::ws_bytes(m, v, false), lgp::ws_bytes(m, v, true));
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
  p.splits = lgp::splits_of(m, v, f32);
  if (p.splits > 1) {
    if (!ws || ws_bytes < lgp::ws_bytes(m, v, f32)) return set_error(EGPT_ERR_WORKSPACE, "token_logprobs: workspace too small");
    if ((uintptr_t)ws % 16) return set_error(EGPT_ERR_ALIGN, "token_logprobs: workspace must be 16-byte aligned");
  }
  p.x = logits, p.ldx = ldx, p.tokens = tokens, p.m = (int)m, p.v = (int)v, p.top = top;
  p.logp = logp, p.entropy = entropy, p.top_logp = top_logp, p.top_ids = top_ids;
  p.cnt = (unsigned *)ws, p.parts = (float4 *)((char *)ws + lgp::kSplitRows * sizeof(unsigned));
  p.keys = (uint32_t *)(p.parts + m * p.splits), p.key_stride = (lgp::most_groups(v, f32) + 3) / 4 * 4;
  const int words = std::max(p.splits == 1 ? lgp::most_groups(v, f32) : 0, top * lgp::group_elems(f32));
  const size_t smem = sizeof(lgp::Smem) + (top ? words * sizeof(uint32_t) : 0);
  const void *fn = f32 ? (const void *)lgp::logprobs_kernel<float> : (const void *)lgp::logprobs_kernel<uint16_t>;
  return check_launch(launch_kernel(fn, dim3((unsigned)p.splits, (unsigned)m), dim3(lgp::kThreads), smem, (cudaStream_t)stream,
                                    (flags & EGPT_FLAG_PDL) != 0, p),
                      "token_logprobs_kernel");
}
