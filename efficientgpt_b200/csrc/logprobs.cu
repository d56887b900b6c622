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
  if (a.m == -INFINITY) {
    a.s = a.w = 0.f;
  } else {
    const float t = (a.m - m) * kLog2e, f = exp2f(t);
    a.w = f == 0.f ? 0.f : f * fmaf(t, a.s, a.w), a.s *= f;
  }
  a.m = m;
}
__device__ __forceinline__ void join(Sums &a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return;
  rescale(a, m), rescale(b, m);
  a.s += b.s, a.w += b.w;
}
template <int E>
__device__ __forceinline__ void take(Sums &a, const float (&y)[E], float largest) {
  if (largest > a.m) rescale(a, largest);
  const float m = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float t = fmaxf((y[e] - m) * kLog2e, -1000.f);  // (2^-1000 is 0, and 0 times it too)
    const float f = apf::ex2(t);
    a.s += f, a.w = fmaf(f, t, a.w);
  }
}

// The `top` largest of a warp's keys (hi, then the lower index first: lo = ~index), N a lane; lane j gets the j-th. Keys of 0 are
// none.
template <int N>
__device__ __forceinline__ uint2 select(uint32_t (&hi)[N], uint32_t (&lo)[N], int top) {
  const int lane = threadIdx.x & 31;
  uint2 mine = make_uint2(0u, 0u);
#pragma unroll 1
  for (int j = 0; j < top; ++j) {
    uint32_t bh = 0u, bl = 0u;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (hi[i] > bh || (hi[i] == bh && lo[i] > bl)) bh = hi[i], bl = lo[i];
    const uint32_t mh = __reduce_max_sync(0xffffffffu, bh);
    if (mh == 0u) break;
    const uint32_t ml = __reduce_max_sync(0xffffffffu, bh == mh ? bl : 0u);
    if (lane == j) mine = make_uint2(mh, ml);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (hi[i] == mh && lo[i] == ml) hi[i] = 0u;
  }
  return mine;
}

struct Smem {
  Sums sums[kWarps];
  uint32_t largest[kWarps];
  uint2 cand[kWarps][kMaxTop];  // the warps' selections
  uint2 best[kMaxTop];
  uint2 found[kMaxTop * kMaxTop];  // elements of the selected groups
  int count, last;
  float m, log_s;
  uint32_t keys[1];  // the row's groups, where no other CTA has some
};

// The `top` largest of keys get(0 .. n - 1), in order, into sm.best (0 where there are fewer). Every thread calls it.
template <typename F>
__device__ __forceinline__ void select_block(Smem &sm, int n, int top, F get) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint2 mine = make_uint2(0u, 0u);
  for (int i0 = warp * 128; i0 < n; i0 += kWarps * 128) {
    uint32_t hi[5], lo[5];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = i0 + 32 * i + lane;
      const uint2 k = at < n ? get(at) : make_uint2(0u, 0u);
      hi[i] = k.x, lo[i] = k.y;
    }
    hi[4] = mine.x, lo[4] = mine.y;
    mine = select<5>(hi, lo, top);
  }
  sm.cand[warp][lane] = mine;
  __syncthreads();
  if (warp == 0) {
    uint32_t hi[kWarps], lo[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const uint2 k = lane < top ? sm.cand[w][lane] : make_uint2(0u, 0u);
      hi[w] = k.x, lo[w] = k.y;
    }
    sm.best[lane] = select<kWarps>(hi, lo, top);
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
  Sums a = {-INFINITY, 0.f, 0.f};
  uint32_t largest = 0u;
  for (int g = g0 + warp; g < g1; g += U * kWarps) {
    float y[U][E];
    bool any[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      any[u] = false;
      if (g + u * kWarps < g1) any[u] = r.load((g + u * kWarps) * 32 + lane, y[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (g + u * kWarps >= g1) break;
      float mx = y[u][0];
      bool nan = false;
#pragma unroll
      for (int e = 0; e < E; ++e) mx = fmaxf(mx, y[u][e]), nan |= y[u][e] != y[u][e];
      if (any[u]) take<E>(a, y[u], mx);
      const uint32_t key = __reduce_max_sync(0xffffffffu, any[u] ? (nan ? 0xffffffffu : key_of(mx)) : 0u);
      largest = max(largest, key);
      if (p.top && lane == 0) keys[g + u * kWarps] = key;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Sums b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
    b.w = __shfl_xor_sync(0xffffffffu, a.w, o);
    if (lane & o) {  // the same order in both lanes
      const Sums t = a;
      a = b, b = t;
    }
    join(a, b);
  }
  if (lane == 0) sm.sums[warp] = a, sm.largest[warp] = largest;
  __syncthreads();
  if (p.splits > 1) {
    if (threadIdx.x == 0) {
      for (int w = 1; w < kWarps; ++w) join(a, sm.sums[w]), largest = max(largest, sm.largest[w]);
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
  }
  // ---- the row: all sums, in the order of the parts (warp 0: a lane takes some, then the lanes')
  const int n = p.splits > 1 ? p.splits : kWarps;
  if (warp == 0) {
    a = {-INFINITY, 0.f, 0.f}, largest = 0u;
    for (int i = lane; i < n; i += 32) {
      Sums b;
      uint32_t k;
      if (p.splits > 1) {
        const float4 t = __ldcg(p.parts + (int64_t)row * p.splits + i);
        b = {t.x, t.y, t.z}, k = __float_as_uint(t.w);
      } else {
        b = sm.sums[i], k = sm.largest[i];
      }
      join(a, b);
      largest = max(largest, k);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      Sums b;
      b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
      b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
      b.w = __shfl_xor_sync(0xffffffffu, a.w, o);
      if (lane & o) {
        const Sums t = a;
        a = b, b = t;
      }
      join(a, b);
    }
    largest = __reduce_max_sync(0xffffffffu, largest);
    const bool none = largest == kNegInf, bad = largest >= kInf;
    // of a row of -inf alone, log p is that too: x - 0 - 0
    const float m = bad ? NAN : (none ? 0.f : a.m), log_s = none ? 0.f : log2f(a.s) * kLn2;
    if (lane == 0) {
      sm.m = m, sm.log_s = log_s, sm.count = 0;
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
  __syncthreads();
  // ---- the groups with the top tokens, then their elements that can be some
  const bool split_keys = p.splits > 1;
  select_block(sm, r.groups, p.top, [&](int i) { return make_uint2(split_keys ? __ldcg(keys + i) : keys[i], ~(uint32_t)i); });
  const int groups = min(p.top, r.groups);
  const uint32_t least = r.groups < p.top ? 1u : sm.best[p.top - 1].x;
#pragma unroll 1
  for (int j = warp; j < groups; j += kWarps) {
    const int c = (int)~sm.best[j].y * 32 + lane;
    float y[E];
    uint32_t hi[E], lo[E];
    r.load(c, y);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = c * E - r.off + e;
      hi[e] = i >= 0 && i < r.v ? key_of(y[e]) : 0u, lo[e] = ~(uint32_t)i;
      if (hi[e] < least) hi[e] = 0u;
    }
    const uint2 mine = select<E>(hi, lo, p.top);
    const unsigned have = __ballot_sync(0xffffffffu, mine.x != 0u);
    int at = 0;
    if (lane == 0) at = atomicAdd(&sm.count, __popc(have));
    at = __shfl_sync(0xffffffffu, at, 0);
    if (mine.x != 0u) sm.found[at + lane] = mine;
  }
  __syncthreads();
  select_block(sm, sm.count, p.top, [&](int i) { return sm.found[i]; });
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
  const size_t smem = sizeof(lgp::Smem) + (p.splits == 1 && top ? (size_t)lgp::most_groups(v, f32) * sizeof(uint32_t) : 0);
  const void *fn = f32 ? (const void *)lgp::logprobs_kernel<float> : (const void *)lgp::logprobs_kernel<uint16_t>;
  return check_launch(launch_kernel(fn, dim3((unsigned)p.splits, (unsigned)m), dim3(lgp::kThreads), smem, (cudaStream_t)stream,
                                    (flags & EGPT_FLAG_PDL) != 0, p),
                      "token_logprobs_kernel");
}
