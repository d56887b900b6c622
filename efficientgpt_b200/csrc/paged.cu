// The paged KV cache: a batch's key and value rows written to the pages of their sequences, and read back.
//
// A pool is `pages` pages of S rows (S a power of two) for every kv head, K and V apart: [page][kv head][S][d], bf16 rows
// or int8 codes with one fp32 scale a row (kv_q8.cu's quantiser). table[i][c] names the page of slots c S .. c S + S - 1 of
// sequence i (-1: none). A page's rows of one head lie together, so that attention streams S d elements at a time and
// a tensor of one page is the contiguous caches' [heads][cap][d] with cap = S. Single passes: few rows are bound by the launch
// and the round trips to memory that find their place (one row 2.4 us on the device), prompts by waiting, for neither HBM nor
// the issue slots are full (3370 rows of 48 heads with norm and rotation 17.7 us, 85 MB, 4.8 TB/s, 58% of the issue slots;
// without both 5.9 TB/s; 4096 rows into int8 pages 22.5 us, 94 MB, 4.2 TB/s, and into bf16 ones 20.8, 102 MB, 4.9 TB/s): every
// wave of CTAs goes through its rows' look-ups (start, position, page, angles) together before it works on them. Reads are
// bound by HBM (32768 rows of 8 heads 36 us from int8, 203 MB, 5.7 TB/s, 43 us from bf16, 268 MB, 6.2 TB/s).
#include "internal.h"
#include "common.cuh"

namespace egpt {
namespace pgd {

constexpr int kThreads = 256;
constexpr int kMostSlots = 1 << 27;  // of a table row, and rows of a read
constexpr int kTurns = 4;  // of a warp at most, each of 32 lanes' heads of a row

struct Pool {
  void *k, *v;
  float *ks, *vs;  // null: bf16 rows
  int64_t pages;
  int shift;  // log2 of the rows of a page
  int nkv;
  const int32_t *table;
  int64_t ldt, cap;  // slots that a table row has pages for
};

// The pool row of slot `slot` of sequence `seq` and kv head 0 (head h: + h << shift), -1 without a page; a name outside the
// pool is reported.
__device__ __forceinline__ int64_t row_of(const Pool &p, int64_t seq, int64_t slot) {
  const int32_t page = p.table[seq * p.ldt + (slot >> p.shift)];
  if (page >= 0 && page < p.pages) return (((int64_t)page * p.nkv) << p.shift) + (slot & ((1 << p.shift) - 1));
  if (page != -1) set_device_error(EGPT_ERR_SHAPE);
  return -1;
}

struct AppendParams {
  Pool pool;
  const uint16_t *q, *k, *v;
  uint16_t *q_out;
  int64_t ldq, ldk, ldv, ldqo;
  const int64_t *position, *starts;  // starts null: row i is sequence i's
  int seqs, m, nq;
  const uint16_t *q_norm_w, *k_norm_w;
  float eps;
  const void *rope_cos, *rope_sin;
  int rope_f32;
  int64_t rope_rows, rope_base;
};

__device__ __forceinline__ uint4 bf16x8(const float (&x)[8]) {
  uint32_t y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y[e]) : "f"(x[2 * e + 1]), "f"(x[2 * e]));
  return make_uint4(y[0], y[1], y[2], y[3]);
}

// Eight fp32 values in pairs: two operations an instruction.
struct Eight {
  uint64_t v[4];
};
__device__ __forceinline__ Eight widen8(uint4 a) {
  return {{f2_pack(bf16_lo(a.x), bf16_hi(a.x)), f2_pack(bf16_lo(a.y), bf16_hi(a.y)), f2_pack(bf16_lo(a.z), bf16_hi(a.z)),
           f2_pack(bf16_lo(a.w), bf16_hi(a.w))}};
}
__device__ __forceinline__ Eight load8(const void *src, int64_t at, bool f32) {
  if (!f32) return widen8(*(const uint4 *)((const uint16_t *)src + at));
  const float4 a = ((const float4 *)((const float *)src + at))[0], b = ((const float4 *)((const float *)src + at))[1];
  return {{f2_pack(a.x, a.y), f2_pack(a.z, a.w), f2_pack(b.x, b.y), f2_pack(b.z, b.w)}};
}
__device__ __forceinline__ void unpack(float (&y)[8], const Eight &x) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 h = f2_unpack(x.v[e]);
    y[2 * e] = h.x, y[2 * e + 1] = h.y;
  }
}

__device__ __forceinline__ void copy16(void *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

// A head of q (KIND 0), k (1) or v (2): norm, rotation by the angles' cosines and sines, and out to `dst` (where `store`).
template <int D, bool Q8, int KIND>
__device__ __forceinline__ void append_head(const AppendParams &p, const uint4 (&x)[2], const Eight &cosine, const Eight &sine,
                                            int e0, bool store, void *dst, float *scale_dst) {
  constexpr int kLanes = D / 16, kHalf = D / 2;
  constexpr bool kCodes = Q8 && KIND != 0;
  const uint16_t *norm_w = KIND == 0 ? p.q_norm_w : (KIND == 1 ? p.k_norm_w : nullptr);
  const bool turned = KIND != 2 && p.rope_cos;
  uint4 y0 = x[0], y1 = x[1];
  if (kCodes || norm_w || turned) {
    Eight lo = widen8(x[0]), hi = widen8(x[1]);
    if (norm_w) {
      uint64_t s2 = 0u;
#pragma unroll
      for (int e = 0; e < 4; ++e) s2 = f2_fma(lo.v[e], lo.v[e], f2_fma(hi.v[e], hi.v[e], s2));
      const float2 s = f2_unpack(s2);
      float ss = s.x + s.y;
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float inv = rsqrtf(ss / (float)D + p.eps);
      const Eight w0 = widen8(*(const uint4 *)(norm_w + e0)), w1 = widen8(*(const uint4 *)(norm_w + kHalf + e0));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        lo.v[e] = f2_mul(f2_mul(lo.v[e], f2_pack(inv, inv)), w0.v[e]);
        hi.v[e] = f2_mul(f2_mul(hi.v[e], f2_pack(inv, inv)), w1.v[e]);
      }
    }
    if (turned) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 a = f2_unpack(f2_mul(lo.v[e], cosine.v[e])), b = f2_unpack(hi.v[e]), s = f2_unpack(sine.v[e]);
        hi.v[e] = f2_fma(lo.v[e], sine.v[e], f2_mul(hi.v[e], cosine.v[e]));
        lo.v[e] = f2_pack(fmaf(-b.x, s.x, a.x), fmaf(-b.y, s.y, a.y));
      }
    }
    float l[8], h[8];
    unpack(l, lo), unpack(h, hi);
    if (kCodes) {
      uint32_t amax = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = max(amax, max(kvq::magnitude(l[e]), kvq::magnitude(h[e])));
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      if (!store) return;
      const float scale = kvq::row_scale(amax);
      *(uint2 *)dst = kvq::codes_of(l, scale);
      *(uint2 *)((int8_t *)dst + kHalf) = kvq::codes_of(h, scale);
      if (e0 == 0) *scale_dst = scale;
      return;
    }
    y0 = bf16x8(l), y1 = bf16x8(h);
  }
  if (!store) return;
  *(uint4 *)dst = y0;
  *(uint4 *)((uint16_t *)dst + kHalf) = y1;
}

// A warp takes one row, or every parts-th of its turns: so the row's sequence, slot and page are found once (the starts 32 at a
// time), the angles are read once, and all of its heads are on their way to shared memory before that (4% less time than with
// one turn ahead in registers). A turn takes heads of one kind, q, k or v, D / 16 lanes to a head: lane l dims 8 l .. 8 l + 7
// and the D / 2 further on that the half-layout rotation pairs them with, so a vector is read once in 16-byte pieces, the
// rotation stays inside a lane, and the norm and the quantiser's maximum take a few shuffles. Norm and rotation are fp32 and
// rounded once, to bf16 or to a code. (With the norm weights in shared memory as fp32 12% longer, for the barrier.)
template <int D, bool Q8>
__global__ void __launch_bounds__(kThreads, 4) append_kernel(const AppendParams p) {
  constexpr int kLanes = D / 16, kHalf = D / 2, kGroups = 32 / kLanes, kBytes = Q8 ? 1 : 2;
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, group = lane / kLanes, e0 = (lane % kLanes) * 8;
  const int row = (int)blockIdx.x * (kThreads / 32) + (int)(threadIdx.x >> 5), part = (int)blockIdx.y, parts = (int)gridDim.y;
  if (row >= p.m) return;
  const int nq = p.nq, nkv = p.pool.nkv;
  const int q_turns = (nq + kGroups - 1) / kGroups, kv_turns = (nkv + kGroups - 1) / kGroups, k_end = q_turns + kv_turns;
  const uint16_t *q_row = p.q + row * p.ldq + e0, *k_row = p.k + row * p.ldk + e0, *v_row = p.v + row * p.ldv + e0;
  __shared__ uint4 inputs[kThreads / 32][kTurns][2][32];  // a lane reads what it has copied itself
  uint4 (*mine)[2][32] = inputs[threadIdx.x >> 5];
  int turn = part;
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const int t = part + i * parts;
    const uint16_t *src = q_row;
    int head = t * kGroups + group, heads = nq;
    if (t >= q_turns) head -= q_turns * kGroups, src = k_row, heads = nkv;
    if (t >= k_end) head -= kv_turns * kGroups, src = v_row;
    if (head < heads) {
      src += head * D;
      copy16(&mine[i][0][lane], src), copy16(&mine[i][1][lane], src + kHalf);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  int taken = 0;
  auto take = [&](uint4 (&x)[2]) {  // the next turn's
    if (taken == 0) asm volatile("cp.async.wait_group %0;" ::"n"(kTurns - 1) : "memory");
    else if (taken == 1) asm volatile("cp.async.wait_group %0;" ::"n"(kTurns - 2) : "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
    x[0] = mine[taken][0][lane], x[1] = mine[taken][1][lane];
    ++taken, turn += parts;
  };

  // the row's sequence and slot
  int64_t seq = row, at = 0;
  if (p.starts) {  // the last start at or before the row
    int n = 0;
    for (int i = 0; i <= p.seqs; i += 32) {
      const int64_t s = i + lane <= p.seqs ? p.starts[i + lane] : INT64_MAX;
      const int here = __popc(__ballot_sync(0xffffffffu, s <= (int64_t)row));
      if (here) at = (int64_t)row - __shfl_sync(0xffffffffu, s, here - 1);
      n += here;
    }
    if (n == 0 || n > p.seqs) {  // rows outside every sequence stay as they are
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      return;
    }
    seq = n - 1;
  }
  const int64_t first = p.position[seq];
  const int64_t slot = first + at;
  const bool in = first >= 0 && first < p.pool.cap && at >= 0 && slot < p.pool.cap &&
                  (!p.rope_cos || slot < p.rope_rows - p.rope_base);
  uint16_t *q_out = p.q_out + row * p.ldqo + e0;
  if (!in) {  // no position to rotate to: q is zeros
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (first != -1) set_device_error(EGPT_ERR_SHAPE);  // -1: an idle slot of the batch
    for (; turn < q_turns; turn += parts) {
      const int head = turn * kGroups + group;
      if (head >= nq) break;
      *(uint4 *)(q_out + head * D) = *(uint4 *)(q_out + head * D + kHalf) = make_uint4(0u, 0u, 0u, 0u);
    }
    return;
  }
  const int64_t dst = row_of(p.pool, seq, slot);
  if (dst < 0) set_device_error(EGPT_ERR_SHAPE);
  Eight cosine, sine;
  if (p.rope_cos) {
    const int64_t angle = (slot + p.rope_base) * kHalf + e0;
    cosine = load8(p.rope_cos, angle, p.rope_f32), sine = load8(p.rope_sin, angle, p.rope_f32);
  }
  uint4 x[2];
  while (turn < q_turns) {
    const int head = turn * kGroups + group;
    take(x);
    append_head<D, Q8, 0>(p, x, cosine, sine, e0, head < nq, q_out + head * D, nullptr);
  }
  uint8_t *k_dst = (uint8_t *)p.pool.k + (dst * D + e0) * kBytes, *v_dst = (uint8_t *)p.pool.v + (dst * D + e0) * kBytes;
  while (turn < k_end) {
    const int head = (turn - q_turns) * kGroups + group, skip = head << p.pool.shift;  // rows to the head's
    take(x);
    append_head<D, Q8, 1>(p, x, cosine, sine, e0, head < nkv && dst >= 0, k_dst + (int64_t)skip * (D * kBytes),
                          p.pool.ks + dst + skip);
  }
  while (turn < k_end + kv_turns) {
    const int head = (turn - k_end) * kGroups + group, skip = head << p.pool.shift;
    take(x);
    append_head<D, Q8, 2>(p, x, cosine, sine, e0, head < nkv && dst >= 0, v_dst + (int64_t)skip * (D * kBytes),
                          p.pool.vs + dst + skip);
  }
}

struct ReadParams {
  Pool pool;
  void *k_out, *v_out;
  int64_t out_head;  // elements between the heads of the outputs
  int64_t start, count;
  const int64_t *starts;  // nullable: every sequence's first slot
  int seqs;
};

// out[i nkv + h][r] = row start_i + r of head h of sequence i: eight elements a thread, of K and of V, so that neighbouring
// threads write neighbouring 16-byte pieces (sixteen codes a thread, whose two pieces leave one after the other, take 8% longer
// for 32768 int8 rows of 8 heads), ROWS rows' on their way at once (two where that fills the GPU twice over: one takes 4% longer
// for those 32768 rows, and four and eight, which leave too few threads to an SM, 5% and 29%; one for shorter stretches:
// two take 7% longer for 4096 rows). The stores are marked as passing through, like the loads (2% less, over bf16 pages 3%).
// Sequence and head come from the grid and slots are 32 bits (a division and 64-bit slots a row: 9% longer), in 32 registers,
// so that an SM has all its threads (40 registers and 10% fewer instructions: 6% longer).
template <int D, bool Q8, bool F32, int ROWS>
__global__ void __launch_bounds__(kThreads) read_kernel(const ReadParams p) {
  constexpr int kElems = 8, kLanes = D / kElems, kStep = kThreads / kLanes;
  pdl_wait();
  pdl_launch_dependents();
  const int e0 = (int)(threadIdx.x % kLanes) * kElems, head = (int)blockIdx.y, count = (int)p.count;
  for (int seq = blockIdx.z; seq < p.seqs; seq += gridDim.z) {
    // rows before slot 0 and behind the last one are zeros (any start further off is as good)
    const int start = (int)min(max(p.starts ? p.starts[seq] : p.start, (int64_t)-kMostSlots), p.pool.cap);
    const int64_t out0 = ((int64_t)seq * p.pool.nkv + head) * p.out_head + e0;
    for (int r0 = (int)blockIdx.x * (kStep * ROWS) + (int)threadIdx.x / kLanes; r0 < count; r0 += (int)gridDim.x * (kStep * ROWS)) {
      uint4 x[ROWS][2];  // (codes: half of it)
      float scale[ROWS][2];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int r = r0 + i * kStep, slot = start + r;
        int64_t src = r < count && slot >= 0 && slot < (int)p.pool.cap ? row_of(p.pool, seq, slot) : -1;
        if (src >= 0) src += (int64_t)head << p.pool.shift;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const uint8_t *rows = (const uint8_t *)(kv ? p.pool.v : p.pool.k) + (src * D + e0) * (Q8 ? 1 : 2);
          x[i][kv] = make_uint4(0u, 0u, 0u, 0u);
          if (src >= 0) {
            if (Q8) {
              const uint2 codes = __ldcs((const uint2 *)rows);
              x[i][kv].x = codes.x, x[i][kv].y = codes.y;
            } else {
              x[i][kv] = __ldcs((const uint4 *)rows);
            }
          }
          scale[i][kv] = Q8 && src >= 0 ? (kv ? p.pool.vs : p.pool.ks)[src] : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int r = r0 + i * kStep;
        if (r >= count) break;
        const int64_t at = out0 + (int64_t)r * D;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const uint32_t w[4] = {x[i][kv].x, x[i][kv].y, x[i][kv].z, x[i][kv].w};
          void *out = kv ? p.v_out : p.k_out;
          if constexpr (!Q8 && !F32) {
            __stcs((uint4 *)((uint16_t *)out + at), x[i][kv]);
          } else {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              // a code plus 128 below 0x4b0000 is 2^23 + 128 + code (conversions of integers run at a quarter of the rate)
              if (Q8) y[j] = (__uint_as_float(__byte_perm(w[j / 4] ^ 0x80808080u, 0x4b000000u, 0x7440 + j % 4)) - 8388736.f) * scale[i][kv];
              else y[j] = j % 2 ? bf16_hi(w[j / 2]) : bf16_lo(w[j / 2]);
            }
            if (F32) {
              float4 *dst = (float4 *)((float *)out + at);
              __stcs(dst, make_float4(y[0], y[1], y[2], y[3]));
              __stcs(dst + 1, make_float4(y[4], y[5], y[6], y[7]));
            } else {
              __stcs((uint4 *)((uint16_t *)out + at), bf16x8(y));
            }
          }
        }
      }
    }
  }
}

template <int D>
static const void *append_fn(bool q8) {
  return q8 ? (const void *)append_kernel<D, true> : (const void *)append_kernel<D, false>;
}
template <int D, int ROWS>
static const void *read_fn(bool q8, bool f32) {
  if (q8) return f32 ? (const void *)read_kernel<D, true, true, ROWS> : (const void *)read_kernel<D, true, false, ROWS>;
  return f32 ? (const void *)read_kernel<D, false, true, ROWS> : (const void *)read_kernel<D, false, false, ROWS>;
}
template <int ROWS>
static const void *read_fn(int d, bool q8, bool f32) {
  return d == 128 ? read_fn<128, ROWS>(q8, f32) : (d == 64 ? read_fn<64, ROWS>(q8, f32) : read_fn<32, ROWS>(q8, f32));
}

// Checks a pool and its table; fills `p`.
static int pool_of(const char *what, Pool &p, const void *k, const float *ks, const void *v, const float *vs, int64_t pages,
                   int page_size, const int32_t *table, int64_t ldt, int64_t columns, int64_t seqs, int nkv, int d) {
  if (!k || !v || !table || (ks == nullptr) != (vs == nullptr)) return set_error(EGPT_ERR_ARG, "%s: null pointer", what);
  if (d != 32 && d != 64 && d != 128) return set_error(EGPT_ERR_SHAPE, "%s: head_dim must be 32, 64 or 128", what);
  if (page_size < 1 || page_size > 1024 || (page_size & (page_size - 1)))
    return set_error(EGPT_ERR_SHAPE, "%s: the rows of a page must be a power of two up to 1024", what);
  if (pages < 1 || pages > 0x7fffffff || nkv < 1 || nkv > 4096 || seqs < 1 || seqs > (1 << 30) / nkv || columns < 1 ||
      ldt < columns || columns > kMostSlots / page_size)
    return set_error(EGPT_ERR_SHAPE, "%s: bad pages, heads, sequences or table", what);
  if ((uintptr_t)k % 16 || (uintptr_t)v % 16 || (uintptr_t)ks % 4 || (uintptr_t)vs % 4 || (uintptr_t)table % 4)
    return set_error(EGPT_ERR_ALIGN, "%s: pages must be 16-byte aligned", what);
  p.k = (void *)k, p.v = (void *)v, p.ks = (float *)ks, p.vs = (float *)vs, p.pages = pages, p.nkv = nkv;
  p.shift = 0;
  while ((1 << p.shift) < page_size) ++p.shift;
  p.table = table, p.ldt = ldt, p.cap = columns * page_size;
  return EGPT_OK;
}

}  // namespace pgd
}  // namespace egpt

using namespace egpt;

extern "C" int egpt_kv_append_paged(void *k_pages, float *k_scale, void *v_pages, float *v_scale, int64_t pages,
                                    int page_size, const int32_t *table, int64_t ldt, int64_t columns, int64_t seqs,
                                    const void *k, int64_t ldk, const void *v, int64_t ldv, const int64_t *position,
                                    const int64_t *starts, int64_t m, int nkv, int d, void *q_out, int64_t ldqo, const void *q,
                                    int64_t ldq, int nq, const void *q_norm_w, const void *k_norm_w, float eps,
                                    const void *rope_cos, const void *rope_sin, int rope_dtype, int64_t rope_rows,
                                    int64_t rope_base, unsigned flags, void *stream) {
  clear_error();
  pgd::AppendParams p{};
  if (int rc = pgd::pool_of("kv_append_paged", p.pool, k_pages, k_scale, v_pages, v_scale, pages, page_size, table, ldt, columns,
                            seqs, nkv, d))
    return rc;
  if (!k || !v || !position || (q == nullptr) != (q_out == nullptr) || (rope_cos == nullptr) != (rope_sin == nullptr))
    return set_error(EGPT_ERR_ARG, "kv_append_paged: null pointer");
  if (!q && q_norm_w) return set_error(EGPT_ERR_ARG, "kv_append_paged: a q norm without q");
  if (!q) nq = 0, ldq = ldqo = 0;
  if (m < 1 || ldk < (int64_t)nkv * d || ldv < (int64_t)nkv * d || (q && (nq < 1 || nq > (1 << 16))) || ldq < (int64_t)nq * d ||
      ldqo < (int64_t)nq * d || (!starts && m != seqs))
    return set_error(EGPT_ERR_SHAPE, "kv_append_paged: bad m, heads or leading dimension (without starts a row a sequence)");
  if (rope_cos && rope_dtype != EGPT_BF16 && rope_dtype != EGPT_F32)
    return set_error(EGPT_ERR_DTYPE, "kv_append_paged: RoPE tables are bf16 or fp32");
  if (rope_cos && (rope_base < 0 || rope_rows < 1 || rope_base >= rope_rows))
    return set_error(EGPT_ERR_SHAPE, "kv_append_paged: bad rope_rows or rope_base");
  if ((uintptr_t)k % 16 || (uintptr_t)v % 16 || (uintptr_t)q % 16 || (uintptr_t)q_out % 16 || ldk % 8 || ldv % 8 || ldq % 8 ||
      ldqo % 8 || (uintptr_t)rope_cos % 16 || (uintptr_t)rope_sin % 16 || (uintptr_t)q_norm_w % 16 || (uintptr_t)k_norm_w % 16)
    return set_error(EGPT_ERR_ALIGN, "kv_append_paged: rows, norm weights and RoPE tables must be 16-byte aligned");
  const int64_t vectors = nq + 2 * (int64_t)nkv, per_cta = pgd::kThreads / 32;
  if (m > 0x7fffffff / vectors) return set_error(EGPT_ERR_SHAPE, "kv_append_paged: too many rows");
  p.q = (const uint16_t *)q, p.k = (const uint16_t *)k, p.v = (const uint16_t *)v, p.q_out = (uint16_t *)q_out;
  p.ldq = ldq, p.ldk = ldk, p.ldv = ldv, p.ldqo = ldqo, p.position = position, p.starts = starts;
  p.seqs = (int)seqs, p.m = (int)m, p.nq = nq;
  // kTurns turns of a row's heads to a warp (three take 1% longer for 4096 rows of 48 heads and 2% less for 3370, six 4% and 5%
  // longer), fewer as long as that makes no more than 16 warps an SM
  const int64_t groups = 512 / d, turns = (nq + groups - 1) / groups + 2 * ((nkv + groups - 1) / groups);
  const int64_t parts = std::max<int64_t>((turns + pgd::kTurns - 1) / pgd::kTurns, std::min<int64_t>(turns, 16 * num_sms() / m));
  p.q_norm_w = (const uint16_t *)q_norm_w, p.k_norm_w = (const uint16_t *)k_norm_w, p.eps = eps;
  p.rope_cos = rope_cos, p.rope_sin = rope_sin, p.rope_f32 = rope_dtype == EGPT_F32;
  p.rope_rows = rope_rows, p.rope_base = rope_base;
  const void *fn = d == 128 ? pgd::append_fn<128>(k_scale) : (d == 64 ? pgd::append_fn<64>(k_scale) : pgd::append_fn<32>(k_scale));
  return check_launch(launch_kernel(fn, dim3((unsigned)((m + per_cta - 1) / per_cta), (unsigned)parts), dim3(pgd::kThreads), 0,
                                    (cudaStream_t)stream, (flags & EGPT_FLAG_PDL) != 0, p),
                      "kv_append_paged_kernel");
}

extern "C" int egpt_kv_read_paged(void *k_out, void *v_out, int64_t out_head_stride, int dtype, const void *k_pages,
                                  const float *k_scale, const void *v_pages, const float *v_scale, int64_t pages,
                                  int page_size, const int32_t *table, int64_t ldt, int64_t columns, int64_t seqs, int nkv,
                                  int d, int64_t start, const int64_t *starts, int64_t count, unsigned flags, void *stream) {
  clear_error();
  pgd::ReadParams p{};
  if (int rc = pgd::pool_of("kv_read_paged", p.pool, k_pages, k_scale, v_pages, v_scale, pages, page_size, table, ldt, columns,
                            seqs, nkv, d))
    return rc;
  if (!k_out || !v_out) return set_error(EGPT_ERR_ARG, "kv_read_paged: null pointer");
  if (dtype != EGPT_BF16 && dtype != EGPT_F32) return set_error(EGPT_ERR_DTYPE, "kv_read_paged: the output is bf16 or fp32");
  if (count < 1 || count > pgd::kMostSlots || out_head_stride < count * d || (!starts && (start < 0 || start > p.pool.cap - count)))
    return set_error(EGPT_ERR_SHAPE, "kv_read_paged: rows [start, start + count) outside the table, or bad output stride");
  const bool f32 = dtype == EGPT_F32, q8 = k_scale != nullptr;
  if ((uintptr_t)k_out % 16 || (uintptr_t)v_out % 16 || (out_head_stride * (f32 ? 4 : 2)) % 16)
    return set_error(EGPT_ERR_ALIGN, "kv_read_paged: outputs must be 16-byte aligned");
  p.k_out = k_out, p.v_out = v_out, p.out_head = out_head_stride, p.start = start, p.count = count, p.starts = starts;
  p.seqs = (int)seqs;
  const int64_t lanes = d / 8;
  const bool two = seqs * nkv * count * lanes >= (int64_t)num_sms() * 4 * 4 * pgd::kThreads;
  const int64_t per_cta = (two ? 2 : 1) * pgd::kThreads / lanes;
  const dim3 grid((unsigned)std::min<int64_t>((count + per_cta - 1) / per_cta, 1 << 16), (unsigned)nkv,
                  (unsigned)std::min<int64_t>(seqs, 65535));
  const void *fn = two ? pgd::read_fn<2>(d, q8, f32) : pgd::read_fn<1>(d, q8, f32);
  return check_launch(launch_kernel(fn, grid, dim3(pgd::kThreads), 0, (cudaStream_t)stream, (flags & EGPT_FLAG_PDL) != 0, p),
                      "kv_read_paged_kernel");
}
