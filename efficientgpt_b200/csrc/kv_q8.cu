// The int8 KV cache: quantising key and value rows as they are written, and reading a stretch of them back.
//
// A cached row is its d codes (int8, layout [heads][cap][d], the bf16 caches' layout) and one fp32 scale
// ([heads][cap]): s = max(max|x| fl32(1/127), 1e-12), q = clamp(rint(x / s), -127, 127), the quantiser of the weight
// rows (quantize_rows_kernel); a code stands for q s. A scale per row and head keeps every key's and value's error
// within half a step of its own largest element whatever its neighbours hold, and lets a row be written without
// touching another one. All kernels here are single passes, bound by HBM for long stretches and by the launch and two
// round trips to memory for a few rows. Measured with 8 heads of 128: 4096 prompt rows of bf16 written in 11.5 us
// (25.4 MB, 2.2 TB/s), of fp32 in 9.6 us (42.2 MB), one row in 2.6 us; 32768 rows read back in 38.6 us (203.4 MB,
// 5.3 TB/s, 81% of a measured copy).
#include "internal.h"
#include "common.cuh"

namespace egpt {
namespace kvq {

constexpr int kThreads = 256;

struct AppendParams {
  int8_t *k_cache, *v_cache;
  float *k_scale, *v_scale;
  int64_t cap;
  const void *k, *v;
  int64_t ldk, ldv;
  const int64_t *position;
  int64_t m;
  int nkv, d, ragged;
  int plain;  // bf16 caches without scales: the rows as they are
  // prologue of a decode step (q non-null): q/k RMSNorm and RoPE as the bf16 append does them
  uint16_t *q_out;
  const uint16_t *q;
  int64_t ldq, ldqo;
  int nq;
  const uint16_t *q_norm_w, *k_norm_w;
  float eps;
  const uint16_t *rope_cos, *rope_sin;
  int64_t rope_base;
};

// The slot of row `row` (-1: nothing is written) and its first cache head.
__device__ __forceinline__ int64_t slot_of(const AppendParams &p, int64_t row, int64_t &head0) {
  const int64_t pos = p.ragged ? p.position[row] : *p.position + row;
  head0 = p.ragged ? row * p.nkv : 0;
  if (pos >= 0 && pos < p.cap) return pos;
  if (!(p.ragged && pos == -1)) set_device_error(EGPT_ERR_SHAPE);  // -1: an idle slot of a ragged batch
  return -1;
}

// The largest magnitude is kept as its bits, whose order is that of the magnitudes with infinity and NaN at the top: a row
// that holds one of those gets the scale NaN, so all that reads it sees it.
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ float row_scale(uint32_t amax) {
  return amax >= 0x7f800000u ? NAN : fmaxf(__uint_as_float(amax) * (1.0f / 127.0f), 1e-12f);
}
__device__ __forceinline__ int code_of(float x, float s) {
  return (int)fminf(fmaxf(rintf(__fdiv_rn(x, s)), -127.f), 127.f);
}

// Codes of eight elements, one to a byte. A product with 1 / s is within 2^-15 of the quotient, so it decides every code
// whose quotient is not that near to a half. One within 1e-4 of a half (one element in 5000) sends its thread's eight
// to the division (one thread in 625, one warp in 20). The rounding is
// that of a sum with 1.5 2^23, whose low byte is the code (|x / s| < 127.5 by the choice of s: nothing to clamp).
__device__ __forceinline__ uint2 codes_of(const float (&x)[8], float s) {
  constexpr float kMagic = 12582912.f;
  const float r = __frcp_rn(s);
  float near = 0.f;
  uint32_t b[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y = x[e] * r, m = y + kMagic;
    near = fmaxf(near, fabsf(y - (m - kMagic)));
    b[e] = __float_as_uint(m);
  }
  if (near > 0.4999f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = (uint32_t)code_of(x[e], s);
  }
  return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
}

// Rows as they are: D / 8 lanes hold a row, 16 bytes (bf16) or 32 bytes (fp32) each, so it is read once and its maximum
// needs a few shuffles; a thread takes the K and the V piece of one (row, head), heads innermost as they lie in the rows
// (with the rows innermost, as they lie in the cache, a third slower).
template <int D, bool F32>
__global__ void __launch_bounds__(kThreads) append_kernel(AppendParams p) {
  constexpr int kLanes = D / 8, kRows = kThreads / kLanes;
  pdl_wait();
  pdl_launch_dependents();
  const int e0 = (int)(threadIdx.x % kLanes) * 8;
  const unsigned item = blockIdx.x * kRows + threadIdx.x / kLanes, nkv = (unsigned)p.nkv;
  const bool live = item < (unsigned)p.m * nkv;
  const unsigned row = live ? item / nkv : 0, head = live ? item - row * nkv : 0;
  float x[2][8];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const int64_t at = (int64_t)row * (kv ? p.ldv : p.ldk) + (int64_t)head * D + e0;  // (row 0 if not live)
    if (F32) {
      const float4 *src = (const float4 *)((const float *)(kv ? p.v : p.k) + at);
      const float4 a = src[0], b = src[1];
      const float y[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) x[kv][e] = y[e];
    } else {
      const uint4 a = *(const uint4 *)((const uint16_t *)(kv ? p.v : p.k) + at);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) x[kv][2 * e] = bf16_lo(w[e]), x[kv][2 * e + 1] = bf16_hi(w[e]);
    }
  }
  int64_t head0 = 0;
  const int64_t slot = live ? slot_of(p, row, head0) : -1;
  const int64_t dst = (head0 + head) * p.cap + slot;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    uint32_t amax = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = max(amax, magnitude(x[kv][e]));
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (slot < 0) continue;
    const float s = row_scale(amax);
    *(uint2 *)((kv ? p.v_cache : p.k_cache) + dst * D + e0) = codes_of(x[kv], s);
    if (e0 == 0) (kv ? p.v_scale : p.k_scale)[dst] = s;
  }
}

// With the decode step's prologue: one warp per head vector of q, k or v (lane l: elements l + 32 i). The norm's sum
// is added in the order of head_norm_rope's block sum, so q and the row that is quantised have the bits that
// egpt_qk_norm_rope_kv_append writes. 32 q heads, 8 kv heads of 128: one row 2.7 us, 16 ragged rows 3.1 us, both a launch;
// 4096 rows 60 us int8, 54 us into bf16 caches (92 and 101 MB, 14 and 15 us of HBM): bound by its 2-byte loads and 1- and
// 2-byte stores, a warp to a vector.
template <int D>
__global__ void __launch_bounds__(kThreads) norm_rope_append_kernel(AppendParams p) {
  constexpr int N = D / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t item = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
  const int vectors = p.nq + 2 * p.nkv;
  if (item >= p.m * vectors) return;
  const int64_t row = item / vectors;
  const int vec = (int)(item - row * vectors);
  const int kind = vec < p.nq ? 0 : (vec < p.nq + p.nkv ? 1 : 2);  // q, k, v
  const int head = vec - (kind == 0 ? 0 : (kind == 1 ? p.nq : p.nq + p.nkv));
  int64_t head0;
  const int64_t slot = slot_of(p, row, head0);
  if (slot < 0) {
    if (kind == 0)  // an idle row has no position to rotate to: its q is zero
      for (int i = 0; i < N; ++i) p.q_out[row * p.ldqo + (int64_t)head * D + lane + 32 * i] = 0;
    return;
  }
  const uint16_t *src = kind == 0 ? p.q + row * p.ldq : (const uint16_t *)(kind == 1 ? p.k : p.v) +
                                                             row * (kind == 1 ? p.ldk : p.ldv);
  float x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = bf16_bits_to_f32(src[(int64_t)head * D + lane + 32 * i]);
  const uint16_t *norm_w = kind == 0 ? p.q_norm_w : p.k_norm_w;
  if (kind != 2 && norm_w) {
    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) part[i] = warp_sum(x[i] * x[i]);
    const float ss = (part[0] + part[2]) + (part[1] + part[3]);
    const float inv = rsqrtf(ss / (float)D + p.eps);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = round_bf16(round_bf16(x[i] * inv) * bf16_bits_to_f32(norm_w[lane + 32 * i]));
  }
  if (kind != 2 && p.rope_cos) {
    constexpr int half = D / 2;
    const int64_t at = (slot + p.rope_base) * half;
    float y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int t = lane + 32 * i;
      // the partner t +- d/2 is N/2 elements on in the same lane, or (d = 32) 16 lanes on
      const float other = N > 1 ? x[(i + N / 2) % N] : __shfl_xor_sync(0xffffffffu, x[i], 16);
      const int f = t < half ? t : t - half;
      const float c = bf16_bits_to_f32(p.rope_cos[at + f]), s = bf16_bits_to_f32(p.rope_sin[at + f]);
      y[i] = round_bf16(round_bf16(x[i] * c) + round_bf16((t < half ? -other : other) * s));
    }
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = y[i];
  }
  if (kind == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) p.q_out[row * p.ldqo + (int64_t)head * D + lane + 32 * i] = f32_to_bf16_bits(x[i]);
    return;
  }
  const int64_t dst = (head0 + head) * p.cap + slot;
  if (p.plain) {
    uint16_t *rows = (uint16_t *)(kind == 1 ? p.k_cache : p.v_cache) + dst * D;
#pragma unroll
    for (int i = 0; i < N; ++i) rows[lane + 32 * i] = f32_to_bf16_bits(x[i]);
    return;
  }
  uint32_t amax = 0u;
#pragma unroll
  for (int i = 0; i < N; ++i) amax = max(amax, magnitude(x[i]));
  const float s = row_scale(__reduce_max_sync(0xffffffffu, amax));
  int8_t *codes = (kind == 1 ? p.k_cache : p.v_cache) + dst * D;
#pragma unroll
  for (int i = 0; i < N; ++i) codes[lane + 32 * i] = (int8_t)code_of(x[i], s);
  if (lane == 0) (kind == 1 ? p.k_scale : p.v_scale)[dst] = s;
}

struct ReadParams {
  void *k_out, *v_out;
  int64_t out_head;  // elements between the heads of the outputs
  const int8_t *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  int64_t cap, start, count, heads;
  const int64_t *starts;  // nullable: one start per group of `group` heads (added to `start`)
  int group;
};

// out[h][r] = q s of row start + r of head h (blockIdx.y; K, then V, in blockIdx.z): 16 codes (one 16-byte load) per
// thread and row, D / 16 threads to a row, ROWS rows' loads on their way at once: four where that still fills the GPU
// (32768 rows of 8 heads: 38.6 us, 43.0 with one), one for short stretches (257 rows of 6 heads: 2.2 us, 3.1 with four).
template <int D, bool F32, int ROWS>
__global__ void __launch_bounds__(kThreads) read_kernel(ReadParams p) {
  constexpr int kLanes = D / 16, kStep = kThreads / kLanes;
  pdl_wait();
  pdl_launch_dependents();
  const int e0 = (int)(threadIdx.x % kLanes) * 16;
  const bool is_v = blockIdx.z != 0;
  for (int64_t h = blockIdx.y; h < p.heads; h += gridDim.y) {
    const int64_t start = p.start + (p.starts ? p.starts[h / p.group] : 0);
    const int8_t *codes = (is_v ? p.v_cache : p.k_cache) + h * p.cap * D + e0;
    const float *scales = (is_v ? p.v_scale : p.k_scale) + h * p.cap;
    for (int64_t r0 = (int64_t)blockIdx.x * kStep * ROWS + threadIdx.x / kLanes; r0 < p.count;
         r0 += (int64_t)gridDim.x * kStep * ROWS) {
      uint4 c[ROWS];
      float s[ROWS];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int64_t r = r0 + i * kStep, slot = start + r;
        const bool in = r < p.count && slot >= 0 && slot < p.cap;  // slots outside the cache read as zeros
        c[i] = in ? __ldcs((const uint4 *)(codes + slot * D)) : make_uint4(0u, 0u, 0u, 0u);
        s[i] = in ? scales[slot] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int64_t r = r0 + i * kStep;
        if (r >= p.count) break;
        const uint32_t w[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = (float)(int8_t)(w[e / 4] >> (8 * (e % 4))) * s[i];
        const int64_t at = h * p.out_head + r * D + e0;
        if (F32) {
          float4 *dst = (float4 *)((float *)(is_v ? p.v_out : p.k_out) + at);
#pragma unroll
          for (int e = 0; e < 4; ++e) dst[e] = make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
        } else {
          uint32_t y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            y[e] = (uint32_t)f32_to_bf16_bits(x[2 * e]) | ((uint32_t)f32_to_bf16_bits(x[2 * e + 1]) << 16);
          uint4 *dst = (uint4 *)((uint16_t *)(is_v ? p.v_out : p.k_out) + at);
          dst[0] = make_uint4(y[0], y[1], y[2], y[3]);
          dst[1] = make_uint4(y[4], y[5], y[6], y[7]);
        }
      }
    }
  }
}

template <int D>
static const void *append_fn(bool f32) {
  return f32 ? (const void *)append_kernel<D, true> : (const void *)append_kernel<D, false>;
}
template <int D>
static const void *read_fn(bool f32, bool four) {
  if (four) return f32 ? (const void *)read_kernel<D, true, 4> : (const void *)read_kernel<D, false, 4>;
  return f32 ? (const void *)read_kernel<D, true, 1> : (const void *)read_kernel<D, false, 1>;
}

}  // namespace kvq
}  // namespace egpt

using namespace egpt;

extern "C" int egpt_kv_append_q8(int8_t *k_cache, float *k_scale, int8_t *v_cache, float *v_scale, int64_t cap,
                                 const void *k, int64_t ldk, const void *v, int64_t ldv, const int64_t *position,
                                 int64_t m, int nkv, int d, int dtype, void *q_out, int64_t ldqo, const void *q,
                                 int64_t ldq, int nq, const void *q_norm_w, const void *k_norm_w, float eps,
                                 const void *rope_cos, const void *rope_sin, int64_t rope_base, unsigned flags,
                                 void *stream) {
  clear_error();
  if (!k_cache || !v_cache || !k || !v || !position || (k_scale == nullptr) != (v_scale == nullptr))
    return set_error(EGPT_ERR_ARG, "kv_append_q8: null pointer");
  if (!k_scale && !q) return set_error(EGPT_ERR_ARG, "kv_append_q8: rows for a bf16 cache (no scales) come with q");
  if (d != 32 && d != 64 && d != 128) return set_error(EGPT_ERR_SHAPE, "kv_append_q8: head_dim must be 32, 64 or 128");
  if (m < 1 || nkv < 1 || cap < 1 || ldk < (int64_t)nkv * d || ldv < (int64_t)nkv * d || m > ((int64_t)1 << 31) / nkv)
    return set_error(EGPT_ERR_SHAPE, "kv_append_q8: bad m, heads, cap or leading dimension");
  if (dtype != EGPT_BF16 && dtype != EGPT_F32) return set_error(EGPT_ERR_DTYPE, "kv_append_q8: dtype");
  const bool f32 = dtype == EGPT_F32, pdl = (flags & EGPT_FLAG_PDL) != 0;
  if ((uintptr_t)k_cache % 16 || (uintptr_t)v_cache % 16 || (uintptr_t)k % 16 || (uintptr_t)v % 16 ||
      (ldk * (f32 ? 4 : 2)) % 16 || (ldv * (f32 ? 4 : 2)) % 16 || (uintptr_t)k_scale % 4 || (uintptr_t)v_scale % 4)
    return set_error(EGPT_ERR_ALIGN, "kv_append_q8: caches and rows must be 16-byte aligned");
  kvq::AppendParams p{};
  p.k_cache = k_cache, p.v_cache = v_cache, p.k_scale = k_scale, p.v_scale = v_scale, p.cap = cap;
  p.k = k, p.v = v, p.ldk = ldk, p.ldv = ldv, p.position = position, p.m = m, p.nkv = nkv, p.d = d;
  p.ragged = (flags & EGPT_FLAG_RAGGED) != 0, p.plain = !k_scale;
  if (q) {
    if (!q_out) return set_error(EGPT_ERR_ARG, "kv_append_q8: q without q_out");
    if (f32) return set_error(EGPT_ERR_DTYPE, "kv_append_q8: fp32 rows have no norm/RoPE");
    if (nq < 1 || ldq < (int64_t)nq * d || ldqo < (int64_t)nq * d || rope_base < 0)
      return set_error(EGPT_ERR_SHAPE, "kv_append_q8: bad nq, leading dimension or rope_base");
    if ((rope_cos == nullptr) != (rope_sin == nullptr)) return set_error(EGPT_ERR_ARG, "kv_append_q8: rope_cos/rope_sin");
    const int64_t vectors = m * (nq + 2 * (int64_t)nkv), per_cta = kvq::kThreads / 32;
    if ((vectors + per_cta - 1) / per_cta > 0x7fffffff) return set_error(EGPT_ERR_SHAPE, "kv_append_q8: too many rows");
    p.q_out = (uint16_t *)q_out, p.ldqo = ldqo, p.q = (const uint16_t *)q, p.ldq = ldq, p.nq = nq;
    p.q_norm_w = (const uint16_t *)q_norm_w, p.k_norm_w = (const uint16_t *)k_norm_w, p.eps = eps;
    p.rope_cos = (const uint16_t *)rope_cos, p.rope_sin = (const uint16_t *)rope_sin, p.rope_base = rope_base;
    const void *fn = d == 128 ? (const void *)kvq::norm_rope_append_kernel<128>
                              : (d == 64 ? (const void *)kvq::norm_rope_append_kernel<64>
                                         : (const void *)kvq::norm_rope_append_kernel<32>);
    return check_launch(launch_kernel(fn, dim3((unsigned)((vectors + per_cta - 1) / per_cta)), dim3(kvq::kThreads), 0,
                                      (cudaStream_t)stream, pdl, p),
                        "norm_rope_append_kernel");
  }
  if (q_out || q_norm_w || k_norm_w || rope_cos || rope_sin)
    return set_error(EGPT_ERR_ARG, "kv_append_q8: norm and RoPE need q");
  const int64_t per_cta = kvq::kThreads / (d / 8);  // (head, row) pairs
  const void *fn = d == 128 ? kvq::append_fn<128>(f32) : (d == 64 ? kvq::append_fn<64>(f32) : kvq::append_fn<32>(f32));
  return check_launch(launch_kernel(fn, dim3((unsigned)((m * nkv + per_cta - 1) / per_cta)), dim3(kvq::kThreads), 0,
                                    (cudaStream_t)stream, pdl, p),
                      "kv_append_q8_kernel");
}

extern "C" int egpt_kv_read_q8(void *k_out, void *v_out, int64_t out_head_stride, int dtype, const int8_t *k_cache,
                               const float *k_scale, const int8_t *v_cache, const float *v_scale, int64_t cap,
                               int64_t heads, int d, int64_t start, const int64_t *starts, int heads_per_start,
                               int64_t count, unsigned flags, void *stream) {
  clear_error();
  if (!k_out || !v_out || !k_cache || !k_scale || !v_cache || !v_scale)
    return set_error(EGPT_ERR_ARG, "kv_read_q8: null pointer");
  if (d != 32 && d != 64 && d != 128) return set_error(EGPT_ERR_SHAPE, "kv_read_q8: head_dim must be 32, 64 or 128");
  if (heads < 1 || cap < 1 || count < 1 || count > ((int64_t)1 << 40) / heads || out_head_stride < count * d)
    return set_error(EGPT_ERR_SHAPE, "kv_read_q8: bad heads, cap, count or output stride");
  if (starts ? (heads_per_start < 1 || heads % heads_per_start) : (start < 0 || count > cap || start > cap - count))
    return set_error(EGPT_ERR_SHAPE, starts ? "kv_read_q8: heads must be a multiple of heads_per_start"
                                            : "kv_read_q8: rows [start, start + count) outside the cache");
  if (dtype != EGPT_BF16 && dtype != EGPT_F32) return set_error(EGPT_ERR_DTYPE, "kv_read_q8: dtype");
  const bool f32 = dtype == EGPT_F32;
  if ((uintptr_t)k_out % 16 || (uintptr_t)v_out % 16 || (uintptr_t)k_cache % 16 || (uintptr_t)v_cache % 16 ||
      (out_head_stride * (f32 ? 4 : 2)) % 16)
    return set_error(EGPT_ERR_ALIGN, "kv_read_q8: caches and outputs must be 16-byte aligned");
  kvq::ReadParams p{};
  p.k_out = k_out, p.v_out = v_out, p.out_head = out_head_stride, p.k_cache = k_cache, p.v_cache = v_cache;
  p.k_scale = k_scale, p.v_scale = v_scale, p.cap = cap, p.start = start, p.count = count, p.heads = heads;
  p.starts = starts, p.group = starts ? heads_per_start : 1;
  const bool four = 2 * heads * count * (d / 16) >= (int64_t)num_sms() * 4 * 4 * kvq::kThreads;
  const int64_t per_cta = (int64_t)(four ? 4 : 1) * kvq::kThreads / (d / 16);
  const dim3 grid((unsigned)std::min<int64_t>((count + per_cta - 1) / per_cta, 1 << 16),
                  (unsigned)std::min<int64_t>(heads, 65535), 2);
  const void *fn = d == 128 ? kvq::read_fn<128>(f32, four)
                              : (d == 64 ? kvq::read_fn<64>(f32, four) : kvq::read_fn<32>(f32, four));
  return check_launch(launch_kernel(fn, grid, dim3(kvq::kThreads), 0, (cudaStream_t)stream,
                                    (flags & EGPT_FLAG_PDL) != 0, p),
                      "kv_read_q8_kernel");
}
