// Decode attention of a batch over int8 KV caches, and over a prefix that the whole batch shares (int8 or bf16).
//
//   egpt_attn_decode_q8:      out[i, h] = sum_j w_j V[j] / sum_j w_j,  w_j = 2^(scale log2(e) q[i, h] . K[j]),
//                             over the L_i = position[i] + 1 keys of sequence i's own cache;
//   egpt_attn_shared_prefix:  the same over prefix_len keys held once and then sequence i's own L_i keys (its tail).
// K[j] = ks_j kq_j and V[j] = vs_j vq_j for int8 codes kq, vq with one scale per row and head (kv_q8.cu). GQA: head h
// reads kv head h / group. A row without any key gives zeros.
//
// Work: a segment is one cache head with the query rows that read it: (i, g) with the group's rows for a sequence's
// own cache, (g, 16 query rows) for the shared prefix, whose rows are all (sequence, head) pairs of kv head g in a
// row. A segment's keys are cut into tiles of kTile keys and all tiles of the call into equal contiguous ranges, one
// per CTA: a batch of one token next to a document leaves no CTA idle, and no length is known to the host. Within a
// range a warp takes every fourth tile through a ring of its own in shared memory (cp.async, rows past the
// segment's end filled with zeros), so warps only meet at a segment's end.
//
// Arithmetic: mma.sync m16n8k16 with the query rows as M. Scores of int8 keys: the codes become f16 exactly (0x6400 |
// (q + 128) is 1152 + q), and q, scaled by a power of two per row to at most 2^15, too, so the scores are those of the
// codes in fp32 and ks_j multiplies them. P.V is in bf16, whose exponents hold every weight times vs_j; its 8 bits
// would cost a weight 2^-9 of itself, so a weight enters as the sum of two bf16 values (16 bits). With 8 query rows
// or fewer the second values ride in the MMA's upper 8 rows, which are idle otherwise; 16 rows take a second MMA.
// Codes become bf16 exactly as (128 + low seven bits) - (128 + sign bit). Sums, maxima and accumulators are fp32; the
// output is rounded once.
#include "internal.h"
#include "common.cuh"

namespace egpt {
namespace aq8 {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxBatch = 512;
constexpr int kRows = 16;  // query rows per tile (the M of the MMA), and rows of a partial record

struct Cache {
  const uint8_t *k, *v;
  const float *ks, *vs;  // null: bf16 rows
  int64_t cap;
};

struct Params {
  uint16_t *out;
  const uint16_t *q;
  int64_t ldo, ldq;
  Cache own, shared;
  int64_t prefix;  // keys of the shared prefix (0: none)
  const int64_t *position;
  int m, nkv, group, row_tiles;  // row_tiles: 16-row tiles of a kv head's (sequence, head) rows under the prefix
  float scale_log2;
  float *ws;       // partial records
  const float *pre;  // records of attn_prefix_kernel (null: the prefix's segments are in the flat list)
  int pre_seqs, pre_tiles, pre_pairs, pre_ranges;
  unsigned *cnt;   // arrivals per (sequence, kv head); zero between calls
};

// Where the tiles of the call lie in its flat list: the prefix's segments first, then the sequences'.
struct Layout {
  int prefix_tiles, prefix_segs, prefix_end;  // tiles per prefix segment, its segments, and the list's place after them
  int total, chunk;                           // tiles of the call, tiles per CTA
};
struct Seg {
  int index, start, end;  // its number and its tiles in the flat list
  int seq, g, tile;       // sequence (-1: prefix), kv head, row tile
  int len;                // keys
};

template <int D, bool Q8>
struct Geo {
  static constexpr int kRowBytes = Q8 ? D : 2 * D;
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kTile = Q8 ? 32 : 16;  // keys per warp tile: K and V 4 KB each at d = 128
  static constexpr int kStageBytes = 2 * kTile * kRowBytes + (Q8 ? 2 * kTile * 4 : 0);
  static constexpr int kRun = (!Q8 && D == 128) ? 8 : D / 8;  // consecutive output dims of one thread
  // chunk permutations of a row so that the fragment reads of 8 lanes hit 8 different 16-byte banks
  __device__ static __forceinline__ int k_swz(int r) { return kChunks >= 8 ? (r & 1) << 2 : 0; }
  __device__ static __forceinline__ int v_swz(int r) {
    return kChunks >= 8 ? ((r >> 1) & 3) << 1 : (kChunks == 4 ? ((r >> 1) & 1) << 1 : 0);
  }
  // output dim of accumulator j, element e (0, 1) of the thread with t = lane % 4
  __device__ static __forceinline__ int out_dim(int j, int e, int t) {
    return 8 * kRun * (j / kRun) + kRun * (2 * t + e) + j % kRun;
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void cp16(void *dst, const void *src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp4(void *dst, const void *src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <bool F16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The f16 values of two bytes of (codes ^ 0x80): bytes 0x64 above them make 1024 + byte, less 1152 the code, exactly.
__device__ __forceinline__ uint32_t codes_f16(uint32_t biased, uint32_t select) {
  uint32_t r;
  const uint32_t pasted = __byte_perm(biased, 0x64646464u, select);
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(pasted), "r"(0x64806480u));
  return r;
}

// The bf16 values of two codes: 0x43 above a byte is 128 + its low seven bits, doubled scale if the sign bit is set; the
// two parts of the byte apart are 128 + low bits and 128 or 256, and their difference is the code, exactly.
__device__ __forceinline__ uint32_t codes_bf16(uint32_t codes, uint32_t select) {
  uint32_t r;
  const uint32_t pasted = __byte_perm(codes, 0x43434343u, select);
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(pasted & 0xff7fff7fu), "r"(pasted & 0xff80ff80u));
  return r;
}

__device__ __forceinline__ int seq_len(const Params &p, int i) {
  const int64_t pos = p.position[i];
  if (pos < -1 || pos >= p.own.cap) {
    set_device_error(EGPT_ERR_SHAPE);
    return 0;
  }
  return (int)(pos + 1);
}

// cum[i] = tiles of the sequences before i (one kv head); every thread of the CTA (kThreads) calls it.
template <int TILE>
__device__ Layout make_layout(const Params &p, int *cum, int *scratch) {
  constexpr int kPer = kMaxBatch / kThreads;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  int tiles[kPer], sum = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int i = t * kPer + e;
    tiles[e] = i < p.m ? (seq_len(p, i) + TILE - 1) / TILE : 0;
    sum += tiles[e];
  }
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) scratch[warp] = inc;
  __syncthreads();
  int before = inc - sum;
  for (int w = 0; w < warp; ++w) before += scratch[w];
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    if (t * kPer + e <= p.m) cum[t * kPer + e] = before;
    before += tiles[e];
  }
  if (t == kThreads - 1) cum[kMaxBatch] = before;
  __syncthreads();
  Layout l;
  l.prefix_tiles = (int)((p.prefix + TILE - 1) / TILE);
  l.prefix_segs = l.prefix_tiles ? p.nkv * p.row_tiles : 0;
  l.prefix_end = l.prefix_segs * l.prefix_tiles;
  l.total = l.prefix_end + p.nkv * cum[p.m];
  l.chunk = max((l.total + (int)gridDim.x - 1) / (int)gridDim.x, kWarps);
  return l;
}
__device__ __forceinline__ Seg own_seg(const Params &p, const Layout &l, const int *cum, int i, int g) {
  Seg s;
  const int tiles = cum[i + 1] - cum[i];
  s.index = l.prefix_segs + i * p.nkv + g;
  s.start = l.prefix_end + p.nkv * cum[i] + g * tiles;
  s.end = s.start + tiles;
  s.seq = i, s.g = g, s.tile = 0;
  s.len = (int)p.position[i] + 1;
  return s;
}
__device__ __forceinline__ Seg prefix_seg(const Params &p, const Layout &l, int index) {
  Seg s;
  s.index = index;
  s.start = index * l.prefix_tiles, s.end = s.start + l.prefix_tiles;
  s.seq = -1, s.g = index / p.row_tiles, s.tile = index % p.row_tiles;
  s.len = (int)p.prefix;
  return s;
}
// The segment that holds tile x < total.
__device__ __forceinline__ Seg find_seg(const Params &p, const Layout &l, const int *cum, int x) {
  if (x < l.prefix_end) return prefix_seg(p, l, x / l.prefix_tiles);
  int lo = 0, hi = p.m - 1;  // the last sequence whose tiles start at or before x and that has any
  const int y = x - l.prefix_end;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.nkv * cum[mid] <= y) lo = mid;
    else hi = mid - 1;
  }
  const int tiles = cum[lo + 1] - cum[lo];
  return own_seg(p, l, cum, lo, (y - p.nkv * cum[lo]) / tiles);
}
// A partial record: kRows rows of (D accumulators), then kRows maxima and kRows sums.
template <int D>
__device__ __forceinline__ float *record(const Params &p, int index) {
  return p.ws + (int64_t)index * kRows * (D + 2);
}

template <int D, bool Q8, int NR, int STAGES>
struct Smem {
  uint8_t ring[kWarps][STAGES][Geo<D, Q8>::kStageBytes];
  float merge[2][NR / 8 * (D / 4 + 2)][32];  // two warps' accumulators, maxima and sums
  int cum[kMaxBatch + 1];
  int scratch[kWarps];
  int last;
};

// NR: query rows in use, 8 or 16. SHARED: segments of the prefix as well, and every (CTA, segment) pair leaves a record
// for combine_kernel; else one CTA's segment goes straight to the output and the last CTA of a split one combines it.
template <int D, bool Q8, int NR, bool SHARED, int STAGES>
__global__ void __launch_bounds__(kThreads) attn_kernel(const Params p) {
  using G = Geo<D, Q8>;
  using S = Smem<D, Q8, NR, STAGES>;
  constexpr int TILE = G::kTile, NT = TILE / 8, ND = D / 8, NC = NR == 16 ? 4 : 2;  // NC: accumulators kept
  extern __shared__ __align__(16) uint8_t smem_raw[];
  S &sm = *(S *)smem_raw;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  pdl_wait();
  pdl_launch_dependents();
  const Layout lay = make_layout<TILE>(p, sm.cum, sm.scratch);

  if (!SHARED)  // sequences without keys
    for (int i = blockIdx.x; i < p.m; i += gridDim.x)
      if (sm.cum[i + 1] == sm.cum[i])
        for (int e = threadIdx.x; e < p.nkv * p.group * D; e += kThreads) p.out[i * p.ldo + e] = 0;

  const int x0 = (int)min((int64_t)lay.total, (int64_t)blockIdx.x * lay.chunk);
  const int x1 = (int)min((int64_t)lay.total, (int64_t)x0 + lay.chunk);
  if (x0 >= x1) return;

  // ---- this warp's loads: every fourth tile of the range, STAGES - 1 tiles ahead
  int lx = x0 + warp, lcount = 0;
  Seg ls = find_seg(p, lay, sm.cum, min(lx, x1 - 1));
  auto load_next = [&]() {
    if (lx < x1) {
      if (lx >= ls.end) ls = find_seg(p, lay, sm.cum, lx);
      uint8_t *st = sm.ring[warp][lcount % STAGES];
      const bool shared = SHARED && ls.seq < 0;
      const Cache &c = shared ? p.shared : p.own;
      const int64_t head = shared ? ls.g : (int64_t)ls.seq * p.nkv + ls.g;
      const int key0 = (lx - ls.start) * TILE;
      const int64_t row0 = head * c.cap + key0;
      const uint8_t *kb = c.k + row0 * G::kRowBytes, *vb = c.v + row0 * G::kRowBytes;
#pragma unroll
      for (int it = 0; it < TILE * G::kChunks / 32; ++it) {
        const int i = it * 32 + lane, r = i / G::kChunks, ch = i % G::kChunks;
        const bool in = key0 + r < ls.len;
        const int64_t off = in ? (int64_t)r * G::kRowBytes + ch * 16 : 0;
        cp16(st + r * G::kRowBytes + ((ch ^ G::k_swz(r)) * 16), kb + off, in ? 16 : 0);
        cp16(st + TILE * G::kRowBytes + r * G::kRowBytes + ((ch ^ G::v_swz(r)) * 16), vb + off, in ? 16 : 0);
      }
      if (Q8) {
        const bool in = lane < TILE && key0 + lane < ls.len;
        float *sc = (float *)(st + 2 * TILE * G::kRowBytes);
        cp4(sc + lane, c.ks + row0 + (in ? lane : 0), in ? 4 : 0);
        cp4(sc + TILE + lane, c.vs + row0 + (in ? lane : 0), in ? 4 : 0);
      }
    }
    cp_commit();
    lx += kWarps;
    ++lcount;
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) load_next();

  int x = x0 + warp, ccount = 0;
  Seg seg = find_seg(p, lay, sm.cum, x0);
  const int first_seg = seg.index;
  for (;;) {
    // ---- the segment's query rows as MMA fragments: row r of the tile, dims d0 .. d0 + 3 of step w
    uint32_t qa[D / 16][4];
    float rowfac[2];  // scale log2(e), and for int8 the power of two that q was divided by
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int r = g + 8 * hh;
      int64_t tok = -1;
      int h = 0;
      if (SHARED && seg.seq < 0) {
        const int flat = seg.tile * kRows + r;
        if (flat < p.m * p.group) tok = flat / p.group, h = seg.g * p.group + flat % p.group;
      } else if (r < p.group) {
        tok = seg.seq, h = seg.g * p.group + r;
      }
      const bool live = tok >= 0 && 8 * hh < NR;
      const uint16_t *qr = p.q + (live ? tok * p.ldq + (int64_t)h * D : 0);
      uint2 w[D / 16];
      float amax = 0.f;
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        const int d0 = Q8 ? (D == 32 ? 8 * t + 4 * s : 16 * (t + 4 * (s / 4)) + 4 * (s % 4))
                          : 8 * (t + 4 * (s / 2)) + 4 * (s % 2);
        w[s] = live ? *(const uint2 *)(qr + d0) : make_uint2(0u, 0u);
        if (Q8)
          amax = fmaxf(amax, fmaxf(fmaxf(fabsf(bf16_lo(w[s].x)), fabsf(bf16_hi(w[s].x))),
                                   fmaxf(fabsf(bf16_lo(w[s].y)), fabsf(bf16_hi(w[s].y)))));
      }
      rowfac[hh] = p.scale_log2;
      if (Q8) {
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // 2^e <= amax < 2^(e + 1) becomes 2^14 <= . < 2^15: bf16's 8 bits stay exact in f16 for elements down to
        // 2^-28 of the row's largest. (The exponent is kept where both factors are normal numbers.)
        const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -112), 127);
        const float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
        rowfac[hh] *= __uint_as_float((uint32_t)(127 - 14 + e) << 23);
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
          qa[s][hh] = f16x2(bf16_lo(w[s].x) * up, bf16_hi(w[s].x) * up);
          qa[s][hh + 2] = f16x2(bf16_lo(w[s].y) * up, bf16_hi(w[s].y) * up);
        }
      } else {
#pragma unroll
        for (int s = 0; s < D / 16; ++s) qa[s][hh] = w[s].x, qa[s][hh + 2] = w[s].y;
      }
    }
    float m_run[2] = {-INFINITY, -INFINITY}, l_part[2] = {0.f, 0.f};
    float acc[ND][4];
#pragma unroll
    for (int j = 0; j < ND; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;

    const int seg_end = min(seg.end, x1);
    for (; x < seg_end; x += kWarps, ++ccount) {
      load_next();
      cp_wait<STAGES - 1>();
      __syncwarp();
      const uint8_t *kt = sm.ring[warp][ccount % STAGES];
      const uint8_t *vt = kt + TILE * G::kRowBytes;
      const float *ksc = (const float *)(vt + TILE * G::kRowBytes), *vsc = ksc + TILE;
      const int left = seg.len - (x - seg.start) * TILE;  // keys from the tile's first to the segment's end

      // ---- scores: n-tile nt holds keys 8 nt .. 8 nt + 7 (this thread loads key 8 nt + g)
      float sc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
        const int r = 8 * nt + g;
        const uint8_t *row = kt + r * G::kRowBytes;
        constexpr int NW = G::kRowBytes / 16;  // words of the row that this thread takes
        uint32_t kw[NW];
        if constexpr (Q8 && D == 32) {
          const uint2 a = *(const uint2 *)(row + 8 * t);
          kw[0] = a.x, kw[1] = a.y;
        } else {
#pragma unroll
          for (int c = 0; c < NW / 4; ++c) {
            const uint4 a = *(const uint4 *)(row + (((t + 4 * c) ^ G::k_swz(r)) * 16));
            kw[4 * c] = a.x, kw[4 * c + 1] = a.y, kw[4 * c + 2] = a.z, kw[4 * c + 3] = a.w;
          }
        }
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
          if (Q8) {
            const uint32_t b = kw[s] ^ 0x80808080u;
            mma<true>(sc[nt], qa[s], codes_f16(b, 0x4140), codes_f16(b, 0x4342));
          } else {
            mma<false>(sc[nt], qa[s], kw[(2 * s) % NW], kw[(2 * s + 1) % NW]);
          }
        }
      }
      // ---- softmax: this thread has rows g, g + 8 of keys 8 nt + 2t, 8 nt + 2t + 1
      float mx[2] = {-INFINITY, -INFINITY};
      float vs[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = 8 * nt + 2 * t + e;
          const bool in = key < left;
          const float kf = Q8 ? ksc[key] : 1.f;
          vs[nt][e] = Q8 && in ? vsc[key] : 0.f;
#pragma unroll
          for (int hh = 0; hh < NR / 8; ++hh) {
            float &v = sc[nt][2 * hh + e];
            v = in ? v * (rowfac[hh] * kf) : -INFINITY;
            mx[hh] = fmaxf(mx[hh], v);
          }
        }
      }
      float ms[2], alpha[2] = {1.f, 1.f};
#pragma unroll
      for (int hh = 0; hh < NR / 8; ++hh) {
        mx[hh] = fmaxf(mx[hh], __shfl_xor_sync(0xffffffffu, mx[hh], 1));
        mx[hh] = fmaxf(mx[hh], __shfl_xor_sync(0xffffffffu, mx[hh], 2));
        const float m_new = fmaxf(m_run[hh], mx[hh]);
        ms[hh] = m_new == -INFINITY ? 0.f : m_new;
        alpha[hh] = ex2(m_run[hh] - ms[hh]);
        m_run[hh] = m_new;
        l_part[hh] *= alpha[hh];
      }
      // weights as sums of two bf16 values: pa the first (NR 8: the second in rows 8 .. 15), pb the second (NR 16)
      uint32_t pa[NT / 2][4], pb[NR == 16 ? NT / 2 : 1][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int hh = 0; hh < NR / 8; ++hh) {
          float p0 = ex2(sc[nt][2 * hh] - ms[hh]), p1 = ex2(sc[nt][2 * hh + 1] - ms[hh]);
          l_part[hh] += p0 + p1;
          if (Q8) p0 *= vs[nt][0], p1 *= vs[nt][1];
          const uint32_t hi = bf16x2(p0, p1), lo = bf16x2(p0 - bf16_lo(hi), p1 - bf16_hi(hi));
          pa[nt / 2][2 * (nt % 2) + hh] = hi;
          if (NR == 16) pb[nt / 2][2 * (nt % 2) + hh] = lo;
          else pa[nt / 2][2 * (nt % 2) + 1] = lo;
        }
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int j = 0; j < ND; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[j][c] *= alpha[NR == 16 ? c / 2 : 0];
      }
      // ---- P.V: step u takes keys 16 u .. 16 u + 15; this thread's pairs are keys 2t, 2t + 1 and 2t + 8, 2t + 9 of them
#pragma unroll
      for (int u = 0; u < NT / 2; ++u) {
        constexpr int NW = G::kRowBytes / 32;  // words of a row that this thread takes
        uint32_t vw[4][NW];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 16 * u + 2 * t + (i & 1) + 8 * (i >> 1);
          const uint8_t *row = vt + r * G::kRowBytes;
          if constexpr (NW == 1) {
            vw[i][0] = *(const uint32_t *)(row + 4 * g);
          } else if constexpr (NW == 2) {
            const uint2 a = *(const uint2 *)(row + (((g >> 1) ^ G::v_swz(r)) * 16) + 8 * (g & 1));
            vw[i][0] = a.x, vw[i][1] = a.y;
          } else {
#pragma unroll
            for (int c = 0; c < NW / 4; ++c) {
              const uint4 a = *(const uint4 *)(row + (((g + 8 * c) ^ G::v_swz(r)) * 16));
              vw[i][4 * c] = a.x, vw[i][4 * c + 1] = a.y, vw[i][4 * c + 2] = a.z, vw[i][4 * c + 3] = a.w;
            }
          }
        }
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          if (Q8) {  // four dims of two key pairs: interleave the pair's bytes, then widen two at a time
            const uint32_t pair[2][2] = {{__byte_perm(vw[0][w], vw[1][w], 0x5140), __byte_perm(vw[0][w], vw[1][w], 0x7362)},
                                         {__byte_perm(vw[2][w], vw[3][w], 0x5140), __byte_perm(vw[2][w], vw[3][w], 0x7362)}};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t select = e & 1 ? 0x4342 : 0x4140;
              const uint32_t b0 = codes_bf16(pair[0][e / 2], select), b1 = codes_bf16(pair[1][e / 2], select);
              mma<false>(acc[4 * w + e], pa[u], b0, b1);
              if (NR == 16) mma<false>(acc[4 * w + e], pb[u % (NR == 16 ? NT / 2 : 1)], b0, b1);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t select = e ? 0x7632 : 0x5410;
              const uint32_t b0 = __byte_perm(vw[0][w], vw[1][w], select), b1 = __byte_perm(vw[2][w], vw[3][w], select);
              mma<false>(acc[(2 * w + e) % ND], pa[u], b0, b1);
              if (NR == 16) mma<false>(acc[(2 * w + e) % ND], pb[u % (NR == 16 ? NT / 2 : 1)], b0, b1);
            }
          }
        }
      }
      __syncwarp();  // the stage is read before the load that reuses it
    }

    if (NR == 8) {  // the two parts of the weights
#pragma unroll
      for (int j = 0; j < ND; ++j) acc[j][0] += acc[j][2], acc[j][1] += acc[j][3];
    }
    // ---- the segment is done: the four warps' states meet in warp 0 (2, 3 -> 0, 1, then 1 -> 0)
#pragma unroll
    for (int hh = 0; hh < NR / 8; ++hh) {
      l_part[hh] += __shfl_xor_sync(0xffffffffu, l_part[hh], 1);
      l_part[hh] += __shfl_xor_sync(0xffffffffu, l_part[hh], 2);
    }
#pragma unroll
    for (int half = kWarps / 2; half >= 1; half >>= 1) {
      __syncthreads();  // the buffer's last readers are done
      if (warp >= half && warp < 2 * half) {
        float(*b)[32] = sm.merge[warp - half];
#pragma unroll
        for (int j = 0; j < ND; ++j)
#pragma unroll
          for (int c = 0; c < NC; ++c) b[j * NC + c][lane] = acc[j][c];
#pragma unroll
        for (int hh = 0; hh < NR / 8; ++hh) b[ND * NC + 2 * hh][lane] = m_run[hh], b[ND * NC + 2 * hh + 1][lane] = l_part[hh];
      }
      __syncthreads();
      if (warp < half) {
        float(*b)[32] = sm.merge[warp];
        float fa[2], fb[2];
#pragma unroll
        for (int hh = 0; hh < NR / 8; ++hh) {
          const float mo = b[ND * NC + 2 * hh][lane], m_new = fmaxf(m_run[hh], mo);
          const float mz = m_new == -INFINITY ? 0.f : m_new;
          fa[hh] = ex2(m_run[hh] - mz), fb[hh] = ex2(mo - mz);
          m_run[hh] = m_new;
          l_part[hh] = l_part[hh] * fa[hh] + b[ND * NC + 2 * hh + 1][lane] * fb[hh];
        }
#pragma unroll
        for (int j = 0; j < ND; ++j)
#pragma unroll
          for (int c = 0; c < NC; ++c) acc[j][c] = acc[j][c] * fa[c / 2] + b[j * NC + c][lane] * fb[c / 2];
      }
    }
    const bool whole = !SHARED && seg.start >= x0 && seg.end <= x1;
    if (warp == 0) {
      if (whole) {
#pragma unroll
        for (int hh = 0; hh < NR / 8; ++hh) {
          const int r = g + 8 * hh;
          if (r < p.group) {
            const float inv = 1.f / l_part[hh];
            uint16_t *dst = p.out + seg.seq * p.ldo + (int64_t)(seg.g * p.group + r) * D;
#pragma unroll
            for (int j = 0; j < ND; j += 4)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int c = 2 * hh + e;
                *(uint2 *)(dst + G::out_dim(j, e, t)) = make_uint2(bf16x2(acc[j][c] * inv, acc[j + 1][c] * inv),
                                                                   bf16x2(acc[j + 2][c] * inv, acc[j + 3][c] * inv));
              }
          }
        }
      } else {
        float *rec = record<D>(p, SHARED ? (int)blockIdx.x + seg.index : 2 * (int)blockIdx.x + (seg.index != first_seg));
        const int rows = (SHARED && seg.seq < 0) ? kRows : p.group;
#pragma unroll
        for (int hh = 0; hh < NR / 8; ++hh) {
          const int r = g + 8 * hh;
          if (r < rows) {
#pragma unroll
            for (int j = 0; j < ND; j += 4)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int c = 2 * hh + e;
                *(float4 *)(rec + r * D + G::out_dim(j, e, t)) = make_float4(acc[j][c], acc[j + 1][c], acc[j + 2][c], acc[j + 3][c]);
              }
            if (t == 0) rec[kRows * D + r] = m_run[hh], rec[kRows * D + kRows + r] = l_part[hh];
          }
        }
      }
    }
    if (!SHARED && !whole) {
      // the last CTA of a segment that several share adds their records up
      const int c0 = seg.start / lay.chunk, c1 = (seg.end - 1) / lay.chunk;
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        unsigned *cnt = p.cnt + seg.index;
        const bool last = atomicAdd(cnt, 1u) == (unsigned)(c1 - c0);
        if (last) *cnt = 0u;
        sm.last = last;
      }
      __syncthreads();
      if (sm.last) {
        __threadfence();
        for (int e = threadIdx.x; e < p.group * D; e += kThreads) {
          const int r = e / D, dd = e - r * D;
          float M = -INFINITY, lsum = 0.f, a = 0.f;
          for (int c = c0; c <= c1; ++c) {
            const float *rec = record<D>(p, 2 * c + (c == c0 && seg.start != c0 * lay.chunk));
            const float mc = __ldcg(rec + kRows * D + r);
            const float lc = __ldcg(rec + kRows * D + kRows + r), ac = __ldcg(rec + r * D + dd);
            const float m_new = fmaxf(M, mc), mz = m_new == -INFINITY ? 0.f : m_new;
            const float fo = ex2(M - mz), fc = ex2(mc - mz);
            M = m_new;
            lsum = lsum * fo + lc * fc;
            a = a * fo + ac * fc;
          }
          p.out[seg.seq * p.ldo + (int64_t)(seg.g * p.group + r) * D + dd] = f32_to_bf16_bits(a / lsum);
        }
      }
    }
    if (seg.end >= x1) break;
    seg = find_seg(p, lay, sm.cum, seg.end);
  }
  cp_wait<0>();
}

// One (sequence, head) row per warp: its records of the prefix's and of its own segment, added up.
template <int D, int TILE>
__global__ void __launch_bounds__(kThreads) combine_kernel(const Params p, int grid) {
  __shared__ int cum[kMaxBatch + 1];
  __shared__ int scratch[kWarps];
  constexpr int N = D / 32;
  pdl_wait();
  pdl_launch_dependents();
  Layout lay = make_layout<TILE>(p, cum, scratch);
  lay.chunk = max((lay.total + grid - 1) / grid, kWarps);  // as the attention kernel's grid cut it
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x * kWarps + warp;
  const int nq = p.nkv * p.group;
  if (row >= p.m * nq) return;
  const int i = row / nq, h = row - i * nq, g = h / p.group, j = h - g * p.group;
  float M = -INFINITY, lsum = 0.f, a[N];
#pragma unroll
  for (int e = 0; e < N; ++e) a[e] = 0.f;
  auto add_record = [&](const float *rec, int rows, int r) {
    const float mc = __ldcg(rec + rows * D + r), lc = __ldcg(rec + rows * D + rows + r);
    if (lc == 0.f) return;  // no keys: nothing was accumulated
    const float m_new = fmaxf(M, mc), mz = m_new == -INFINITY ? 0.f : m_new;
    const float fo = ex2(M - mz), fc = ex2(mc - mz);
    M = m_new;
    lsum = lsum * fo + lc * fc;
#pragma unroll
    for (int e = 0; e < N; ++e) a[e] = a[e] * fo + __ldcg(rec + r * D + lane + 32 * e) * fc;
  };
  auto add = [&](const Seg &s, int r) {
    if (s.start >= s.end) return;
    for (int c = s.start / lay.chunk; c <= (s.end - 1) / lay.chunk; ++c) add_record(record<D>(p, c + s.index), kRows, r);
  };
  if (D == apx::kD && p.pre) {
    const int tile = i / p.pre_seqs, pair = tile / 2;
    const bool two = 2 * pair + 1 < p.pre_tiles;  // the pair's streams are two tiles, or both this one
    const float *rec = p.pre + (int64_t)(g * p.pre_pairs + pair) * p.pre_ranges * 2 * apx::kRecord;
    for (int c = 0; c < 2 * p.pre_ranges; ++c)
      if (!two || (c & 1) == (tile & 1))
        add_record(rec + (int64_t)c * apx::kRecord, apx::kRowsT, (i % p.pre_seqs) * p.group + j);
  }
  if (lay.prefix_segs) {
    const int flat = i * p.group + j;
    add(prefix_seg(p, lay, g * p.row_tiles + flat / kRows), flat % kRows);
  }
  add(own_seg(p, lay, cum, i, g), j);
  const float inv = lsum == 0.f ? 0.f : 1.f / lsum;  // no keys at all: zeros
#pragma unroll
  for (int e = 0; e < N; ++e) p.out[i * p.ldo + (int64_t)h * D + lane + 32 * e] = f32_to_bf16_bits(a[e] * inv);
}

template <int D, bool Q8, int NR, bool SHARED>
static cudaError_t launch(const Params &p, cudaStream_t st, bool pdl) {
  constexpr int kStages = NR == 16 ? 2 : 3;
  auto fn = attn_kernel<D, Q8, NR, SHARED, kStages>;
  const size_t smem = sizeof(Smem<D, Q8, NR, kStages>);
  static int configured[64] = {0};  // the shared-memory opt-in, per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    configured[dev] = 1;
  }
  const int grid = 2 * num_sms();
  const cudaError_t e = launch_kernel((const void *)fn, dim3(grid), dim3(kThreads), smem, st, pdl, p);
  if (e != cudaSuccess || !SHARED) return e;
  const unsigned rows = (unsigned)(p.m * p.nkv * p.group);
  return launch_kernel((const void *)combine_kernel<D, Geo<D, Q8>::kTile>, dim3((rows + kWarps - 1) / kWarps),
                       dim3(kThreads), 0, st, true, p, grid);
}
template <bool Q8, int NR, bool SHARED>
static cudaError_t launch_d(const Params &p, int d, cudaStream_t st, bool pdl) {
  return d == 128 ? launch<128, Q8, NR, SHARED>(p, st, pdl)
                  : (d == 64 ? launch<64, Q8, NR, SHARED>(p, st, pdl) : launch<32, Q8, NR, SHARED>(p, st, pdl));
}

// Whether the prefix goes to attn_prefix_kernel: bf16, head_dim 128, more rows than one tile of the mma.sync kernel.
static bool prefix_on_tcgen05(const Params &p, int d, bool q8) {
  return !q8 && d == apx::kD && p.prefix > 0 && p.scale_log2 > 0.f && p.m * p.group > kRows;
}
static int row_tiles(int64_t m, int group) { return (int)((m * group + kRows - 1) / kRows); }
static size_t counter_bytes(int64_t m, int nkv) { return ((size_t)m * nkv * 4 + 255) / 256 * 256; }

static int check(const char *what, int64_t ldo, int64_t ldq, const void *out, const void *q, int64_t cap, int64_t m,
                 int nq, int nkv, int d, float scale, const void *ws, size_t ws_bytes) {
  if (d != 32 && d != 64 && d != 128) return set_error(EGPT_ERR_SHAPE, "%s: head_dim must be 32, 64 or 128", what);
  if (nq < 1 || nkv < 1 || nq % nkv || nq / nkv > kRows)
    return set_error(EGPT_ERR_SHAPE, "%s: nq must be a multiple of nkv, at most %d to one", what, kRows);
  if (m < 1 || m > kMaxBatch || cap < 1 || cap > 0x3fffffff || ldq < (int64_t)nq * d || ldo < (int64_t)nq * d)
    return set_error(EGPT_ERR_SHAPE, "%s: bad m (1 to %d), cap or leading dimension", what, kMaxBatch);
  if (m * nkv * ((cap + 15) / 16) > 0x3fffffff) return set_error(EGPT_ERR_SHAPE, "%s: cache too long for the batch", what);
  if (!(fabsf(scale) <= 3e38f)) return set_error(EGPT_ERR_ARG, "%s: scale must be finite", what);
  if ((uintptr_t)out % 16 || (uintptr_t)q % 16 || ldq % 8 || ldo % 8)
    return set_error(EGPT_ERR_ALIGN, "%s: q and out must be 16-byte aligned rows", what);
  if (!ws || ws_bytes < egpt_attn_q8_ws_bytes(m, nq, nkv, d))
    return set_error(EGPT_ERR_WORKSPACE, "%s: workspace too small", what);
  if ((uintptr_t)ws % 16) return set_error(EGPT_ERR_ALIGN, "%s: workspace must be 16-byte aligned", what);
  return EGPT_OK;
}

}  // namespace aq8
}  // namespace egpt

using namespace egpt;

extern "C" size_t egpt_attn_q8_ws_bytes(int64_t m, int nq, int nkv, int d) {
  if (m < 1 || nkv < 1 || nq < nkv || d < 1) return 0;
  // counters, then a record for every (CTA, segment) pair: CTA c and segment s keep theirs at c + s
  const size_t records = (size_t)2 * num_sms() + (size_t)nkv * aq8::row_tiles(m, nq / nkv) + (size_t)m * nkv;
  const size_t prefix = d == apx::kD && nq / nkv <= aq8::kRows ? apx::record_floats(m, nq / nkv, nkv) * 4 : 0;
  return aq8::counter_bytes(m, nkv) + std::max(records, (size_t)4 * num_sms()) * aq8::kRows * ((size_t)d + 2) * 4 + prefix;
}

extern "C" int egpt_attn_decode_q8(void *out, int64_t ldo, const void *q, int64_t ldq, const int8_t *k_cache,
                                   const float *k_scale, const int8_t *v_cache, const float *v_scale, int64_t cap,
                                   const int64_t *position, int64_t m, int nq, int nkv, int d, float scale, void *ws,
                                   size_t ws_bytes, unsigned flags, void *stream) {
  clear_error();
  if (!out || !q || !k_cache || !k_scale || !v_cache || !v_scale || !position)
    return set_error(EGPT_ERR_ARG, "attn_decode_q8: null pointer");
  if (int rc = aq8::check("attn_decode_q8", ldo, ldq, out, q, cap, m, nq, nkv, d, scale, ws, ws_bytes)) return rc;
  if ((uintptr_t)k_cache % 16 || (uintptr_t)v_cache % 16 || (uintptr_t)k_scale % 4 || (uintptr_t)v_scale % 4)
    return set_error(EGPT_ERR_ALIGN, "attn_decode_q8: caches must be 16-byte aligned");
  aq8::Params p{};
  p.out = (uint16_t *)out, p.ldo = ldo, p.q = (const uint16_t *)q, p.ldq = ldq;
  p.own = {(const uint8_t *)k_cache, (const uint8_t *)v_cache, k_scale, v_scale, cap};
  p.position = position, p.m = (int)m, p.nkv = nkv, p.group = nq / nkv, p.scale_log2 = scale * 1.4426950408889634f;
  p.cnt = (unsigned *)ws, p.ws = (float *)((char *)ws + aq8::counter_bytes(m, nkv));
  const bool pdl = (flags & EGPT_FLAG_PDL) != 0;
  return check_launch(p.group <= 8 ? aq8::launch_d<true, 8, false>(p, d, (cudaStream_t)stream, pdl)
                                   : aq8::launch_d<true, 16, false>(p, d, (cudaStream_t)stream, pdl),
                      "attn_decode_q8_kernel");
}

extern "C" int egpt_attn_shared_prefix(void *out, int64_t ldo, const void *q, int64_t ldq, const void *pk,
                                       const float *pk_scale, const void *pv, const float *pv_scale, int64_t prefix_cap,
                                       int64_t prefix_len, const void *tk, const float *tk_scale, const void *tv,
                                       const float *tv_scale, int64_t cap, const int64_t *position, int64_t m, int nq,
                                       int nkv, int d, float scale, int cache_dtype, void *ws, size_t ws_bytes,
                                       unsigned flags, void *stream) {
  clear_error();
  if (!out || !q || !pk || !pv || !tk || !tv || !position) return set_error(EGPT_ERR_ARG, "attn_shared_prefix: null pointer");
  if (cache_dtype != EGPT_I8 && cache_dtype != EGPT_BF16)
    return set_error(EGPT_ERR_DTYPE, "attn_shared_prefix: caches are int8 or bf16");
  const bool q8 = cache_dtype == EGPT_I8;
  if (q8 && (!pk_scale || !pv_scale || !tk_scale || !tv_scale))
    return set_error(EGPT_ERR_ARG, "attn_shared_prefix: int8 caches need their scales");
  if (int rc = aq8::check("attn_shared_prefix", ldo, ldq, out, q, cap, m, nq, nkv, d, scale, ws, ws_bytes)) return rc;
  if (prefix_cap < 1 || prefix_len < 0 || prefix_len > prefix_cap ||
      (int64_t)nkv * (aq8::row_tiles(m, nq / nkv) * ((prefix_len + 15) / 16) + m * ((cap + 15) / 16)) > 0x3fffffff)
    return set_error(EGPT_ERR_SHAPE, "attn_shared_prefix: bad prefix_len (0 to prefix_cap) or caches too long");
  if ((uintptr_t)pk % 16 || (uintptr_t)pv % 16 || (uintptr_t)tk % 16 || (uintptr_t)tv % 16)
    return set_error(EGPT_ERR_ALIGN, "attn_shared_prefix: caches must be 16-byte aligned");
  aq8::Params p{};
  p.out = (uint16_t *)out, p.ldo = ldo, p.q = (const uint16_t *)q, p.ldq = ldq;
  p.own = {(const uint8_t *)tk, (const uint8_t *)tv, tk_scale, tv_scale, cap};
  p.shared = {(const uint8_t *)pk, (const uint8_t *)pv, pk_scale, pv_scale, prefix_cap};
  p.prefix = prefix_len, p.position = position, p.m = (int)m, p.nkv = nkv, p.group = nq / nkv;
  p.row_tiles = aq8::row_tiles(m, p.group), p.scale_log2 = scale * 1.4426950408889634f;
  p.cnt = (unsigned *)ws, p.ws = (float *)((char *)ws + aq8::counter_bytes(m, nkv));
  const bool pdl = (flags & EGPT_FLAG_PDL) != 0;
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (aq8::prefix_on_tcgen05(p, d, q8)) {
    apx::Args A{};
    const apx::Shape sh = apx::shape_of(m, p.group, nkv, prefix_len);
    // its records lie behind those of the tails
    const size_t head = egpt_attn_q8_ws_bytes(m, nq, nkv, d) - apx::record_floats(m, p.group, nkv) * 4;
    A.ws = (float *)((char *)ws + head);
    A.prefix = prefix_len, A.m = (int)m, A.nkv = nkv, A.group = p.group, A.scale_log2 = p.scale_log2;
    bool maps_ok = false;
    e = apx::launch(A, q, ldq, pk, pv, prefix_cap, sh, st, pdl, maps_ok);
    if (!maps_ok) return set_error(EGPT_ERR_ALIGN, "attn_shared_prefix: tensor maps rejected");
    if (e != cudaSuccess) return check_launch(e, "attn_prefix_kernel");
    p.pre = A.ws, p.pre_seqs = sh.seqs, p.pre_tiles = sh.tiles, p.pre_pairs = sh.pairs, p.pre_ranges = sh.ranges;
    p.prefix = 0;  // what is left in the flat list are the tails
    e = p.group <= 8 ? aq8::launch<128, false, 8, true>(p, st, true) : aq8::launch<128, false, 16, true>(p, st, true);
    return check_launch(e, "attn_shared_prefix_kernel");
  }
  if (m * p.group <= 8) e = q8 ? aq8::launch_d<true, 8, true>(p, d, st, pdl) : aq8::launch_d<false, 8, true>(p, d, st, pdl);
  else e = q8 ? aq8::launch_d<true, 16, true>(p, d, st, pdl) : aq8::launch_d<false, 16, true>(p, d, st, pdl);
  return check_launch(e, "attn_shared_prefix_kernel");
}
