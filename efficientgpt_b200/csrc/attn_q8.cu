// Decode attention of a batch over int8 KV caches, and over a prefix that the whole batch shares (int8 or bf16).
//
//   egpt_attn_decode_q8:      out[i, h] = sum_j w_j V[j] / sum_j w_j,  w_j = 2^(scale log2(e) q[i, h] . K[j]),
//                             over the L_i = position[i] + 1 keys of sequence i's own cache;
//   egpt_attn_shared_prefix:  the same over prefix_len keys held once and then sequence i's own L_i keys (its tail).
// K[j] = ks_j kq_j and V[j] = vs_j vq_j for int8 codes kq, vq with one scale per row and head (kv_q8.cu). GQA: head h
// reads kv head h / group. A row without any key, or whose scores are all -inf, gives zeros.
//
// Work: a segment is one cache head with the query rows that read it: (i, g) with the group's rows for a sequence's
// own cache, (g, 16 query rows) for the shared prefix, whose rows are all (sequence, head) pairs of kv head g in a
// row. A segment's keys are cut into tiles of kTile keys and the tiles of a launch into contiguous ranges, one per CTA,
// on the device, so no length is known to the host. Where the segments allow it ranges are parts of one segment each
// (split by the smallest range length that gives every CTA at most one); else they are equal stretches of the flat
// list of all tiles and may hold several segments (each counted with kExtra tiles more, about what its start and
// end cost), cut inside a segment only if that is a long one, so that neither many short sequences nor one token
// next to a document leave CTAs idle. Many segments of a few tiles each go to the warps whole, which then have
// nothing to add up (make_layout weighs it). Of a segment's part a warp takes every kWarps-th tile, through a ring
// of its own in shared memory (cp.async, rows past the segment's end filled with zeros), running ahead into the
// next segment; warps only meet at a segment's end.
//
// A prefix and the sequences' own keys behind it leave partial records: from one launch, in which the prefix's CTAs come
// first (4 rows behind 512 bf16 keys a call 15.7 us, 19.5 with a launch for each), or, where attn_prefix.cu takes
// the prefix, from its launch and a dependent one: on the SMs that the prefix leaves free where those are at least half
// (a short prefix), else as its CTAs end. A last launch adds both up, a warp to a row.
//
// Arithmetic: mma.sync with the query rows as M. Scores of int8 keys, up to 8 rows: q as fixed point X 2^(e - 29),
// |X| <= 2^30, in four balanced base-256 digits, two of them in the MMA's rows 0-7 and 8-15, so two int8 MMAs per 32
// dims give the exact dot products with the codes as they lie in memory, and ks_j multiplies their fp32 value. 16
// rows: the codes become f16 exactly (0x6400 | (q + 128) is 1152 + q), and q, scaled by a power of two per row to at
// most 2^15, too, so the sums are those of the codes in fp32. P.V is in bf16, whose exponents hold every weight times
// vs_j; its 8 bits would cost a weight 2^-9 of itself, so a weight enters as the sum of two bf16 values (16 bits).
// With 8 query rows or fewer the second values ride in the MMA's upper 8 rows, which are idle otherwise; 16 rows take
// a second MMA. Codes become bf16 exactly as (128 + low seven bits) - (128 + sign bit). Sums, maxima and
// accumulators are fp32; the output is rounded once.
//
// What bounds it: HBM for long contexts (the 8 warps' loops run at 5.3 TB/s, 81% of a measured copy: about 800
// instructions per 32-key tile, a third of them widening V), and for everything else the way in (positions, cuts, first
// tile: 3 us) and out (the warps' merge, and for split segments the fence, the arrival and the other CTAs' records: 5 us
// with 18 of those), whose parts have not been timed apart. Measured, d = 128, 8 kv heads, a call on the device: one row
// of 16 heads over 512 / 2048 / 8192 / 32768 keys 8.2 / 10.8 / 12.7 / 22.1 us (32768: 69.2 MB, 3.1 TB/s); 16 rows of
// 32 heads over 1 to 8191 keys 24 us; 64 rows over 32 to 512 keys 22 us. Tried: f16 weights (fewer instructions, but weights below 2^-29 of a row's
// largest vanish), 16 warps with 16-key tiles (one row over 32768 keys 28.4 us for 24.1 then), adding up in every CTA
// behind a prefix instead of in a launch for it (64 rows over 32768 shared keys 81 us for 66).
#include <cmath>

#include "internal.h"
#include "common.cuh"

namespace egpt {
namespace aq8 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxBatch = 512;
constexpr int kRows = 16;        // query rows per tile (the M of the MMA), and rows of a partial record
constexpr int kMinKeys = 512;    // keys of a range at least
constexpr int kExtraKeys = 512;  // what a segment's start and end cost, in keys

struct Cache {
  const uint8_t *k, *v;
  const float *ks, *vs;  // null: bf16 rows
  int64_t cap;
};

// The prefix's partial records, by the kernel that made them.
struct Prefix {
  const float *rec;                // null: no prefix
  int grid;                        // its CTAs
  int big;                         // 1: attn_prefix_kernel's
  int seqs, pairs, ranges;         // its shape
  int row_tiles, pad, chunk, seg_tiles;  // else the list of prefix segments, cut as below
};

struct Params {
  uint16_t *out;
  const uint16_t *q;
  int64_t ldo, ldq;
  Cache cache;
  const int64_t *position;
  int m, nkv, group;
  int head_share;  // CTAs per kv head
  float scale_log2;
  float *ws;      // partial records of this launch
  unsigned *cnt;  // arrivals at a split segment, by the first CTA of it; zero between calls
  int2 *parts;    // beside a prefix: first record and records of each (sequence, kv head)
  int keys;       // keys of the shared prefix (as its own segments' params)
  Prefix pre;     // the prefix's records to add up and how its segments are cut
};

// How the tiles of the launch are cut: a CTA takes `chunk` places of the flat list of segments.
struct Layout {
  int total, chunk;
  int pad;    // > 1: a segment takes up a multiple of pad (= chunk) places and every range lies in one segment
  int uncut;  // else equal stretches, and the tiles up to which a segment is not split
  bool solo;  // no ranges: every warp takes whole segments of its own
};
struct Seg {
  int index, start, end, next;  // its number, its tiles in the flat list, and the place after it
  int seq, g, tile;       // sequence, kv head; row tile (prefix)
  int len;                // keys
};

// Shape of a CTA (one per SM) by type and query rows.
template <bool Q8, int NR>
struct Cfg {
  static constexpr int kWarps = 8;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kTile = Q8 ? 32 : 16;  // keys per warp tile: K and V 4 KB each at d = 128
  static constexpr int kStages = NR == 8 ? 3 : 2;
  static constexpr int kMinChunk = kMinKeys / kTile, kExtra = kExtraKeys / kTile;
};
template <int D, bool Q8, int NR>
struct Geo {
  static constexpr int kRowBytes = Q8 ? D : 2 * D;
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kTile = Cfg<Q8, NR>::kTile;
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

using apf::ex2;
using apx::widen2;

// A row's accumulators over their sum; a sum of zero (no key, or every score -inf) gives zeros.
__device__ __forceinline__ float inverse_sum(float sum) { return sum == 0.f ? 0.f : 1.f / sum; }
__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp16z(uint32_t dst, const void *src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void *src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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
__device__ __forceinline__ void mma_i8(int (&c)[4], const uint32_t *a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The f16 values of two bytes of (codes ^ 0x80): bytes 0x64 above them make 1024 + byte, less 1152 the code, exactly.
__device__ __forceinline__ uint32_t codes_f16(uint32_t biased, uint32_t select) {
  uint32_t r;
  const uint32_t pasted = __byte_perm(biased, 0x64646464u, select);
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(pasted), "r"(0x64806480u));
  return r;
}

__device__ __forceinline__ int seq_len(const Params &p, int i) {
  const int64_t pos = p.position[i];
  if (pos < -1 || pos >= p.cache.cap) {
    set_device_error(EGPT_ERR_SHAPE);
    return 0;
  }
  return (int)(pos + 1);
}

__host__ __device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }
// The same for 0 <= a, 0 < b, a + b <= 2^24, where a float quotient is off by one at most.
__device__ __forceinline__ int ceil_div_small(int a, int b) {
  const int n = a + b - 1;
  int q = (int)((float)n * __frcp_rn((float)b));
  const int r = n - q * b;
  return q + (r >= b) - (r < 0);
}

// cum[i] = places of the sequences before i (one kv head). The ranges: with up to 32 sequences the lanes try eight range
// lengths from the even share of the tiles to 1.5 times it, and the smallest that gives at most one range per CTA is taken;
// failing that, and for more sequences, equal stretches, or whole segments to single warps where that takes less time: a
// CTA's part of a segment costs about one round of its warps' tiles besides its rounds, a warp's half a tile besides
// its tiles, and the slowest warp has the longest segments. Every thread of the CTA calls it.
template <typename C>
__device__ __forceinline__ Layout make_layout(const Params &p, int grid, int *cum, int *len_of, int *scratch) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  Layout l;
  l.pad = 1, l.solo = false;
  int segs = 0, rounds = 0, longest = 0;  // segments, their rounds and most tiles, of one kv head
  if (p.m <= 32) {  // every warp for itself
    const int keys = lane < p.m ? seq_len(p, lane) : 0, tiles = ceil_div(keys, C::kTile);
    bool fits = true;
    if (p.m == 1 && p.head_share) {  // all CTAs of a head for its one segment
      l.pad = max(C::kMinChunk, ceil_div_small(__shfl_sync(0xffffffffu, tiles, 0), p.head_share));
    } else {
      // lane: length number lane % 8, every fourth sequence from lane / 8 on
      const int share = ceil_div(p.nkv * __reduce_add_sync(0xffffffffu, tiles), grid);
      const int least = max(C::kMinChunk, share), len = least + (least * (lane & 7) + 13) / 14;
      int parts = 0;
#pragma unroll 4
      for (int i = lane >> 3; i < ((p.m + 3) & ~3); i += 4)
        parts += ceil_div_small(__shfl_sync(0xffffffffu, tiles, i), len);
      parts += __shfl_xor_sync(0xffffffffu, parts, 8);
      parts += __shfl_xor_sync(0xffffffffu, parts, 16);
      const unsigned good = __ballot_sync(0xffffffffu, p.nkv * parts <= grid);
      fits = good != 0u;
      if (fits) l.pad = __shfl_sync(0xffffffffu, len, __ffs(good) - 1);
    }
    if (!fits) {
      segs = __popc(__ballot_sync(0xffffffffu, tiles > 0));
      rounds = __reduce_add_sync(0xffffffffu, ceil_div(tiles, C::kWarps));
      longest = __reduce_max_sync(0xffffffffu, tiles);
    }
    const int places = fits ? ceil_div_small(tiles, l.pad) * l.pad : (tiles ? tiles + C::kExtra : 0);
    int inc = places;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (warp == 0) {
      cum[lane] = inc - places, len_of[lane] = keys;
      if (lane == 31) cum[32] = inc;
    }
    __syncthreads();
  } else {
    constexpr int kPer = kMaxBatch / C::kThreads;
    int places[kPer], sum = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int i = t * kPer + e, keys = i < p.m ? seq_len(p, i) : 0, tiles = ceil_div(keys, C::kTile);
      len_of[i] = keys;
      places[e] = tiles ? tiles + C::kExtra : 0;
      sum += places[e];
      segs += tiles > 0, rounds += ceil_div(tiles, C::kWarps), longest = max(longest, tiles);
    }
    segs = __reduce_add_sync(0xffffffffu, segs), rounds = __reduce_add_sync(0xffffffffu, rounds);
    longest = __reduce_max_sync(0xffffffffu, longest);
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) {
      scratch[warp] = inc;
      scratch[C::kWarps + warp] = segs, scratch[2 * C::kWarps + warp] = rounds, scratch[3 * C::kWarps + warp] = longest;
    }
    __syncthreads();
    int before = inc - sum;
    for (int w = 0; w < warp; ++w) before += scratch[w];
    segs = rounds = longest = 0;
    for (int w = 0; w < C::kWarps; ++w) {
      segs += scratch[C::kWarps + w], rounds += scratch[2 * C::kWarps + w];
      longest = max(longest, scratch[3 * C::kWarps + w]);
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      cum[t * kPer + e] = before;
      before += places[e];
    }
    if (t == C::kThreads - 1) cum[kMaxBatch] = before;
    __syncthreads();
  }
  l.total = p.nkv * cum[p.m];
  l.chunk = l.pad > 1 ? l.pad : max(1, ceil_div(l.total, grid));
  l.uncut = max(C::kMinChunk, l.chunk / 2);
  if (l.pad == 1) {
    const float by_cta = (float)(p.nkv * (segs + rounds)) / (float)grid;
    l.solo = (float)ceil_div(p.nkv * segs, grid * C::kWarps) * (longest + 0.5f) < by_cta;
  }
  return l;
}
template <int TILE>
__device__ __forceinline__ Seg own_seg(const Params &p, const int *cum, const int *len_of, int i, int g) {
  Seg s;
  const int places = cum[i + 1] - cum[i];
  s.seq = i, s.g = g, s.tile = 0;
  s.index = i * p.nkv + g;
  s.start = p.nkv * cum[i] + g * places, s.next = s.start + places;
  s.len = len_of[i];
  s.end = s.start + ceil_div(s.len, TILE);
  return s;
}
__device__ __forceinline__ Seg prefix_seg(const Params &p, int index) {
  Seg s;
  const int places = ceil_div(p.pre.seg_tiles, p.pre.pad) * p.pre.pad;
  s.index = index;
  s.start = index * places, s.end = s.start + p.pre.seg_tiles, s.next = s.start + places;
  s.seq = -1, s.g = index / p.pre.row_tiles, s.tile = index % p.pre.row_tiles;
  s.len = p.keys;
  return s;
}
// The segment that holds place x < total.
template <int TILE, bool PREFIX>
__device__ __forceinline__ Seg find_seg(const Params &p, const int *cum, const int *len_of, int x) {
  if (PREFIX) return prefix_seg(p, x / (ceil_div(p.pre.seg_tiles, p.pre.pad) * p.pre.pad));
  int lo = 0, hi = p.m - 1;  // the last sequence whose places start at or before x: it has some
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.nkv * cum[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return own_seg<TILE>(p, cum, len_of, lo, (x - p.nkv * cum[lo]) / (cum[lo + 1] - cum[lo]));
}
// The segment after s, whose next is < total.
template <int TILE, bool PREFIX>
__device__ __forceinline__ Seg next_seg(const Params &p, const int *cum, const int *len_of, const Seg &s) {
  if (PREFIX) return prefix_seg(p, s.index + 1);
  if (s.g + 1 < p.nkv) {
    Seg r = s;
    const int places = s.next - s.start;
    ++r.g, ++r.index, r.start += places, r.end += places, r.next += places;
    return r;
  }
  int i = s.seq + 1;
  while (cum[i + 1] == cum[i]) ++i;
  return own_seg<TILE>(p, cum, len_of, i, 0);
}
// Where a stretch whose even cut is place x begins: not past the tiles of a segment, nor inside a short one.
template <int TILE, bool PREFIX>
__device__ __noinline__ int cut_at(const Params &p, const Layout &l, const int *cum, const int *len_of, int64_t x) {
  if (x >= l.total) return l.total;
  const Seg s = find_seg<TILE, PREFIX>(p, cum, len_of, (int)x);
  return x >= s.end || (x > s.start && s.end - s.start <= l.uncut) ? s.next : (int)x;
}
// A partial record: kRows rows of (D accumulators), then kRows maxima and kRows sums.
template <int D>
__device__ __forceinline__ float *record(const Params &p, int index) {
  return p.ws + (int64_t)index * kRows * (D + 2);
}

template <int D, bool Q8, int NR>
struct Smem {
  static constexpr int kWarps = Cfg<Q8, NR>::kWarps, kPass = NR / 2;
  uint8_t ring[kWarps][Cfg<Q8, NR>::kStages][Geo<D, Q8, NR>::kStageBytes];
  union {
    float merge[kWarps][kPass][D];  // the warps' accumulators, kPass rows at a time
    float fin[kWarps][D];           // shares of a row's records
  };
  float warp_m[kWarps][NR], warp_l[kWarps][NR];  // their maxima and sums
  float row_m[NR], row_l[NR];                    // and the CTA's
  int cum[kMaxBatch + 1], len[kMaxBatch];
  int scratch[4 * kWarps];
  int last[2];
};

// Adds up a row's records: own_n of this launch (own0: the row's accumulators in the first) and, with PRE, pre_n of the
// prefix's (records of pre_rows rows, pre_step floats apart). A warp takes every parts-th of them, all of their maxima and
// sums: lanes read 32 of those at once while the first accumulators are on their way, so a short list costs one
// round trip. The order is fixed by the shapes. -> the share's accumulators over the whole sum (zeros without any key).
template <int D, bool PRE, int BATCH>
__device__ __forceinline__ void add_records(const float *own0, int own_n, int row, const float *pre0, int pre_n,
                                            int64_t pre_step, int pre_row, int pre_rows, int part, int parts,
                                            float (&a)[D / 32]) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31, n = own_n + (PRE ? pre_n : 0);
  auto row_of = [&](int k) -> const float * {
    return !PRE || k < own_n ? own0 + (int64_t)k * (kRows * (D + 2)) : pre0 + (int64_t)(k - own_n) * pre_step;
  };
  float M = -INFINITY, lsum = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) a[e] = 0.f;
#pragma unroll 1
  for (int k0 = 0; k0 < n; k0 += 32) {
    float mk = -INFINITY, lk = 0.f;
    if (k0 + lane < n) {
      const bool own = !PRE || k0 + lane < own_n;
      const int rows = own ? kRows : pre_rows, r = own ? row : pre_row;
      const float *stat = row_of(k0 + lane) + (rows - r) * D + r;  // past the accumulators: maxima, then sums
      mk = __ldcg(stat), lk = __ldcg(stat + rows);
    }
    const int cnt = min(32, n - k0);
    float fk = 0.f;
    int c = part;
    do {
      float v[BATCH][N];
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        if (c + b * parts < cnt) {
          const float *src = row_of(k0 + c + b * parts) + N * lane;
          if constexpr (N == 4) {
            const float4 t = __ldcg((const float4 *)src);
            v[b][0] = t.x, v[b][1] = t.y, v[b][2] = t.z, v[b][3] = t.w;
          } else if constexpr (N == 2) {
            const float2 t = __ldcg((const float2 *)src);
            v[b][0] = t.x, v[b][1] = t.y;
          } else {
            v[b][0] = __ldcg(src);
          }
        }
      }
      if (c == part) {  // a record without keys (sum 0) has no accumulators
        const float mx = fmaxf(M, warp_max(lk != 0.f ? mk : -INFINITY)), mz = mx == -INFINITY ? 0.f : mx;
        const float fo = ex2(M - mz);
        fk = lk != 0.f ? ex2(mk - mz) : 0.f;
        M = mx;
        lsum = lsum * fo + warp_sum(lk * fk);
#pragma unroll
        for (int e = 0; e < N; ++e) a[e] *= fo;
      }
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        const float fc = __shfl_sync(0xffffffffu, fk, (c + b * parts) & 31);
        if (c + b * parts < cnt && fc != 0.f)
#pragma unroll
          for (int e = 0; e < N; ++e) a[e] += v[b][e] * fc;
      }
      c += BATCH * parts;
    } while (c < cnt);
  }
  const float inv = inverse_sum(lsum);
#pragma unroll
  for (int e = 0; e < N; ++e) a[e] *= inv;
}
template <int N>
__device__ __forceinline__ void store_row(uint16_t *dst, const float (&a)[N]) {
  if constexpr (N == 4) *(uint2 *)dst = make_uint2(bf16x2(a[0], a[1]), bf16x2(a[2], a[3]));
  else if constexpr (N == 2) *(uint32_t *)dst = bf16x2(a[0], a[1]);
  else *dst = f32_to_bf16_bits(a[0]);
}

// The keys of a launch: the sequences' own, alone or beside a prefix, or the prefix's.
enum Mode { kOwn, kBeside, kPrefix };

// NR: query rows in use, 8 or 16. A (CTA, segment) pair leaves its record in slot CTA + segment: both only grow along the
// list, so slots are the pairs' own and a segment's are consecutive. Alone, a segment that one CTA holds goes
// straight to the output, and a split one's records are added up by the last of its CTAs to get there.
template <int D, bool Q8, int NR, Mode MODE>
__device__ __forceinline__ void attn_body(const Params &p, int block, int grid) {
  using C = Cfg<Q8, NR>;
  using G = Geo<D, Q8, NR>;
  using S = Smem<D, Q8, NR>;
  constexpr int kWarps = C::kWarps, STAGES = C::kStages;
  constexpr int TILE = G::kTile, NT = TILE / 8, ND = D / 8;
  constexpr bool PREFIX = MODE == kPrefix;
  constexpr bool PLANES = Q8 && NR == 8;  // scores by int8 MMAs on the digits of q
  extern __shared__ __align__(16) uint8_t smem_raw[];
  S &sm = *(S *)smem_raw;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  Layout lay;
  if (PREFIX) {
    lay.chunk = p.pre.chunk, lay.pad = p.pre.pad, lay.uncut = 0, lay.solo = false;
    lay.total = p.nkv * p.pre.row_tiles * ceil_div(p.pre.seg_tiles, lay.pad) * lay.pad;
  } else {
    lay = make_layout<C>(p, grid, sm.cum, sm.len, sm.scratch);
  }
  int x0 = (int)min((int64_t)lay.total, (int64_t)block * lay.chunk), x1 = min(lay.total, x0 + lay.chunk);
  const int stride = grid * kWarps;  // whole segments to warps: every stride-th
  int solo_seg = warp * grid + block;
  if (lay.solo) {
    while (solo_seg < p.m * p.nkv && sm.len[solo_seg / p.nkv] == 0) solo_seg += stride;
    x0 = 0, x1 = solo_seg < p.m * p.nkv ? lay.total : 0;
  } else if (lay.pad == 1) {  // both cuts at once, in the even and in the odd lanes
    const int cut = cut_at<TILE, PREFIX>(p, lay, sm.cum, sm.len, (int64_t)(block + (lane & 1)) * lay.chunk);
    x0 = __shfl_sync(0xffffffffu, cut, 0), x1 = __shfl_sync(0xffffffffu, cut, 1);
  }
  int split_n = 0;  // segments that this CTA shares with others: its first, its last
  int3 split[2] = {};  // their number, first CTA and CTAs
  if (x0 < x1) {
    Seg seg;
    if (!PREFIX && lay.solo) seg = own_seg<TILE>(p, sm.cum, sm.len, solo_seg / p.nkv, solo_seg % p.nkv);
    else seg = find_seg<TILE, PREFIX>(p, sm.cum, sm.len, x0);
    if (lay.pad > 1) x1 = min(x1, seg.end);
    const int first = lay.solo ? 0 : warp, step = lay.solo ? 1 : kWarps;  // this warp's tiles of a segment's part
    auto advance = [&](Seg &s) -> bool {  // to the next segment of this CTA's range, or of this warp
      if (!PREFIX && lay.solo) {
        int i = s.index + stride;
        while (i < p.m * p.nkv && sm.len[i / p.nkv] == 0) i += stride;
        if (i >= p.m * p.nkv) return false;
        s = own_seg<TILE>(p, sm.cum, sm.len, i / p.nkv, i % p.nkv);
        return true;
      }
      if (s.next >= x1) return false;
      s = next_seg<TILE, PREFIX>(p, sm.cum, sm.len, s);
      return true;
    };

    // ---- this warp's loads, STAGES - 1 tiles ahead. 32 lanes take 512 consecutive bytes of a full tile at a time; the
    // swizzles split into a part of the lane and one of the step.
    int lx = max(x0, seg.start) + first, lslot = 0;
    bool more = true;
    Seg ls = seg;
    constexpr int kStep = 32 / G::kChunks;  // rows per 512 bytes
    const int lr = lane / G::kChunks, lc = lane % G::kChunks;
    const uint32_t ring = smem_u32(sm.ring[warp][0]);
    const uint32_t k_dst = ring + lr * G::kRowBytes + ((lc ^ G::k_swz(lr)) * 16);
    const uint32_t v_dst = lr * G::kRowBytes + ((lc ^ G::v_swz(lr)) * 16);
    auto load_next = [&]() {
      while (lx >= ls.end && more) {
        more = advance(ls);
        if (more) lx = ls.start + first;
      }
      if (lx < min(ls.end, x1)) {
        const uint32_t st = (uint32_t)(lslot * G::kStageBytes);
        const Cache &c = p.cache;
        const int key0 = (lx - ls.start) * TILE, left = ls.len - key0;
        const int64_t row0 = (PREFIX ? ls.g : (int64_t)ls.seq * p.nkv + ls.g) * c.cap + key0;
        const uint8_t *kb = c.k + row0 * G::kRowBytes + lane * 16, *vb = c.v + row0 * G::kRowBytes + lane * 16;
        // v_swz(it kStep + lr) = v_swz(it kStep) ^ v_swz(lr) (the row bits it uses do not carry)
        const uint32_t kd = st + k_dst, vd = st + ring + TILE * G::kRowBytes;
        if (left >= TILE) {
#pragma unroll
          for (int it = 0; it < TILE / kStep; ++it) {
            cp16(kd + it * 512, kb + it * 512);
            cp16(vd + (v_dst ^ (G::v_swz(it * kStep) * 16)) + it * 512, vb + it * 512);
          }
        } else {
#pragma unroll 1
          for (int it = 0; it < TILE / kStep; ++it) {
            const bool in = it * kStep + lr < left;
            cp16z(kd + it * 512, in ? kb + it * 512 : c.k, in ? 16 : 0);
            cp16z(vd + (v_dst ^ (G::v_swz(it * kStep) * 16)) + it * 512, in ? vb + it * 512 : c.v, in ? 16 : 0);
          }
        }
        if (Q8) {
          const uint32_t sc = ring + st + 2 * TILE * G::kRowBytes + lane * 4;  // [ks of the tile][vs of the tile]
          const bool in = lane < left;
          cp4(sc, c.ks + row0 + (in ? lane : 0), in ? 4 : 0);
          cp4(sc + TILE * 4, c.vs + row0 + (in ? lane : 0), in ? 4 : 0);
        }
      }
      cp_commit();
      lx += step;
      lslot = lslot + 1 == STAGES ? 0 : lslot + 1;
    };
    // the segment's query rows, dims d0 .. d0 + 3 of every 16-dim step: those of the key words that this thread loads
    uint2 qw[NR / 8][D / 16];
    auto load_q = [&](const Seg &sg) {
#pragma unroll
      for (int hh = 0; hh < NR / 8; ++hh) {
        const int r = g + 8 * hh;
        int64_t tok = -1;
        int h = 0;
        if (PREFIX) {
          const int flat = sg.tile * kRows + r;
          if (flat < p.m * p.group) tok = flat / p.group, h = sg.g * p.group + flat % p.group;
        } else if (r < p.group) {
          tok = sg.seq, h = sg.g * p.group + r;
        }
        const uint16_t *qr = p.q + (tok >= 0 ? tok * p.ldq + (int64_t)h * D : 0);
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
          const int d0 = Q8 ? (D == 32 ? 8 * t + 4 * s : 16 * (t + 4 * (s / 4)) + 4 * (s % 4))
                            : 8 * (t + 4 * (s / 2)) + 4 * (s % 2);
          qw[hh][s] = tok >= 0 ? *(const uint2 *)(qr + d0) : make_uint2(0u, 0u);
        }
      }
    };
    load_q(seg);  // before the keys and values queue up in front of it
#pragma unroll 1
    for (int s = 0; s < STAGES - 1; ++s) load_next();

    int cslot = 0;
    for (;;) {
      // ---- the segment's query rows as MMA fragments
      uint32_t qa[PLANES ? D / 32 : D / 16][PLANES ? 8 : 4];
      float rowfac[2] = {p.scale_log2, p.scale_log2};  // and for int8 the power of two that q was divided by
#pragma unroll
      for (int hh = 0; hh < NR / 8; ++hh) {
        const uint2(&w)[D / 16] = qw[hh];
        uint32_t amax2 = 0u;  // the largest magnitudes of the even and odd elements, as bf16 bits (NaN above infinity)
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
          if (Q8) amax2 = __vmaxu2(amax2, __vmaxu2(w[s].x & 0x7fff7fffu, w[s].y & 0x7fff7fffu));
        if (Q8) {
          amax2 = __vmaxu2(amax2, __shfl_xor_sync(0xffffffffu, amax2, 1));
          amax2 = __vmaxu2(amax2, __shfl_xor_sync(0xffffffffu, amax2, 2));
          const int amax = (int)max(amax2 & 0xffffu, amax2 >> 16);
          // a largest magnitude in [2^e, 2^(e + 1)) becomes one in [2^B, 2^(B + 1)): as fixed point (B = 29) bf16's 8 bits stay exact for
          // elements down to 2^-22 of the row's largest, in f16 (B = 14) down to 2^-28. (The exponent is kept where both
          // factors are normal numbers.)
          constexpr int B = PLANES ? 29 : 14;
          const int e = min(max((amax >> 7) - 127, B - 126), 127);
          const float up = __uint_as_float((uint32_t)(127 + B - e) << 23);
          rowfac[hh] *= __uint_as_float((uint32_t)(127 - B + e) << 23);
          if (amax >= 0x7f80) rowfac[hh] = NAN;  // an infinity or NaN in the row: its scores are NaN
#pragma unroll
          for (int s = 0; s < D / 16; ++s) {
            const float y[4] = {bf16_lo(w[s].x) * up, bf16_hi(w[s].x) * up, bf16_lo(w[s].y) * up, bf16_hi(w[s].y) * up};
            if constexpr (PLANES) {
              // bytes of X + 0x80808080 are the digits plus 128; a 4 x 4 byte transpose makes words of one digit (d[0] the
              // lowest) of the four dims
              uint32_t Y[4], d[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) Y[i] = ((uint32_t)__float2int_rn(y[i]) + 0x80808080u) ^ 0x80808080u;
              const uint32_t lo01 = __byte_perm(Y[0], Y[1], 0x5140), hi01 = __byte_perm(Y[0], Y[1], 0x7362);
              const uint32_t lo23 = __byte_perm(Y[2], Y[3], 0x5140), hi23 = __byte_perm(Y[2], Y[3], 0x7362);
              d[0] = __byte_perm(lo01, lo23, 0x5410), d[1] = __byte_perm(lo01, lo23, 0x7632);
              d[2] = __byte_perm(hi01, hi23, 0x5410), d[3] = __byte_perm(hi01, hi23, 0x7632);
              // MMA 0: planes 3 and 2 in rows g and g + 8; MMA 1: planes 1 and 0
              const int c = 2 * (s & 1);
              qa[s / 2][c] = d[3], qa[s / 2][c + 1] = d[2], qa[s / 2][4 + c] = d[1], qa[s / 2][4 + c + 1] = d[0];
            } else {
              qa[s][hh] = f16x2(y[0], y[1]), qa[s][hh + 2] = f16x2(y[2], y[3]);
            }
          }
        } else {
#pragma unroll
          for (int s = 0; s < D / 16; ++s) qa[s][hh] = w[s].x, qa[s][hh + 2] = w[s].y;
        }
      }
      if (NR == 8 && !PLANES) {
#pragma unroll
        for (int s = 0; s < D / 16; ++s) qa[s][1] = qa[s][3] = 0u;
      }
      float m_run[2] = {-INFINITY, -INFINITY}, l_part[2] = {0.f, 0.f};
      float acc[ND][4];
#pragma unroll
      for (int j = 0; j < ND; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;

      const int seg_end = min(seg.end, x1);
      for (int x = max(x0, seg.start) + first; x < seg_end; x += step) {
        load_next();
        cp_wait<STAGES - 1>();
        __syncwarp();
        const uint8_t *kt = sm.ring[warp][cslot];
        cslot = cslot + 1 == STAGES ? 0 : cslot + 1;
        const uint8_t *vt = kt + TILE * G::kRowBytes;
        const float *ksc = (const float *)(vt + TILE * G::kRowBytes), *vsc = ksc + TILE;
        const int left = seg.len - (x - seg.start) * TILE;  // keys from the tile's first to the segment's end

        // ---- scores in log2 units: n-tile nt holds keys 8 nt .. 8 nt + 7 (this thread loads key 8 nt + g and gets rows g,
        // g + 8 of keys 8 nt + 2t, 8 nt + 2t + 1)
        float sc[NT][4];
        float2 vs[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
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
          float2 ks = make_float2(1.f, 1.f);
          if (Q8) ks = *(const float2 *)(ksc + 8 * nt + 2 * t), vs[nt] = *(const float2 *)(vsc + 8 * nt + 2 * t);
          if constexpr (PLANES) {
            int hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < D / 32; ++s) {
              mma_i8(hi, qa[s], kw[2 * s], kw[2 * s + 1]);
              mma_i8(lo, qa[s] + 4, kw[2 * s], kw[2 * s + 1]);
            }
            // |digit sums| <= 2^21, so both halves of the 32-bit digits' sum fit an int
            sc[nt][0] = fmaf((float)(hi[0] * 256 + hi[2]), 65536.f, (float)(lo[0] * 256 + lo[2])) * (rowfac[0] * ks.x);
            sc[nt][1] = fmaf((float)(hi[1] * 256 + hi[3]), 65536.f, (float)(lo[1] * 256 + lo[3])) * (rowfac[0] * ks.y);
            sc[nt][2] = sc[nt][3] = 0.f;
          } else {
            sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
            for (int s = 0; s < D / 16; ++s) {
              if (Q8) {
                const uint32_t b = kw[s] ^ 0x80808080u;
                mma<true>(sc[nt], qa[s], codes_f16(b, 0x4140), codes_f16(b, 0x4342));
              } else {
                mma<false>(sc[nt], qa[s], kw[(2 * s) % NW], kw[(2 * s + 1) % NW]);
              }
            }
#pragma unroll
            for (int hh = 0; hh < NR / 8; ++hh) sc[nt][2 * hh] *= rowfac[hh] * ks.x, sc[nt][2 * hh + 1] *= rowfac[hh] * ks.y;
          }
        }
        if (left < TILE) {  // the segment's last tile
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const int key = 8 * nt + 2 * t;
            if (key >= left) sc[nt][0] = sc[nt][2] = -INFINITY;
            if (key + 1 >= left) sc[nt][1] = sc[nt][3] = -INFINITY;
          }
        }
        float ms[2], alpha[2] = {1.f, 1.f};
#pragma unroll
        for (int hh = 0; hh < NR / 8; ++hh) {
          float mx = -INFINITY;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mx = fmaxf(mx, fmaxf(sc[nt][2 * hh], sc[nt][2 * hh + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float m_new = fmaxf(m_run[hh], mx);
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
            if (Q8) p0 *= vs[nt].x, p1 *= vs[nt].y;  // (past the segment's end both are zeros)
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
                const uint32_t b0 = widen2(pair[0][e / 2], select), b1 = widen2(pair[1][e / 2], select);
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
      const Seg done = seg;
      const bool another = lay.pad == 1 && advance(seg);
      if (another) load_q(seg);  // on its way while this one is added up
      // ---- the segment is done: the warps' states, each relative to the largest maximum, are added up in shared memory
#pragma unroll
      for (int hh = 0; hh < NR / 8; ++hh) {
        l_part[hh] += __shfl_xor_sync(0xffffffffu, l_part[hh], 1);
        l_part[hh] += __shfl_xor_sync(0xffffffffu, l_part[hh], 2);
        if (t == 0 && !lay.solo) sm.warp_m[warp][g + 8 * hh] = m_run[hh], sm.warp_l[warp][g + 8 * hh] = l_part[hh];
      }
      if (!PREFIX && lay.solo) {  // the warp's own: to the output, or a record in the segment's slot
        float *rec = record<D>(p, done.index);
        uint16_t *out = p.out + done.seq * p.ldo + (int64_t)done.g * p.group * D;
#pragma unroll
        for (int hh = 0; hh < NR / 8; ++hh) {
          const int r = g + 8 * hh;
          if (r < p.group) {
            const float inv = inverse_sum(l_part[hh]);
#pragma unroll
            for (int j = 0; j < ND; j += 4)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int c = 2 * hh + e, dim = r * D + G::out_dim(j, e, t);
                if (MODE == kOwn)
                  *(uint2 *)(out + dim) = make_uint2(bf16x2(acc[j][c] * inv, acc[j + 1][c] * inv),
                                                     bf16x2(acc[j + 2][c] * inv, acc[j + 3][c] * inv));
                else
                  *(float4 *)(rec + dim) = make_float4(acc[j][c], acc[j + 1][c], acc[j + 2][c], acc[j + 3][c]);
              }
            if (MODE != kOwn && t == 0) rec[kRows * D + r] = m_run[hh], rec[kRows * D + kRows + r] = l_part[hh];
          }
        }
        if (MODE == kBeside && lane == 0) p.parts[done.index] = make_int2(done.index, 1);
        if (!another) break;
        continue;
      }
      __syncthreads();
      float fac[NR / 8];
#pragma unroll
      for (int hh = 0; hh < NR / 8; ++hh) {
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm.warp_m[w][g + 8 * hh]);
        fac[hh] = ex2(m_run[hh] - (mx == -INFINITY ? 0.f : mx));
      }
      if (threadIdx.x < NR) {
        float mx = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm.warp_m[w][threadIdx.x]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
          l += sm.warp_l[w][threadIdx.x] * ex2(sm.warp_m[w][threadIdx.x] - (mx == -INFINITY ? 0.f : mx));
        sm.row_m[threadIdx.x] = mx, sm.row_l[threadIdx.x] = l;
      }
      const bool whole = done.start >= x0 && done.end <= x1;
      const bool final = MODE == kOwn && whole;
      const int rows = PREFIX ? NR : p.group;  // of the record, whose stride is kRows either way
      float *rec = record<D>(p, block + done.index);
      constexpr int kPass = S::kPass;
#pragma unroll 1
      for (int r0 = 0; r0 < rows; r0 += kPass) {
        if (r0) __syncthreads();  // the last pass has been read
#pragma unroll
        for (int hh = 0; hh < NR / 8; ++hh) {
          const int r = g + 8 * hh - r0;
          if (r >= 0 && r < kPass && r + r0 < rows) {
#pragma unroll
            for (int j = 0; j < ND; j += 4)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int c = 2 * hh + e;
                *(float4 *)&sm.merge[warp][r][G::out_dim(j, e, t)] =
                    make_float4(acc[j][c] * fac[hh], acc[j + 1][c] * fac[hh], acc[j + 2][c] * fac[hh], acc[j + 3][c] * fac[hh]);
              }
          }
        }
        __syncthreads();
#pragma unroll 1
        for (int e = threadIdx.x; e < min(kPass, rows - r0) * D; e += C::kThreads) {
          float a = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) a += sm.merge[w][e / D][e % D];
          if (final) {
            const float l = sm.row_l[r0 + e / D];
            p.out[done.seq * p.ldo + (int64_t)(done.g * p.group + r0) * D + e] = f32_to_bf16_bits(l == 0.f ? 0.f : a / l);
          } else {
            rec[r0 * D + e] = a;
          }
        }
      }
      if (!final && threadIdx.x < rows) {
        rec[kRows * D + threadIdx.x] = sm.row_m[threadIdx.x];
        rec[kRows * D + kRows + threadIdx.x] = sm.row_l[threadIdx.x];
      }
      if (MODE != kPrefix && !final) {
        const int c0 = done.start / lay.chunk, c1 = (done.end - 1) / lay.chunk;
        if (MODE == kOwn) {
          (split_n ? split[1] : split[0]) = make_int3(done.index, c0, c1 - c0 + 1);
          ++split_n;
        } else if (done.start >= x0 && threadIdx.x == 0) {  // (a short segment lies in one CTA wherever the even cuts are)
          p.parts[done.index] = make_int2(whole ? block + done.index : c0 + done.index, whole ? 1 : c1 - c0 + 1);
        }
      }
      if (!another) break;
    }
    cp_wait<0>();
  }
  if (MODE == kBeside) {
    for (int e = block * C::kThreads + threadIdx.x; e < p.m * p.nkv; e += grid * C::kThreads)
      if (sm.len[e / p.nkv] == 0) p.parts[e] = make_int2(0, 0);
  }
  if constexpr (MODE == kOwn) {
    for (int e = block; e < p.m * p.nkv; e += grid)  // sequences without keys
      if (sm.len[e / p.nkv] == 0)
        for (int c = threadIdx.x; c < p.group * D; c += C::kThreads)
          p.out[(e / p.nkv) * p.ldo + (int64_t)(e % p.nkv) * p.group * D + c] = 0;
    if (!split_n) return;
    __syncthreads();
    if ((int)threadIdx.x < split_n) {  // (the fence covers the CTA's records, which the barrier ordered before it)
      const int3 e = threadIdx.x ? split[1] : split[0];
      __threadfence();
      const bool last = atomicAdd(p.cnt + e.y, 1u) == (unsigned)(e.z - 1);
      if (last) {
        __threadfence();
        p.cnt[e.y] = 0u;
      }
      sm.last[threadIdx.x] = last;
    }
    __syncthreads();
#pragma unroll 1
    for (int s = 0; s < split_n; ++s) {
      if (!sm.last[s]) continue;
      // a warp takes a row, or with fewer rows than warps every parts-th record of one
      const int3 e = s ? split[1] : split[0];
      const int parts = p.group < kWarps ? kWarps / p.group : 1, part = parts > 1 ? warp / p.group : 0;
      uint16_t *out = p.out + (e.x / p.nkv) * p.ldo + (int64_t)(e.x % p.nkv) * p.group * D;
      const float *rec = record<D>(p, e.y + e.x);
#pragma unroll 1
      for (int j = warp - part * p.group; j < p.group && part < parts; j += kWarps) {
        float a[D / 32];
        add_records<D, false, 8>(rec + j * D, e.z, j, nullptr, 0, 0, 0, 0, part, parts, a);
        if (parts == 1) {
          store_row(out + j * D + D / 32 * lane, a);
        } else {
#pragma unroll
          for (int i = 0; i < D / 32; ++i) sm.fin[warp][D / 32 * lane + i] = a[i];
        }
      }
      if (parts == 1) continue;
      __syncthreads();
      for (int i = threadIdx.x; i < p.group * D; i += C::kThreads) {
        float v = 0.f;
        for (int q = 0; q < parts; ++q) v += sm.fin[q * p.group + i / D][i % D];
        out[i] = f32_to_bf16_bits(v);
      }
      __syncthreads();  // sm.fin is free again
    }
  }
}

// The sequences' own keys, alone or beside attn_prefix_kernel's launch.
template <int D, bool Q8, int NR, Mode MODE>
__global__ void __launch_bounds__(Cfg<Q8, NR>::kThreads, 1) attn_kernel(const Params p) {
  if (MODE == kOwn) pdl_wait();  // (what precedes the prefix's launch is done once that has started)
  pdl_launch_dependents();
  attn_body<D, Q8, NR, MODE>(p, (int)blockIdx.x, (int)gridDim.x);
  if (MODE == kBeside) pdl_wait();  // the prefix's launch: what waits for this one has waited for both
}
// A prefix (NP query rows in use) and the sequences' own keys (NO) in one launch: the prefix's CTAs first, no CTA waits for
// another.
template <int D, bool Q8, int NP, int NO>
__global__ void __launch_bounds__(Cfg<Q8, NP>::kThreads, 1) attn_both_kernel(const Params pre, const Params own) {
  pdl_wait();
  pdl_launch_dependents();
  const int ctas = own.pre.grid;
  if ((int)blockIdx.x < ctas) attn_body<D, Q8, NP, kPrefix>(pre, (int)blockIdx.x, ctas);
  else attn_body<D, Q8, NO, kBeside>(own, (int)blockIdx.x - ctas, (int)gridDim.x - ctas);
}

// Beside a prefix: one (sequence, head) row per warp, its own records and the prefix's. Bound by three dependent round
// trips to L2 (the segment's parts, then two batches of records): 2048 rows of 19 records 5.6 us.
constexpr int kAddWarps = 4;
template <int D>
__global__ void __launch_bounds__(32 * kAddWarps) add_kernel(const Params p) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, unit = blockIdx.x * kAddWarps + (threadIdx.x >> 5);
  const int nq = p.nkv * p.group;
  if (unit >= p.m * nq) return;
  const int i = unit / nq, h = unit - i * nq, g = h / p.group, j = h - g * p.group;
  const int2 own = p.parts[i * p.nkv + g];
  const float *pre0;  // the row's accumulators in the prefix's first record
  int pre_n, pre_rows = kRows, pre_row;
  int64_t pre_step;
  if (p.pre.big) {
    const int tile = i / p.pre.seqs, pair = tile / 2;
    pre_n = p.pre.ranges, pre_step = 2 * apx::record_size(D);
    pre_row = (i - tile * p.pre.seqs) * p.group + j, pre_rows = apx::kRowsT;
    pre0 = p.pre.rec + ((int64_t)(g * p.pre.pairs + pair) * p.pre.ranges * 2 + (tile & 1)) * apx::record_size(D);
  } else {
    const int flat = i * p.group + j, seg = g * p.pre.row_tiles + flat / kRows;
    const int start = seg * ceil_div(p.pre.seg_tiles, p.pre.pad) * p.pre.pad;
    const int c0 = start / p.pre.chunk;
    pre_n = (start + p.pre.seg_tiles - 1) / p.pre.chunk - c0 + 1;
    pre_step = kRows * (D + 2);
    pre_row = flat % kRows;
    pre0 = p.pre.rec + (int64_t)(c0 + seg) * pre_step;
  }
  float a[D / 32];
  add_records<D, true, 10>(record<D>(p, own.x) + j * D, own.y, j, pre0 + pre_row * D, pre_n, pre_step, pre_row, pre_rows,
                           0, 1, a);
  store_row(p.out + i * p.ldo + (int64_t)h * D + D / 32 * lane, a);
}

// The shared-memory opt-in of a kernel, once per device.
template <typename F>
static cudaError_t configure(F *fn, size_t smem, int (&configured)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || configured[dev]) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess) configured[dev] = 1;
  return e;
}
template <int D, bool Q8, int NR, Mode MODE>
static cudaError_t launch(const Params &p, int grid, cudaStream_t st, bool pdl) {
  static int configured[64] = {0};
  const auto fn = attn_kernel<D, Q8, NR, MODE>;
  const size_t smem = sizeof(Smem<D, Q8, NR>);
  if (const cudaError_t e = configure(fn, smem, configured); e != cudaSuccess) return e;
  return launch_kernel((const void *)fn, dim3(grid), dim3(Cfg<Q8, NR>::kThreads), smem, st, pdl, p);
}
template <int D, bool Q8, int NP, int NO>
static cudaError_t launch_both(const Params &pre, const Params &own, int grid, cudaStream_t st, bool pdl) {
  static int configured[64] = {0};
  const auto fn = attn_both_kernel<D, Q8, NP, NO>;
  const size_t smem = std::max(sizeof(Smem<D, Q8, NP>), sizeof(Smem<D, Q8, NO>));
  if (const cudaError_t e = configure(fn, smem, configured); e != cudaSuccess) return e;
  return launch_kernel((const void *)fn, dim3(own.pre.grid + grid), dim3(Cfg<Q8, NP>::kThreads), smem, st, pdl, pre, own);
}

static int row_tiles(int64_t m, int group) { return (int)((m * group + kRows - 1) / kRows); }
static int max_grid() { return num_sms(); }
// CTAs that the sequences' own keys can need: no more than their ranges if each has the fewest keys a range may have;
// beside a prefix on less than half of the SMs, those that it leaves free (neither kernel shares an SM).
template <typename C>
static int own_grid(const Params &p) {
  const int free = max_grid() - p.pre.grid;
  const int64_t most = ((p.cache.cap + C::kTile - 1) / C::kTile + C::kMinChunk - 1) / C::kMinChunk;
  return (int)std::min<int64_t>(free >= max_grid() / 2 ? free : max_grid(), most * p.m * p.nkv);
}
// How the prefix's segments are cut: as make_layout does it, on the host.
template <typename C>
static void cut_prefix(Params &p) {
  Prefix &c = p.pre;
  const int grid = max_grid();
  c.row_tiles = row_tiles(p.m, p.group);
  c.seg_tiles = ceil_div(p.keys, C::kTile);
  const int segs = p.nkv * c.row_tiles, share = ceil_div(segs * c.seg_tiles, grid), least = std::max(C::kMinChunk, share);
  c.pad = 1, c.chunk = share;
  for (int j = 0; j < 32; ++j) {
    const int len = least + ceil_div(least * j, 64);
    if ((int64_t)segs * ceil_div(c.seg_tiles, len) <= grid) {
      c.pad = c.chunk = len;
      break;
    }
  }
  c.grid = ceil_div(segs * ceil_div(c.seg_tiles, c.pad) * c.pad, c.chunk);
}
template <bool Q8, int NR, Mode MODE>
static cudaError_t launch_d(Params &p, int d, cudaStream_t st, bool pdl) {
  const int grid = own_grid<Cfg<Q8, NR>>(p);
  p.head_share = grid / p.nkv;
  if (d == 128) return launch<128, Q8, NR, MODE>(p, grid, st, pdl);
  if constexpr (MODE == kOwn)  // (attn_prefix_kernel has no head_dim 32)
    if (d == 32) return launch<32, Q8, NR, MODE>(p, grid, st, pdl);
  return launch<64, Q8, NR, MODE>(p, grid, st, pdl);
}
template <Mode MODE>
static cudaError_t launch_any(Params &p, int d, bool q8, cudaStream_t st, bool pdl) {
  if (p.group <= 8) return q8 ? launch_d<true, 8, MODE>(p, d, st, pdl) : launch_d<false, 8, MODE>(p, d, st, pdl);
  return q8 ? launch_d<true, 16, MODE>(p, d, st, pdl) : launch_d<false, 16, MODE>(p, d, st, pdl);
}
template <bool Q8, int NP, int NO>
static cudaError_t launch_both_d(Params &pre, Params &own, int d, cudaStream_t st, bool pdl) {
  cut_prefix<Cfg<Q8, NP>>(pre);
  own.pre = pre.pre;
  const int grid = own_grid<Cfg<Q8, NO>>(own);
  own.head_share = grid / own.nkv;
  return d == 128 ? launch_both<128, Q8, NP, NO>(pre, own, grid, st, pdl)
                  : (d == 64 ? launch_both<64, Q8, NP, NO>(pre, own, grid, st, pdl)
                             : launch_both<32, Q8, NP, NO>(pre, own, grid, st, pdl));
}
static cudaError_t launch_both_any(Params &pre, Params &own, int d, bool q8, cudaStream_t st, bool pdl) {
  if (own.m * own.group <= 8)
    return q8 ? launch_both_d<true, 8, 8>(pre, own, d, st, pdl) : launch_both_d<false, 8, 8>(pre, own, d, st, pdl);
  if (own.group <= 8)
    return q8 ? launch_both_d<true, 16, 8>(pre, own, d, st, pdl) : launch_both_d<false, 16, 8>(pre, own, d, st, pdl);
  return q8 ? launch_both_d<true, 16, 16>(pre, own, d, st, pdl) : launch_both_d<false, 16, 16>(pre, own, d, st, pdl);
}
// Whether the prefix goes to attn_prefix_kernel (head_dim 64 or 128) or to the mma.sync kernel's 16-row tiles, whose time
// grows with rows x keys: above 1.5 million (query head, key) pairs of the batch for bf16, and for int8, whose tiles the
// tcgen05 kernel has to widen first, above 3.5 million and 64 rows. Measured at 8 kv heads and head_dim 128 alone, and
// there 1.6 us off at 256 bf16 rows x 1024 keys. Whole calls in us, tcgen05 / mma.sync, rows of each kv head:
//              64 rows, keys 1024, 4096, 16384     128 rows                         256 rows
//   bf16       15.4/11.8  17.7/20.2  28.1/40.1     16.4/16.5  18.4/27.4  28.5/69.6   22.0/20.4  24.2/39.5  38.6/127.7
//   int8       21.0/13.2  24.6/23.1  49.6/42.9     22.2/18.7  25.0/30.0  49.1/72.1   30.8/22.7  32.8/41.6  61.5/130.3
static bool prefix_on_tcgen05(int64_t m, int group, int nkv, int64_t keys, int d, float scale, bool q8) {
  const int64_t rows = m * group, pairs = rows * nkv * keys;
  return d >= 64 && scale > 0.f && (q8 ? rows > 64 && pairs > 3500000 : rows > kRows && pairs > 1500000);
}
// The workspace: arrival counters, one per CTA (a CTA is the first of at most one split segment) whatever the call's
// sizes, so that calls of different sizes can share it; the segments' (first record, records) pairs; the records.
static size_t counter_bytes() { return ((size_t)max_grid() * sizeof(unsigned) + 255) / 256 * 256; }
static size_t parts_bytes(int64_t m, int nkv) { return ((size_t)m * nkv * sizeof(int2) + 255) / 256 * 256; }
static void set_workspace(Params &p, void *ws) {
  p.cnt = (unsigned *)ws, p.parts = (int2 *)((char *)ws + counter_bytes());
  p.ws = (float *)((char *)p.parts + parts_bytes(p.m, p.nkv));
}

static int check(const char *what, int64_t ldo, int64_t ldq, const void *out, const void *q, int64_t cap, int64_t m,
                 int nq, int nkv, int d, float scale, const void *ws, size_t ws_bytes) {
  if (d != 32 && d != 64 && d != 128) return set_error(EGPT_ERR_SHAPE, "%s: head_dim must be 32, 64 or 128", what);
  if (nq < 1 || nkv < 1 || nq % nkv || nq / nkv > kRows)
    return set_error(EGPT_ERR_SHAPE, "%s: nq must be a multiple of nkv, at most %d to one", what, kRows);
  if (m < 1 || m > kMaxBatch || cap < 1 || cap > (1 << 27) || ldq < (int64_t)nq * d || ldo < (int64_t)nq * d)
    return set_error(EGPT_ERR_SHAPE, "%s: bad m (1 to %d), cap or leading dimension", what, kMaxBatch);
  if (nkv > (1 << 24) / m || m * nkv * ((cap + 15) / 16) > 0x1fffffff)
    return set_error(EGPT_ERR_SHAPE, "%s: cache too long for the batch", what);
  if (!std::isfinite(scale * kLog2e)) return set_error(EGPT_ERR_ARG, "%s: scale log2(e) must be finite", what);
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
  // arrival counters; a record for every (CTA, segment) pair of the launch over the sequences' own keys; the prefix's
  // records: attn_kernel's, one for every pair again, or attn_prefix_kernel's
  const size_t rec = aq8::kRows * ((size_t)d + 2) * 4;
  const size_t small = ((size_t)aq8::max_grid() + (size_t)nkv * aq8::row_tiles(m, nq / nkv)) * rec;
  const size_t big = (d == 64 || d == 128) && nq / nkv <= aq8::kRows ? apx::record_floats(m, nq / nkv, nkv, d) * 4 : 0;
  return aq8::counter_bytes() + aq8::parts_bytes(m, nkv) + ((size_t)aq8::max_grid() + (size_t)m * nkv) * rec + std::max(small, big);
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
  p.cache = {(const uint8_t *)k_cache, (const uint8_t *)v_cache, k_scale, v_scale, cap};
  p.position = position, p.m = (int)m, p.nkv = nkv, p.group = nq / nkv, p.scale_log2 = scale * aq8::kLog2e;
  aq8::set_workspace(p, ws);
  return check_launch(aq8::launch_any<aq8::kOwn>(p, d, true, (cudaStream_t)stream, (flags & EGPT_FLAG_PDL) != 0),
                      "attn_decode_q8_kernel");
}

extern "C" int egpt_attn_shared_prefix_on_tcgen05(int64_t m, int nq, int nkv, int d, int64_t prefix_len, float scale,
                                                  int cache_dtype) {
  return m >= 1 && nkv >= 1 && nq >= nkv && (d == 64 || d == 128) && prefix_len >= 1 &&
         aq8::prefix_on_tcgen05(m, nq / nkv, nkv, prefix_len, d, scale * aq8::kLog2e, cache_dtype == EGPT_I8);
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
  if (prefix_cap < 1 || prefix_len < 0 || prefix_len > prefix_cap || prefix_len > (1 << 27) ||
      (int64_t)nkv * aq8::row_tiles(m, nq / nkv) * ((prefix_len + 15) / 16) > 0x1fffffff)
    return set_error(EGPT_ERR_SHAPE, "attn_shared_prefix: bad prefix_len (0 to prefix_cap), or too long for the batch");
  if ((uintptr_t)pk % 16 || (uintptr_t)pv % 16 || (uintptr_t)tk % 16 || (uintptr_t)tv % 16)
    return set_error(EGPT_ERR_ALIGN, "attn_shared_prefix: caches must be 16-byte aligned");
  const cudaStream_t st = (cudaStream_t)stream;
  const bool pdl = (flags & EGPT_FLAG_PDL) != 0;
  aq8::Params p{};
  p.out = (uint16_t *)out, p.ldo = ldo, p.q = (const uint16_t *)q, p.ldq = ldq;
  p.position = position, p.m = (int)m, p.nkv = nkv, p.group = nq / nkv, p.scale_log2 = scale * aq8::kLog2e;
  aq8::set_workspace(p, ws);
  float *pre_rec = p.ws + ((size_t)aq8::max_grid() + (size_t)m * nkv) * aq8::kRows * (d + 2);
  p.cache = {(const uint8_t *)tk, (const uint8_t *)tv, tk_scale, tv_scale, cap};
  if (prefix_len == 0) return check_launch(aq8::launch_any<aq8::kOwn>(p, d, q8, st, pdl), "attn_shared_prefix_kernel");
  p.pre.rec = pre_rec;
  if (aq8::prefix_on_tcgen05(m, p.group, nkv, prefix_len, d, p.scale_log2, q8)) {
    apx::Args A{};
    const apx::Shape sh = apx::shape_of(m, p.group, nkv, prefix_len);
    A.ws = pre_rec, A.prefix = prefix_len, A.m = (int)m, A.nkv = nkv, A.group = p.group, A.scale_log2 = p.scale_log2;
    A.ks = pk_scale, A.vs = pv_scale, A.cap = prefix_cap;
    bool maps_ok = false;
    cudaError_t e = d == 128 ? (q8 ? apx::launch<128, true>(A, q, ldq, pk, pv, sh, st, pdl, maps_ok)
                                   : apx::launch<128, false>(A, q, ldq, pk, pv, sh, st, pdl, maps_ok))
                             : (q8 ? apx::launch<64, true>(A, q, ldq, pk, pv, sh, st, pdl, maps_ok)
                                   : apx::launch<64, false>(A, q, ldq, pk, pv, sh, st, pdl, maps_ok));
    if (!maps_ok) return set_error(EGPT_ERR_ALIGN, "attn_shared_prefix: tensor maps rejected");
    if (e != cudaSuccess) return check_launch(e, "attn_prefix_kernel");
    p.pre.grid = nkv * sh.pairs * sh.ranges;
    p.pre.big = 1, p.pre.seqs = sh.seqs, p.pre.pairs = sh.pairs, p.pre.ranges = sh.ranges;
    e = aq8::launch_any<aq8::kBeside>(p, d, q8, st, true);
    if (e != cudaSuccess) return check_launch(e, "attn_shared_prefix_kernel");
  } else {
    aq8::Params a = p;
    a.cache = {(const uint8_t *)pk, (const uint8_t *)pv, pk_scale, pv_scale, prefix_cap};
    a.keys = (int)prefix_len, a.ws = pre_rec;
    const cudaError_t e = aq8::launch_both_any(a, p, d, q8, st, pdl);
    if (e != cudaSuccess) return check_launch(e, "attn_shared_prefix_both_kernel");
  }
  const void *fn = d == 128 ? (const void *)aq8::add_kernel<128>
                            : (d == 64 ? (const void *)aq8::add_kernel<64> : (const void *)aq8::add_kernel<32>);
  return check_launch(launch_kernel(fn, dim3((unsigned)((m * nq + aq8::kAddWarps - 1) / aq8::kAddWarps)),
                                    dim3(32 * aq8::kAddWarps), 0, st, true, p),
                      "attn_shared_prefix_add_kernel");
}
