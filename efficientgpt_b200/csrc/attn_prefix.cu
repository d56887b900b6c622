// The shared prefix's part of egpt_attn_shared_prefix on the 5th-generation tensor cores (tcgen05): bf16 and int8 caches,
// head_dim 64 or 128, batches of more query rows than the mma.sync kernel's tiles are good for (attn_q8.cu has the rule).
//
// The (sequence, head) rows of a kv head, up to 128 of them, are the M of the MMAs: row r of tile t is head r % group of
// sequence t * seqs + r / group. A CTA owns one kv head, one pair of row tiles and one range of 128-key blocks, and
// runs two streams, each with 128 columns of TMEM for scores and D for its output:
//   two row tiles:  both streams take every block, one tile each, so a block is loaded once for 256 rows;
//   one row tile:   the streams take alternate blocks of the same rows.
// Either way one stream's softmax runs under the other's MMAs. Roles:
//   warp 0    lane 0 issues the TMA loads (this GPU's memory, no multicast): the query tiles, then K and V blocks, 128-byte
//             swizzle, into operand rings (bf16) or a ring of raw code tiles (int8); the cache maps end at the prefix's
//             last key;
//   warp 1    allocates TMEM; lane 0 issues S = Q K^T and O += P V, P read from TMEM where the scores were (the next
//             block's scores of the stream are issued after the P.V that reads it, and MMAs run in order);
//   warps 2-5 and 6-9: the softmax of stream 0 and 1, one row per thread: the row's 128 scores read for their maximum and
//             once more for the weights, the running maximum moved only when a block's exceeds it by more than 2^8 (O is
//             then rescaled in TMEM, where no P.V of the stream can be in flight between a block's scores and its
//             weights), weights as bf16 back to TMEM, partial sums in fp32. Warps whose rows do not exist skip all of it;
//   warps 10-13 (int8): widen a code tile to bf16, exactly, one key per thread, into the operand rings, and put the
//             block's scales (the keys' times scale log2(e)) beside them: a key's scale multiplies its column of scores,
//             a value's its column of weights.
// A row tile's range ends with a partial record (unnormalised output, maximum, sum of each row) for add_kernel. With bf16 caches
// weights enter P.V as bf16 relative to the maximum in use, as in the other bf16 attention kernels; with int8 caches as
// the sum of two bf16 values (16 bits), a second P.V: the values' own rounding is then the only one that counts.
// Everything else is fp32. Every wait is bounded by time; issued loads and MMAs are drained before the CTA exits.
//
// What bounds it (d = 128, one step = two streams' blocks): the chain of a stream's step, not a unit. P lies over S, so a
// stream's next scores wait for its P.V, and its step is scores, softmax and P.V in a row: the scores are read twice, 32
// columns at a time, each read waited for, and P.V starts once all 128 weights of every row are written; the other stream
// hides part of that. With 256 rows of each of 8 kv heads a step takes 2.2 us with bf16 caches (by the slope over 32768 to
// 131072 keys), where the MMAs' reads of shared memory (192 KB at 128 bytes a clock) are 0.8 us and the exponentials (16
// a clock) 1.0, and 5.1 us with int8, whose scaled scores go back to TMEM between the two reads, whose weights enter
// twice and whose codes are widened by four warps in the order of the blocks. Whole calls on the device, 256 rows over
// 32768 keys without own keys: 50 us bf16 (34.4 GFLOP, 690 TFLOP/s, 41% of measured), 99 us int8; 64 rows: 35 us bf16
// (134 MB, 3.8 TB/s; each further 32768 keys add 18.5 us, which is HBM), 72 us int8.
#include "internal.h"
#include "common.cuh"

namespace egpt {
namespace apx {

constexpr int kBK = 128, kRowsT = 128;
constexpr uint32_t kOCol = 256;  // S0 | S1 | O0 | O1, 128 columns each; P_s in S_s
constexpr int record_size(int d) { return kRowsT * (d + 2); }  // floats: [128 rows][d], maxima, sums

template <int D, bool Q8>
struct Cfg {
  static constexpr int kHalves = D / 64;            // 64-column groups of an operand tile
  static constexpr int kHalf = kRowsT * 128;        // bytes: 128 rows x 64 bf16, one 128-byte swizzle column
  static constexpr int kTile = kHalves * kHalf;
  static constexpr int kKStages = Q8 ? 2 : 3, kVStages = 2;
  static constexpr int kRaw = kBK * D;              // bytes of a code tile
  static constexpr int kThreads = 64 + 256 + (Q8 ? 128 : 0);
  static constexpr size_t kScales = Q8 ? 2 * 2 * kBK * 4 : 0;  // two blocks' [ks scale log2(e)][vs]
  // int8: two code tiles and two blocks' scales behind two query tiles; three and four where the second tile's place is free
  static constexpr size_t kUsed = (size_t)(2 + kKStages + kVStages) * kTile + (Q8 ? 2 * kRaw : 0) + kScales + 256;
  static constexpr size_t kSlack = 768;             // alignment: the CTA's shared memory starts 1024-aligned, or nearly
  static constexpr size_t kSmem = kUsed + kSlack;
};

struct Args {
  CUtensorMap qmap;  // q bf16 [m][nq][D], box {64, group, seqs}, 128-byte swizzle
  CUtensorMap kmap;  // K bf16 or int8 [nkv][prefix_len][D] (head stride prefix_cap rows), box {64 | D, 128, 1}
  CUtensorMap vmap;
  const float *ks, *vs;  // int8: [nkv][cap]
  int64_t cap;
  float *ws;         // records [nkv][pairs][ranges][2 row tiles]
  int64_t prefix;
  int m, nkv, group;
  int seqs;          // sequences per row tile: 128 / group
  int tiles, pairs, ranges;
  float scale_log2;  // > 0
};

// Shared memory by its own addresses (a pointer that is one of two places is a generic one to the compiler).
__device__ __forceinline__ ulonglong2 lds_2x64(uint32_t at) {
  ulonglong2 r;
  asm volatile("ld.shared.v2.u64 {%0, %1}, [%2];" : "=l"(r.x), "=l"(r.y) : "r"(at));
  return r;
}
__device__ __forceinline__ uint4 lds_4x32(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at));
  return r;
}
__device__ __forceinline__ void sts_4x32(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// The barrier of the two warps that take it (both do, whatever their waits returned); -> whether both came with ok.
__device__ __forceinline__ bool both_warps(int barrier, bool ok) {
  int r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.s32 p, %2, 0;\n"
      " barrier.cta.red.and.pred q, %1, 64, p;\n selp.s32 %0, 1, 0, q;\n}"
      : "=r"(r)
      : "r"(barrier), "r"((int)ok)
      : "memory");
  return r != 0;
}
// The bf16 values of two codes: 0x43 above a byte is 128 + its low seven bits, doubled scale if the sign bit is set; the
// two parts of the byte apart are 128 + low bits and 128 or 256, and their difference is the code, exactly.
__device__ __forceinline__ uint32_t widen2(uint32_t codes, uint32_t select) {
  uint32_t r;
  const uint32_t pasted = __byte_perm(codes, 0x43434343u, select);
  // (the second part with its sign set: a sum is one instruction, a difference two)
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(pasted & 0xff7fff7fu), "r"((pasted & 0xff80ff80u) | 0x80008000u));
  return r;
}

template <int D, bool Q8>
__global__ void __launch_bounds__(Cfg<D, Q8>::kThreads, 1) attn_prefix_kernel(const __grid_constant__ Args A) {
  using C = Cfg<D, Q8>;
  constexpr int kTile = C::kTile, kHalf = C::kHalf, kKStages = C::kKStages, kVStages = C::kVStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);  // 1024-aligned operand tiles
  if ((size_t)(smem - smem_raw) > C::kSlack) {
    if (threadIdx.x == 0) set_device_error(EGPT_ERR_ALIGN);
    return;
  }
  uint8_t *sq = smem;                            // two query tiles, each of [128 rows][128 B] halves
  uint8_t *sk = sq + 2 * kTile;                  // K slots
  uint8_t *sv = sk + (size_t)kKStages * kTile;   // V slots
  uint8_t *raw0 = sv + (size_t)kVStages * kTile;  // code tiles 0, 1; the third in the second query tile's place
  float *scales = (float *)(raw0 + (Q8 ? 2 * C::kRaw : 0));
  uint64_t *bars = (uint64_t *)((uint8_t *)scales + C::kScales);
  uint64_t *q_full = bars, *k_full = q_full + 1, *k_empty = k_full + kKStages, *v_full = k_empty + kKStages;
  uint64_t *v_empty = v_full + kVStages, *s_full = v_empty + kVStages, *p_full = s_full + 2, *o_done = p_full + 2;
  uint64_t *mma_done = o_done + 2, *raw_full = mma_done + 1, *raw_empty = raw_full + 3;
  uint64_t *scale_full = raw_empty + 3;
  uint32_t *tmem_slot = (uint32_t *)(scale_full + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_wait();
  pdl_launch_dependents();
  const int range = (int)(blockIdx.x % (unsigned)A.ranges);
  const int gp = (int)(blockIdx.x / (unsigned)A.ranges);
  const int pair = gp % A.pairs, g = gp / A.pairs;
  const bool two = 2 * pair + 1 < A.tiles;  // two row tiles, else alternate blocks
  const int nb = (int)((A.prefix + kBK - 1) / kBK);
  const int b0 = (int)((int64_t)nb * range / A.ranges), n = (int)((int64_t)nb * (range + 1) / A.ranges) - b0;  // n >= 1
  const int steps[2] = {two ? n : (n + 1) / 2, two ? n : n / 2};
  int rows[2];  // rows of the stream's tile that exist
#pragma unroll
  for (int s = 0; s < 2; ++s)
    rows[s] = steps[s] ? min(A.seqs, A.m - (2 * pair + (two ? s : 0)) * A.seqs) * A.group : 0;

  if (threadIdx.x == 0) {
    gtc::mbar_init(q_full, 1);
    for (int s = 0; s < kKStages; ++s) gtc::mbar_init(k_full + s, Q8 ? 128 : 1), gtc::mbar_init(k_empty + s, 1);
    for (int s = 0; s < kVStages; ++s) gtc::mbar_init(v_full + s, Q8 ? 128 : 1), gtc::mbar_init(v_empty + s, 1);
    for (int s = 0; s < 2; ++s) {
      gtc::mbar_init(s_full + s, 1);
      gtc::mbar_init(p_full + s, max(1, (rows[s] + 31) / 32) * 32);  // every thread of the warps that have rows
      gtc::mbar_init(o_done + s, 1);
    }
    gtc::mbar_init(mma_done, 1);
    for (int s = 0; s < 3; ++s) gtc::mbar_init(raw_full + s, 1), gtc::mbar_init(raw_empty + s, 128);
    for (int s = 0; s < 4; ++s) gtc::mbar_init(scale_full + s, 128);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(apf::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  gtc::tc_fence_before();
  __syncthreads();
  gtc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int raws = two ? 2 : 3, scale_slots = two ? 2 : 4;  // code tiles in flight (K, V, K, ...), blocks with scales
  auto raw_tile = [&](int u) { return u < 2 ? raw0 + u * C::kRaw : sq + kTile; };
  auto scale_of = [&](int b) {  // [ks scale log2(e)][vs] of block b
    const int j = b % scale_slots;
    return (j < 2 ? scales : (float *)(sq + kTile + C::kRaw) - 4 * kBK) + j * 2 * kBK;
  };

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer
    if (lane == 0) {
      const unsigned qbytes = (unsigned)(A.seqs * A.group) * 128u;  // one half of a query tile
      gtc::mbar_arrive_tx(q_full, (two ? 2u : 1u) * C::kHalves * qbytes);
      for (int s = 0; s < (two ? 2 : 1); ++s)
        for (int h = 0; h < C::kHalves; ++h)
          apf::tma_load_3d(sq + s * kTile + h * kHalf, &A.qmap, 64 * h, g * A.group, (2 * pair + s) * A.seqs, q_full);
      if constexpr (Q8) {
        int u = 0;  // tile 2 b is block b's K, 2 b + 1 its V
        for (; u < 2 * n; ++u) {
          const int slot = u % raws;
          if (u >= raws && !gtc::mbar_wait(raw_empty + slot, (unsigned)((u / raws) - 1) & 1u)) break;
          gtc::mbar_arrive_tx(raw_full + slot, C::kRaw);
          apf::tma_load_3d(raw_tile(slot), u & 1 ? &A.vmap : &A.kmap, 0, (b0 + u / 2) * kBK, g, raw_full + slot);
        }
        for (int t = max(0, u - raws); t < u; ++t) gtc::mbar_drain(raw_full + t % raws, (unsigned)(t / raws) & 1u);
      } else {
        int nk = 0, nv = 0;
        auto load = [&](int b, const CUtensorMap *map, uint8_t *ring, int stages, uint64_t *full, uint64_t *empty) -> bool {
          const int slot = b % stages;
          if (b >= stages && !gtc::mbar_wait(empty + slot, (unsigned)((b / stages) - 1) & 1u)) return false;
          uint8_t *t = ring + (size_t)slot * kTile;
          gtc::mbar_arrive_tx(full + slot, kTile);
          for (int h = 0; h < C::kHalves; ++h)
            apf::tma_load_3d(t + h * kHalf, map, 64 * h, (b0 + b) * kBK, g, full + slot);
          return true;
        };
        auto load_k = [&](int b) -> bool {
          if (!load(b, &A.kmap, sk, kKStages, k_full, k_empty)) return false;
          ++nk;
          return true;
        };
        bool ok = load_k(0) && (n < 2 || load_k(1));
        for (int b = 0; b < n && ok; ++b) {  // K runs two blocks ahead of V: scores come first
          ok = load(b, &A.vmap, sv, kVStages, v_full, v_empty);
          if (ok) ++nv;
          if (ok && b + 2 < n) ok = load_k(b + 2);
        }
        for (int b = max(0, nk - kKStages); b < nk; ++b)
          gtc::mbar_drain(k_full + b % kKStages, (unsigned)(b / kKStages) & 1u);
        for (int b = max(0, nv - kVStages); b < nv; ++b)
          gtc::mbar_drain(v_full + b % kVStages, (unsigned)(b / kVStages) & 1u);
      }
      gtc::mbar_drain(q_full, 0);  // none of this CTA's copies may still be landing when it exits
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    if (lane == 0) {
      constexpr uint32_t kIdescO = (apf::kIdescO & ~(0x3fu << 17)) | ((uint32_t)(D >> 3) << 17);  // N = D
      auto block_of = [&](int s, int i) { return two ? i : 2 * i + s; };
      // with two row tiles a slot is free once stream 1's MMAs, issued after stream 0's, have read it
      auto issue_scores = [&](int s, int i) -> bool {
        const int b = block_of(s, i), slot = b % kKStages;
        if (!gtc::mbar_wait(k_full + slot, (unsigned)(b / kKStages) & 1u)) return false;
        gtc::tc_fence_after();
        const uint8_t *q = sq + (two ? s : 0) * kTile, *k = sk + (size_t)slot * kTile;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint64_t off = (uint64_t)(2 * (kk & 3));
          apf::umma(tmem + (uint32_t)(128 * s), gtc::sw128_desc(q + (kk >> 2) * kHalf) + off,
                    gtc::sw128_desc(k + (kk >> 2) * kHalf) + off, apf::kIdescS, kk > 0 ? 1u : 0u);
        }
        if (!two || s == 1) gtc::umma_commit(k_empty + slot);
        gtc::umma_commit(s_full + s);
        return true;
      };
      bool ok = gtc::mbar_wait(q_full, 0) && issue_scores(0, 0) && (!steps[1] || issue_scores(1, 0));
      for (int i = 0; i < steps[0] && ok; ++i)
        for (int s = 0; s < 2 && ok; ++s) {
          if (i >= steps[s]) continue;
          const int b = block_of(s, i), slot = b % kVStages;
          ok = gtc::mbar_wait(p_full + s, (unsigned)i & 1u) && gtc::mbar_wait(v_full + slot, (unsigned)(b / kVStages) & 1u);
          if (!ok) break;
          gtc::tc_fence_after();
          const uint8_t *v = sv + (size_t)slot * kTile;
#pragma unroll
          for (int part = 0; part < (Q8 ? 2 : 1); ++part)
#pragma unroll
            for (int kk = 0; kk < kBK / 16; ++kk)  // 16 keys per step: 8 columns of P, 16 rows of 128 bytes of V
              apf::umma_ts(tmem + kOCol + (uint32_t)(128 * s),
                           tmem + (uint32_t)(128 * s + (Q8 ? 32 * (kk / 2) + 16 * part + 8 * (kk % 2) : 8 * kk)),
                           apf::sw128_mn_desc(v + (size_t)kk * 16 * 128), kIdescO, (i > 0 || part > 0 || kk > 0) ? 1u : 0u);
          if (!two || s == 1) gtc::umma_commit(v_empty + slot);
          if (i + 1 < steps[s]) ok = issue_scores(s, i + 1);
          else gtc::umma_commit(o_done + s);
        }
      gtc::umma_commit(mma_done);  // completes once every MMA issued above has finished
      gtc::mbar_drain(mma_done, 0);
    }
  } else if (warp < 10) {
    // ---------------------------------------------------------------- softmax: one row per thread
    const int s = (warp - 2) >> 2;
    const int quarter = warp & 3;  // TMEM lanes this warp may access: 32 (warp % 4) ..
    const int row = 32 * quarter + lane;
    if (32 * quarter < rows[s]) {
      const uint32_t ts = tmem + ((uint32_t)(32 * quarter) << 16) + (uint32_t)(128 * s), to = ts + kOCol;
      float m_run = -INFINITY, l_sum = 0.f;
      bool ok = true;
      for (int i = 0; i < steps[s] && ok; ++i) {
        const int b = two ? i : 2 * i + s;
        ok = apf::warp_wait(s_full + s, (unsigned)i & 1u);
        // (a slot's next phase waits for the P.V of the block that holds it now)
        if (Q8) ok = ok && apf::warp_wait(scale_full + b % scale_slots, (unsigned)(b / scale_slots) & 1u);
        if (!ok) break;
        gtc::tc_fence_after();
        const uint32_t ks = Q8 ? smem_u32(scale_of(b)) : 0u, vs = ks + kBK * 4;
        const uint64_t one2 = f2_pack(A.scale_log2, A.scale_log2);
        const int left = (int)min((int64_t)kBK, A.prefix - (int64_t)(b0 + b) * kBK);
        auto mask = [&](int c, uint32_t *sc) {  // -inf past the prefix
          if (left < c + 32) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (c + e >= left) sc[e] = __float_as_uint(-INFINITY);
          }
        };
        // scores to log2 units in place: bf16 later, in one fma with the maximum
        auto scaled = [&](int c, uint32_t *sc) {
          if constexpr (Q8) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const ulonglong2 f = lds_2x64(ks + (uint32_t)(c + e) * 4);
              const float2 x = f2_unpack(f2_mul(f2_pack(__uint_as_float(sc[e]), __uint_as_float(sc[e + 1])), f.x));
              const float2 y = f2_unpack(f2_mul(f2_pack(__uint_as_float(sc[e + 2]), __uint_as_float(sc[e + 3])), f.y));
              sc[e] = __float_as_uint(x.x), sc[e + 1] = __float_as_uint(x.y);
              sc[e + 2] = __float_as_uint(y.x), sc[e + 3] = __float_as_uint(y.y);
            }
          }
          mask(c, sc);
        };
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < kBK; c += 32) {
          uint32_t sc[32];
          apf::tmem_ld32(ts + (uint32_t)c, sc);
          apf::tmem_wait_ld();
          scaled(c, sc);
#pragma unroll
          for (int e = 0; e < 32; ++e) mx[e & 3] = fmaxf(mx[e & 3], __uint_as_float(sc[e]));
          if (Q8) apf::tmem_st32(ts + (uint32_t)c, sc);  // scaled: the second pass needs no factors from shared memory
        }
        if (Q8) apf::tmem_wait_st();
        const float bm = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * (Q8 ? 1.f : A.scale_log2);
        float alpha = 1.f;
        if (bm > m_run + apf::kStale) {
          alpha = apf::ex2(m_run - bm);  // 0 on the first block
          m_run = bm;
        }
        if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
          // the stream's P.V so far has finished: the scores that were just read completed after it
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            apf::tmem_ld32(to + (uint32_t)c, o);
            apf::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            apf::tmem_st32(to + (uint32_t)c, o);
          }
        }
        const float base = m_run == -INFINITY ? 0.f : m_run;  // (every score so far is -inf: their weights are zeros)
        const uint64_t nm2 = f2_pack(-base, -base);
        uint64_t sum[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
        // weights of 32 keys over scores that have been read: bf16 in columns c / 2 ..; int8 in the 32 columns of their
        // own scores, the second parts in the upper 16
        auto weights = [&](int c, const uint32_t *sc) {
          uint32_t pk[16], pl[Q8 ? 16 : 1];
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            ulonglong2 vf = make_ulonglong2(0ull, 0ull);
            if constexpr (Q8) vf = lds_2x64(vs + (uint32_t)(c + e) * 4);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int k = e + 2 * h;
              const uint64_t raw = f2_pack(__uint_as_float(sc[k]), __uint_as_float(sc[k + 1]));
              const float2 x = f2_unpack(Q8 ? f2_add(raw, nm2) : f2_fma(raw, one2, nm2));
              float2 w = make_float2(apf::ex2(x.x), apf::ex2(x.y));
              sum[h] = f2_add(sum[h], f2_pack(w.x, w.y));
              if constexpr (Q8) w = f2_unpack(f2_mul(f2_pack(w.x, w.y), h ? vf.y : vf.x));
              pk[k / 2] = gtc::pack_bf16x2(w.x, w.y);
              if constexpr (Q8) pl[k / 2] = gtc::pack_bf16x2(w.x - bf16_lo(pk[k / 2]), w.y - bf16_hi(pk[k / 2]));
            }
          }
          apf::tmem_st16(ts + (uint32_t)(Q8 ? c : c / 2), pk);
          if constexpr (Q8) apf::tmem_st16(ts + (uint32_t)(c + 16), pl);
        };
#pragma unroll
        for (int c = 0; c < kBK; c += 32) {
          uint32_t sc[32];
          apf::tmem_ld32(ts + (uint32_t)c, sc);
          apf::tmem_wait_ld();
          if (!Q8) mask(c, sc);
          weights(c, sc);
        }
        const float2 t = f2_unpack(f2_add(sum[0], sum[1]));
        l_sum = l_sum * alpha + (t.x + t.y);
        apf::tmem_wait_st();
        gtc::tc_fence_before();
        gtc::mbar_arrive(p_full + s);
      }
      // ---- the record. Once both streams are done the operand tiles are free: a row goes through a place of its own
      // there and leaves in one bulk copy; alternate blocks' two states are added up first. Where a wait gave up the sums
      // are NaN, and with them the outputs: what the record held before is never added up.
      ok = ok && apf::warp_wait(o_done, 0) && (!steps[1] || apf::warp_wait(o_done + 1, 0));
      gtc::tc_fence_after();
      constexpr int kPitch = D + 4;  // floats of a staged row
      float *stage = (float *)sk + (size_t)(two ? 4 * s + quarter : quarter) * 32 * kPitch;
      const bool merge = !two && steps[1];
      float f0 = 1.f, f1 = 0.f;
      const float *other = stage + lane * kPitch;
      if (merge) {
        // stream 1's state to shared memory (maximum and sum in the row's padding), stream 0 takes it
        if (s == 1 && ok) {
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            apf::tmem_ld32(to + (uint32_t)c, o);
            apf::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *(uint4 *)(stage + lane * kPitch + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
          *(float2 *)(stage + lane * kPitch + D) = make_float2(m_run, l_sum);
        }
        ok = both_warps(1 + quarter, ok);
        if (s == 0 && ok) {
          const float2 ml = *(const float2 *)(other + D);
          const float mx = fmaxf(m_run, ml.x), mz = mx == -INFINITY ? 0.f : mx;
          f0 = apf::ex2(m_run - mz), f1 = apf::ex2(ml.x - mz);
          m_run = mx, l_sum = l_sum * f0 + ml.y * f1;
        }
      }
      if (!(merge && s == 1)) {
        float *rec = A.ws + ((int64_t)blockIdx.x * 2 + s) * record_size(D);
        if (ok) {
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            apf::tmem_ld32(to + (uint32_t)c, o);
            apf::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              float *at = stage + lane * kPitch + c + e;
              float4 v = make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]),
                                     __uint_as_float(o[e + 3]));
              if (merge) {
                const float4 w = *(const float4 *)at;
                v = make_float4(v.x * f0 + w.x * f1, v.y * f0 + w.y * f1, v.z * f0 + w.z * f1, v.w * f0 + w.w * f1);
              }
              *(float4 *)at = v;
            }
          }
          if (row < rows[s]) {  // the row's own copy engine transfer
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(rec + row * D),
                         "r"(smem_u32(stage + lane * kPitch)), "n"(D * 4)
                         : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
          }
        }
        rec[kRowsT * D + row] = m_run;
        rec[kRowsT * D + kRowsT + row] = ok ? l_sum : NAN;
      }
    }
  } else if constexpr (Q8) {
    // ---------------------------------------------------------------- widening: one key per thread
    const int r = (int)threadIdx.x - 320;
    auto widen = [&](int u, uint8_t *dst) -> bool {  // code tile u to an operand tile
      const int slot = u % raws;
      if (!gtc::mbar_wait(raw_full + slot, (unsigned)(u / raws) & 1u)) return false;
      const uint32_t src = smem_u32(raw_tile(slot)) + r * D, to = smem_u32(dst) + r * 128;
      const int swz = D == 128 ? (r & 7) : ((r >> 1) & 3);  // the map's 128- or 64-byte swizzle
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        const uint4 w = lds_4x32(src + ((c ^ swz) * 16));
        const uint32_t half = to + (c >> 2) * kHalf;
        const int cc = 2 * (c & 3);
        sts_4x32(half + ((cc ^ (r & 7)) * 16), widen2(w.x, 0x4140), widen2(w.x, 0x4342), widen2(w.y, 0x4140),
                 widen2(w.y, 0x4342));
        sts_4x32(half + (((cc + 1) ^ (r & 7)) * 16), widen2(w.z, 0x4140), widen2(w.z, 0x4342), widen2(w.w, 0x4140),
                 widen2(w.w, 0x4342));
      }
      gtc::mbar_arrive(raw_empty + slot);
      return true;
    };
    auto scale_at = [&](const float *p, int b) {
      const int64_t key = (int64_t)(b0 + b) * kBK + r;
      return b < n && key < A.prefix ? p[g * A.cap + key] : 0.f;
    };
    float next_ks = scale_at(A.ks, 0), next_vs = scale_at(A.vs, 0);
    for (int b = 0; b < n; ++b) {
      const float ks = next_ks * A.scale_log2, vs = next_vs;
      next_ks = scale_at(A.ks, b + 1), next_vs = scale_at(A.vs, b + 1);
      const int kslot = b % kKStages, vslot = b % kVStages;
      // an operand slot is free once its MMAs have run, a scale slot once the P.V of its last block has: with two of
      // them that is block b - 2's, with four b - 4's, which V(b - 2) has waited for
      if (scale_slots == 2 && b >= 2 && !gtc::mbar_wait(v_empty + vslot, (unsigned)((b / kVStages) - 1) & 1u)) break;
      float *sc = scale_of(b);
      sc[r] = ks;
      sc[kBK + r] = vs;
      gtc::mbar_arrive(scale_full + b % scale_slots);
      if (b >= kKStages && !gtc::mbar_wait(k_empty + kslot, (unsigned)((b / kKStages) - 1) & 1u)) break;
      if (!widen(2 * b, sk + (size_t)kslot * kTile)) break;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      gtc::mbar_arrive(k_full + kslot);
      if (b >= kVStages && !gtc::mbar_wait(v_empty + vslot, (unsigned)((b / kVStages) - 1) & 1u)) break;
      if (!widen(2 * b + 1, sv + (size_t)vslot * kTile)) break;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      gtc::mbar_arrive(v_full + vslot);
    }
  }
  gtc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    gtc::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(apf::kTmemCols) : "memory");
  }
}

// Row tiles, their pairs, and key ranges per kv head and pair: about one CTA per SM, at least four blocks to a range
// (a range costs about 5 us besides its blocks, and its record has to be added up).
struct Shape {
  int seqs, tiles, pairs, ranges;
};
static Shape shape_of(int64_t m, int group, int nkv, int64_t prefix) {
  Shape s;
  s.seqs = kRowsT / group;
  s.tiles = (int)((m + s.seqs - 1) / s.seqs);
  s.pairs = (s.tiles + 1) / 2;
  const int64_t blocks = (prefix + kBK - 1) / kBK;
  s.ranges = (int)std::max<int64_t>(1, std::min<int64_t>(num_sms() / ((int64_t)nkv * s.pairs), (blocks + 3) / 4));
  return s;
}
// Floats of the records of any prefix: as many ranges as the SMs allow.
static size_t record_floats(int64_t m, int group, int nkv, int d) {
  const Shape s = shape_of(m, group, nkv, (int64_t)1 << 40);
  return (size_t)nkv * s.pairs * s.ranges * 2 * record_size(d);
}

template <int D, bool Q8>
static cudaError_t launch(Args &A, const void *q, int64_t ldq, const void *k, const void *v, const Shape &sh,
                          cudaStream_t st, bool pdl, bool &maps_ok) {
  using C = Cfg<D, Q8>;
  auto fn = df::encode_fn();
  maps_ok = fn != nullptr;
  if (!fn) return cudaSuccess;
  const cuuint32_t ones[3] = {1, 1, 1};
  const cuuint64_t qdims[3] = {D, (cuuint64_t)A.nkv * A.group, (cuuint64_t)A.m};
  const cuuint64_t qstrides[2] = {D * 2, (cuuint64_t)ldq * 2};
  const cuuint32_t qbox[3] = {64, (cuuint32_t)A.group, (cuuint32_t)sh.seqs};
  const int esz = Q8 ? 1 : 2;
  const cuuint64_t kdims[3] = {D, (cuuint64_t)A.prefix, (cuuint64_t)A.nkv};
  const cuuint64_t kstrides[2] = {(cuuint64_t)D * esz, (cuuint64_t)A.cap * D * esz};
  const cuuint32_t kbox[3] = {Q8 ? D : 64, kBK, 1};
  auto encode = [&](CUtensorMap *map, bool codes, const void *p, const cuuint64_t *dims, const cuuint64_t *strides,
                    const cuuint32_t *box) {
    return fn(map, codes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(p), dims,
              strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
              codes && D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  maps_ok = encode(&A.qmap, false, q, qdims, qstrides, qbox) && encode(&A.kmap, Q8, k, kdims, kstrides, kbox) &&
            encode(&A.vmap, Q8, v, kdims, kstrides, kbox);
  if (!maps_ok) return cudaSuccess;
  static int configured[64] = {0};  // the shared-memory opt-in, per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(attn_prefix_kernel<D, Q8>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)C::kSmem);
    if (e != cudaSuccess) return e;
    configured[dev] = 1;
  }
  A.seqs = sh.seqs, A.tiles = sh.tiles, A.pairs = sh.pairs, A.ranges = sh.ranges;
  return launch_kernel((const void *)attn_prefix_kernel<D, Q8>, dim3((unsigned)(A.nkv * sh.pairs * sh.ranges)),
                       dim3(C::kThreads), C::kSmem, st, pdl, A);
}

}  // namespace apx
}  // namespace egpt
