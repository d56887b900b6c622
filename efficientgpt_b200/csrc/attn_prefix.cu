// The shared prefix's part of egpt_attn_shared_prefix on the 5th-generation tensor cores (tcgen05): bf16 caches, head_dim
// 128, batches of more query rows than the mma.sync kernel's tiles are good for (attn_q8.cu has the rule).
//
// The (sequence, head) rows of a kv head, up to 128 of them, are the M of the MMAs: row r of tile t is head r % group of
// sequence t * seqs + r / group. A CTA of 320 threads owns one kv head, one pair of row tiles and one range of 128-key
// blocks, and runs two streams, each with 128 columns of TMEM for scores and 128 for its output:
//   two row tiles:  both streams take every block, one tile each, so a block is loaded once for 256 rows;
//   one row tile:   the streams take alternate blocks of the same rows.
// Either way one stream's softmax runs under the other's MMAs. Roles:
//   warp 0    lane 0 issues the TMA loads (this GPU's memory, no multicast): the query tiles, then K blocks into a 3-slot
//             ring and V blocks into a 2-slot ring, 128-byte swizzle; the cache maps end at the prefix's last key;
//   warp 1    allocates TMEM; lane 0 issues S = Q K^T and O += P V, P read from TMEM where the scores were (the next
//             block's scores of the stream are issued after the P.V that reads it, and MMAs run in order);
//   warps 2-5 and 6-9: the softmax of stream 0 and 1, one row per thread: the row's 128 scores read for their maximum and once
//             more for the weights, the running maximum (moved only when a block's exceeds it by more than 2^8; O is then rescaled in TMEM, where no P.V
//             of the stream can be in flight between a block's scores and its weights), weights as bf16 back to
//             TMEM, partial sums in fp32. Warps whose rows do not exist skip all of it.
// A stream ends with a partial record (unnormalised output, maximum, sum of each row) for combine_kernel. Weights
// enter P.V as bf16 relative to the maximum in use, as in the other bf16 attention kernels; everything else is fp32.
// Every wait is bounded; issued loads and MMAs are drained before the CTA exits.
#include "internal.h"
#include "common.cuh"

namespace egpt {
namespace apx {

using apf::kHalf;
using apf::kTile;

constexpr int kD = 128, kBK = 128, kRowsT = 128;
constexpr int kKStages = 3, kVStages = 2;
constexpr int kThreads = 64 + 2 * 128;
constexpr uint32_t kOCol = 256;  // S0 | S1 | O0 | O1, 128 columns each; P_s in the first 64 columns of S_s
constexpr size_t kSmem = 1024 /* alignment slack */ + (size_t)(2 + kKStages + kVStages) * kTile + 256;
constexpr int kRecord = kRowsT * (kD + 2);  // floats: [128 rows][128], maxima, sums

struct Args {
  CUtensorMap qmap;  // q bf16 [m][nq][128], box {64, group, seqs}, 128-byte swizzle
  CUtensorMap kmap;  // K bf16 [nkv][prefix_len][128] (head stride prefix_cap rows), box {64, 128, 1}
  CUtensorMap vmap;
  float *ws;         // records [nkv][pairs][ranges][2 streams]
  int64_t prefix;
  int m, nkv, group;
  int seqs;          // sequences per row tile: 128 / group
  int tiles, pairs, ranges;
  float scale_log2;  // > 0
};

__global__ void __launch_bounds__(kThreads, 1) attn_prefix_kernel(const __grid_constant__ Args A) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);  // 1024-aligned operand tiles
  uint8_t *sq = smem;                            // two query tiles, each two [128 rows][128 B] halves
  uint8_t *sk = sq + 2 * kTile;                  // K slots
  uint8_t *sv = sk + (size_t)kKStages * kTile;   // V slots
  uint64_t *bars = (uint64_t *)(sv + (size_t)kVStages * kTile);
  uint64_t *q_full = bars, *k_full = q_full + 1, *k_empty = k_full + kKStages, *v_full = k_empty + kKStages;
  uint64_t *v_empty = v_full + kVStages, *s_full = v_empty + kVStages, *p_full = s_full + 2, *o_done = p_full + 2;
  uint64_t *mma_done = o_done + 2;
  uint32_t *tmem_slot = (uint32_t *)(mma_done + 1);
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
    for (int s = 0; s < kKStages; ++s) gtc::mbar_init(k_full + s, 1), gtc::mbar_init(k_empty + s, 1);
    for (int s = 0; s < kVStages; ++s) gtc::mbar_init(v_full + s, 1), gtc::mbar_init(v_empty + s, 1);
    for (int s = 0; s < 2; ++s) {
      gtc::mbar_init(s_full + s, 1);
      gtc::mbar_init(p_full + s, max(1, (rows[s] + 31) / 32) * 32);  // every thread of the warps that have rows
      gtc::mbar_init(o_done + s, 1);
    }
    gtc::mbar_init(mma_done, 1);
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

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer
    if (lane == 0) {
      const unsigned qbytes = (unsigned)(A.seqs * A.group) * 128u;  // one half of a query tile
      gtc::mbar_arrive_tx(q_full, (two ? 4u : 2u) * qbytes);
      for (int s = 0; s < (two ? 2 : 1); ++s)
        for (int h = 0; h < 2; ++h)
          apf::tma_load_3d(sq + s * kTile + h * kHalf, &A.qmap, 64 * h, g * A.group, (2 * pair + s) * A.seqs, q_full);
      int nk = 0, nv = 0;
      auto load = [&](int b, const CUtensorMap *map, uint8_t *ring, int stages, uint64_t *full, uint64_t *empty) -> bool {
        const int slot = b % stages;
        if (b >= stages && !gtc::mbar_wait(empty + slot, (unsigned)((b / stages) - 1) & 1u)) return false;
        uint8_t *t = ring + (size_t)slot * kTile;
        gtc::mbar_arrive_tx(full + slot, kTile);
        apf::tma_load_3d(t, map, 0, (b0 + b) * kBK, g, full + slot);
        apf::tma_load_3d(t + kHalf, map, 64, (b0 + b) * kBK, g, full + slot);
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
      // none of this CTA's copies may still be landing when it exits
      gtc::mbar_drain(q_full, 0);
      for (int b = max(0, nk - kKStages); b < nk; ++b) gtc::mbar_drain(k_full + b % kKStages, (unsigned)(b / kKStages) & 1u);
      for (int b = max(0, nv - kVStages); b < nv; ++b) gtc::mbar_drain(v_full + b % kVStages, (unsigned)(b / kVStages) & 1u);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    if (lane == 0) {
      auto block_of = [&](int s, int i) { return two ? i : 2 * i + s; };
      // with two row tiles a slot is free once stream 1's MMAs, issued after stream 0's, have read it
      auto issue_scores = [&](int s, int i) -> bool {
        const int b = block_of(s, i), slot = b % kKStages;
        if (!gtc::mbar_wait(k_full + slot, (unsigned)(b / kKStages) & 1u)) return false;
        gtc::tc_fence_after();
        const uint8_t *q = sq + (two ? s : 0) * kTile, *k = sk + (size_t)slot * kTile;
#pragma unroll
        for (int kk = 0; kk < kD / 16; ++kk) {
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
          for (int kk = 0; kk < kBK / 16; ++kk)  // 16 keys per step: 8 columns of P, 16 rows of 128 bytes of V
            apf::umma_ts(tmem + kOCol + (uint32_t)(128 * s), tmem + (uint32_t)(128 * s + 8 * kk),
                         apf::sw128_mn_desc(v + (size_t)kk * 16 * 128), apf::kIdescO, (i > 0 || kk > 0) ? 1u : 0u);
          if (!two || s == 1) gtc::umma_commit(v_empty + slot);
          if (i + 1 < steps[s]) ok = issue_scores(s, i + 1);
          else gtc::umma_commit(o_done + s);
        }
      gtc::umma_commit(mma_done);  // completes once every MMA issued above has finished
      gtc::mbar_drain(mma_done, 0);
    }
  } else {
    // ---------------------------------------------------------------- softmax: one row per thread
    const int s = (warp - 2) >> 2;
    const int quarter = warp & 3;  // TMEM lanes this warp may access: 32 (warp % 4) ..
    const int row = 32 * quarter + lane;
    if (32 * quarter < rows[s]) {
      const uint32_t ts = tmem + ((uint32_t)(32 * quarter) << 16) + (uint32_t)(128 * s), to = ts + kOCol;
      float m_run = -INFINITY, l_sum = 0.f;
      bool ok = true;
      for (int i = 0; i < steps[s] && ok; ++i) {
        ok = apf::warp_wait(s_full + s, (unsigned)i & 1u);
        if (!ok) break;
        gtc::tc_fence_after();
        const int left = (int)min((int64_t)kBK, A.prefix - (int64_t)(b0 + (two ? i : 2 * i + s)) * kBK);
        auto load_scores = [&](int c, uint32_t *sc) {  // 32 of the row's scores; -inf past the prefix
          apf::tmem_ld32(ts + (uint32_t)c, sc);
          apf::tmem_wait_ld();
          if (left < c + 32) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (c + e >= left) sc[e] = __float_as_uint(-INFINITY);
          }
        };
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < kBK; c += 32) {
          uint32_t sc[32];
          load_scores(c, sc);
#pragma unroll
          for (int e = 0; e < 32; ++e) mx[e & 3] = fmaxf(mx[e & 3], __uint_as_float(sc[e]));
        }
        const float bm = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * A.scale_log2;
        float alpha = 1.f;
        if (bm > m_run + apf::kStale) {
          alpha = apf::ex2(m_run - bm);  // 0 on the first block
          m_run = bm;
        }
        if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
          // the stream's P.V so far has finished: the scores that were just read completed after it
#pragma unroll
          for (int c = 0; c < kD; c += 32) {
            uint32_t o[32];
            apf::tmem_ld32(to + (uint32_t)c, o);
            apf::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            apf::tmem_st32(to + (uint32_t)c, o);
          }
        }
        const uint64_t sc2 = apf::f2_pack(A.scale_log2, A.scale_log2), nm2 = apf::f2_pack(-m_run, -m_run);
        uint64_t sum[2] = {apf::f2_pack(0.f, 0.f), apf::f2_pack(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < kBK; c += 32) {
          uint32_t sc[32], pk[16];
          load_scores(c, sc);
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 x = apf::f2_unpack(apf::f2_fma(
                apf::f2_pack(__uint_as_float(sc[e]), __uint_as_float(sc[e + 1])), sc2, nm2));
            const float p0 = apf::ex2(x.x), p1 = apf::ex2(x.y);
            sum[(e >> 1) & 1] = apf::f2_add(sum[(e >> 1) & 1], apf::f2_pack(p0, p1));
            pk[e / 2] = gtc::pack_bf16x2(p0, p1);
          }
          apf::tmem_st16(ts + (uint32_t)(c / 2), pk);  // over scores that have been read
        }
        const float2 t = apf::f2_unpack(apf::f2_add(sum[0], sum[1]));
        l_sum = l_sum * alpha + (t.x + t.y);
        apf::tmem_wait_st();
        gtc::tc_fence_before();
        gtc::mbar_arrive(p_full + s);
      }
      if (ok && apf::warp_wait(o_done + s, 0)) {
        gtc::tc_fence_after();
        float *rec = A.ws + ((int64_t)blockIdx.x * 2 + s) * kRecord;
#pragma unroll
        for (int c = 0; c < kD; c += 32) {
          uint32_t o[32];
          apf::tmem_ld32(to + (uint32_t)c, o);
          apf::tmem_wait_ld();
          if (row < rows[s]) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *(uint4 *)(rec + row * kD + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        rec[kRowsT * kD + row] = m_run;
        rec[kRowsT * kD + kRowsT + row] = l_sum;
      }
    }
    if (!steps[s]) {  // a range of one block: the second stream has no record to add
      float *rec = A.ws + ((int64_t)blockIdx.x * 2 + s) * kRecord;
      rec[kRowsT * kD + row] = -INFINITY;
      rec[kRowsT * kD + kRowsT + row] = 0.f;
    }
  }
  gtc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    gtc::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(apf::kTmemCols) : "memory");
  }
}

// Row tiles, their pairs, and key ranges per kv head and pair: about one CTA per SM, at least two blocks to a range.
struct Shape {
  int seqs, tiles, pairs, ranges;
};
static Shape shape_of(int64_t m, int group, int nkv, int64_t prefix) {
  Shape s;
  s.seqs = kRowsT / group;
  s.tiles = (int)((m + s.seqs - 1) / s.seqs);
  s.pairs = (s.tiles + 1) / 2;
  const int64_t blocks = (prefix + kBK - 1) / kBK;
  s.ranges = (int)std::max<int64_t>(1, std::min<int64_t>(num_sms() / ((int64_t)nkv * s.pairs), (blocks + 1) / 2));
  return s;
}
// Floats of the records of any prefix: as many ranges as the SMs allow.
static size_t record_floats(int64_t m, int group, int nkv) {
  const Shape s = shape_of(m, group, nkv, (int64_t)1 << 40);
  return (size_t)nkv * s.pairs * s.ranges * 2 * kRecord;
}

static cudaError_t launch(Args &A, const void *q, int64_t ldq, const void *k, const void *v, int64_t prefix_cap,
                          const Shape &sh, cudaStream_t st, bool pdl, bool &maps_ok) {
  auto fn = df::encode_fn();
  maps_ok = fn != nullptr;
  if (!fn) return cudaSuccess;
  const cuuint32_t ones[3] = {1, 1, 1};
  const cuuint64_t qdims[3] = {kD, (cuuint64_t)A.nkv * A.group, (cuuint64_t)A.m};
  const cuuint64_t qstrides[2] = {kD * 2, (cuuint64_t)ldq * 2};
  const cuuint32_t qbox[3] = {64, (cuuint32_t)A.group, (cuuint32_t)sh.seqs};
  const cuuint64_t kdims[3] = {kD, (cuuint64_t)A.prefix, (cuuint64_t)A.nkv};
  const cuuint64_t kstrides[2] = {kD * 2, (cuuint64_t)prefix_cap * kD * 2};
  const cuuint32_t kbox[3] = {64, kBK, 1};
  auto encode = [&](CUtensorMap *map, const void *p, const cuuint64_t *dims, const cuuint64_t *strides,
                    const cuuint32_t *box) {
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(p), dims, strides, box, ones,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  maps_ok = encode(&A.qmap, q, qdims, qstrides, qbox) && encode(&A.kmap, k, kdims, kstrides, kbox) &&
            encode(&A.vmap, v, kdims, kstrides, kbox);
  if (!maps_ok) return cudaSuccess;
  static int configured[64] = {0};  // the shared-memory opt-in, per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(attn_prefix_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
    if (e != cudaSuccess) return e;
    configured[dev] = 1;
  }
  A.seqs = sh.seqs, A.tiles = sh.tiles, A.pairs = sh.pairs, A.ranges = sh.ranges;
  return launch_kernel((const void *)attn_prefix_kernel, dim3((unsigned)(A.nkv * sh.pairs * sh.ranges)), dim3(kThreads),
                       kSmem, st, pdl, A);
}

}  // namespace apx
}  // namespace egpt
