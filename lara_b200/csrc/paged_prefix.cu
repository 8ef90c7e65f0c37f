// The shared part of a decode behind a prefix that the batch has in common
// (lara_gqa_decode_shared), on the 5th-generation tensor cores.
//
// For each kv head the G query heads of all sequences are the rows of one
// attention over the prefix: tiles of floor(128 / G) sequences (rows = TMEM
// lanes) against tiles of 128 tokens, as two streams in ping-pong, so that the
// tensor core works on one while the other's softmax runs.  kPair: the streams
// are two row tiles and share every K/V tile; otherwise (one row tile) they are
// the even and the odd tokens tiles of the same rows, joined at the end.
//
//   warp 9 (TMA)   : the row tiles' queries, then K and V tiles, each through a
//                    ring of its own (K is free when its scores are there, long
//                    before V), a page or a piece of one per copy.
//   warp 8 (MMA)   : step i belongs to stream i % 2: PV(i), S(i + 2), ...
//                      S = Q K^T  (both from shared memory, fp32 in TMEM)
//                      O += P V   (P from TMEM as the sum of two bf16 numbers)
//   warps 0-7      : softmax, two threads to a row: online in the log2 domain,
//                    the reference moves when a score passes it by 2^8.
//
// A CTA takes a range of token tiles of one (kv head, row tiles) and leaves
// (reference, sum, unnormalised output) of its rows for the join.  Every wait is
// bounded; on a timeout the CTA flags the status word, drains its own work and
// returns.
#include <cuda.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "paged.cuh"
#include "tcgen05.cuh"

namespace lara {

using namespace tc;
using namespace paged;

namespace {

constexpr int kTileM = 128, kTileN = 128;
constexpr int kSoftmaxWarps = 8, kMmaWarp = 8, kTmaWarp = 9, kThreads = 320;
constexpr float kRescaleThreshold = 8.0f;
constexpr uint32_t kTmemCols = 512;  // S_0 | S_1 | O_0 | O_1, 128 columns each

template <int D, bool kPair>
struct Cfg {
  static constexpr int kHalves = D / 64;            // 128-byte-swizzled parts of a row
  static constexpr int kHalfBytes = 128 * 128;      // [128 rows][64 bf16]
  static constexpr int kTileBytes = kHalves * kHalfBytes;
  static constexpr int kQTiles = kPair ? 2 : 1;
  static constexpr int kKStages = D == 128 ? (kPair ? 2 : 3) : 4;
  static constexpr int kVStages = D == 128 ? 2 : 4;
  static constexpr int kKOff = kQTiles * kTileBytes;
  static constexpr int kVOff = kKOff + kKStages * kTileBytes;
  static constexpr int kBarOff = kVOff + kVStages * kTileBytes;
  static constexpr int kRedOff = kBarOff + 256;     // row maxima and sums of the pairs [2][2][128] floats
  static constexpr int kSmem = kRedOff + 2 * 2 * kTileM * 4 + 1024;
};

struct Bars {
  uint64_t q_full;
  uint64_t k_full[4], k_empty[4];
  uint64_t v_full[4], v_empty[4];
  uint64_t s_full[2], p_full[2], o_full[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
  int k_issued, v_issued;
};
static_assert(sizeof(Bars) <= 256, "barrier block");

struct PrefixArgs {
  const int32_t* table;  // the prefix's pages
  int tokens, batch, n_q_heads, n_kv_heads, group;
  int seqs;              // sequences of a row tile
  int units;             // row tiles (pairs of them) of a kv head
  int splits;
  int page_log2, num_pages;
  float scale_log2;
  float2* ml;            // [splits][rows] (reference, sum)
  float* acc;            // [splits][rows][D]
  int* status;
};

template <int D, bool kPair>
__global__ void __launch_bounds__(kThreads, 1)
    prefix_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PrefixArgs a) {
  using C = Cfg<D, kPair>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + (-smem_addr(smem_raw) & 1023);
  Bars* const bars = reinterpret_cast<Bars*>(smem + C::kBarOff);
  volatile int* const abort = &bars->abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x % a.splits, unit = blockIdx.x / a.splits;
  const int kvh = unit / a.units, b0 = unit % a.units * (C::kQTiles * a.seqs);
  const int all_tiles = (a.tokens + kTileN - 1) / kTileN;
  const int j0 = (int)((long long)split * all_tiles / a.splits);
  const int ntiles = (int)((long long)(split + 1) * all_tiles / a.splits) - j0;  // at least 1
  // step i: stream i & 1, tile i / 2 (pair) or i
  const int steps = kPair ? 2 * ntiles : ntiles;
  auto tile_of = [](int i) { return kPair ? i >> 1 : i; };

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    for (int s = 0; s < 4; ++s) {
      mbar_init(&bars->k_full[s], 1);
      mbar_init(&bars->k_empty[s], 1);
      mbar_init(&bars->v_full[s], 1);
      mbar_init(&bars->v_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars->s_full[t], 1);
      mbar_init(&bars->p_full[t], kSoftmaxWarps * 32);
      mbar_init(&bars->o_full[t], 1);
    }
    mbar_init(&bars->drain, 1);
    bars->abort = 0;
    bars->k_issued = bars->v_issued = 0;
    mbar_fence_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&bars->tmem_base)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  grid_dependency_wait();
  // the pass over the own tokens reads nothing of this kernel's and may start where there is room
  allow_dependent_launch();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  if (warp == kTmaWarp) {
    // ---------------------------------------------------------------- TMA
    const int log2 = a.page_log2, piece = min(kTileN, 1 << log2), pieces = kTileN / piece;
    if (lane == 0) {
      const uint32_t q_bytes = (uint32_t)(C::kQTiles * C::kHalves * a.seqs * a.group * 128);
      mbar_arrive_expect_tx(&bars->q_full, q_bytes);
      for (int t = 0; t < C::kQTiles; ++t)
        for (int x = 0; x < C::kHalves; ++x)
          tma_load_4d(smem + t * C::kTileBytes + x * C::kHalfBytes, &tm_q, 64 * x, 0, kvh, b0 + t * a.seqs,
                      &bars->q_full);
    }
    // lane i copies piece i of every tile; its page is looked up a tile ahead.  Behind the
    // prefix's end a page that is not there: the copy writes zeros
    auto page_of = [&](int j) {
      const int tok = (j0 + j) * kTileN + lane * piece;
      if (j >= ntiles || lane >= pieces || tok >= a.tokens) return a.num_pages;
      int pg = __ldg(a.table + (tok >> log2));
      if ((unsigned)pg >= (unsigned)a.num_pages) {
        atomicOr(a.status, kDevBadPage);
        pg = 0;
      }
      return pg;
    };
    auto load = [&](const CUtensorMap* map, uint8_t* to, uint64_t* full, uint64_t* empty, int j, int stages, int pg) {
      int good = 1;
      if (lane == 0) {
        if (j >= stages && !wait_or_abort(empty, ((j / stages) - 1) & 1, abort)) good = 0;
        if (good) mbar_arrive_expect_tx(full, C::kTileBytes);
      }
      if (!__shfl_sync(0xffffffffu, good, 0)) return false;
      if (lane < pieces) {
        const int row = (j0 + j) * kTileN & ((1 << log2) - 1);  // 0 where pages are smaller than a tile
        for (int x = 0; x < C::kHalves; ++x)
          tma_load_4d(to + x * C::kHalfBytes + lane * piece * 128, map, 64 * x, row, kvh, pg, full);
      }
      return true;
    };
    int pg = page_of(0);
    for (int j = 0; j < ntiles; ++j) {
      const int next = page_of(j + 1), ks = j % C::kKStages, vs = j % C::kVStages;
      if (!load(&tm_k, smem + C::kKOff + ks * C::kTileBytes, &bars->k_full[ks], &bars->k_empty[ks], j, C::kKStages, pg))
        break;
      if (lane == 0) bars->k_issued = j + 1;
      if (!load(&tm_v, smem + C::kVOff + vs * C::kTileBytes, &bars->v_full[vs], &bars->v_empty[vs], j, C::kVStages, pg))
        break;
      if (lane == 0) bars->v_issued = j + 1;
      pg = next;
    }
  } else if (warp == kMmaWarp) {
    // ---------------------------------------------------------------- MMA
    if (lane == 0) {
      const uint32_t id_s = idesc_bf16(kTileM, kTileN, 0), id_pv = idesc_bf16(kTileM, D, 1);
      auto issue_s = [&](int i) {
        const int t = i & 1, j = tile_of(i), st = j % C::kKStages;
        if (!wait_or_abort(&bars->k_full[st], (j / C::kKStages) & 1, abort)) return false;
        tc_fence_after();
        const uint32_t k_base = smem_addr(smem + C::kKOff + st * C::kTileBytes);
        const uint32_t q_base = smem_addr(smem + (kPair ? t : 0) * C::kTileBytes);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * C::kHalfBytes + (kk & 3) * 32;
          mma_ss(tmem + t * 128, desc_sw128(q_base + off, 16, 1024), desc_sw128(k_base + off, 16, 1024), id_s, kk > 0);
        }
        mma_commit(&bars->s_full[t]);
        if (!kPair || t == 1) mma_commit(&bars->k_empty[st]);
        return true;
      };
      auto issue_pv = [&](int i) {
        const int t = i & 1, j = tile_of(i), st = j % C::kVStages;
        if (!wait_or_abort(&bars->v_full[st], (j / C::kVStages) & 1, abort)) return false;
        tc_fence_after();
        const uint32_t v_base = smem_addr(smem + C::kVOff + st * C::kTileBytes);
        const uint32_t p_tmem = tmem + t * 128, o_tmem = tmem + 256 + t * 128;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          mma_ts(o_tmem, p_tmem + kk * 8, desc_sw128(v_base + kk * 16 * 128, C::kHalfBytes, 1024), id_pv,
                 (i > 1 || kk > 0) ? 1u : 0u);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          mma_ts(o_tmem, p_tmem + 64 + kk * 8, desc_sw128(v_base + kk * 16 * 128, C::kHalfBytes, 1024), id_pv, 1u);
        mma_commit(&bars->o_full[t]);
        if (!kPair || t == 1) mma_commit(&bars->v_empty[st]);
        return true;
      };
      bool ok = wait_or_abort(&bars->q_full, 0, abort) && issue_s(0) && (steps < 2 || issue_s(1));
      for (int i = 0; ok && i < steps; ++i) {
        if (!wait_or_abort(&bars->p_full[i & 1], (i >> 1) & 1, abort)) break;
        tc_fence_after();
        ok = issue_pv(i) && (i + 2 >= steps || issue_s(i + 2));  // in order: P(i) is read before S(i + 2) replaces it
      }
      mma_commit(&bars->drain);
      (void)mbar_wait_bounded(&bars->drain, 0);
    }
  } else {
    // ------------------------------------------------------------ softmax
    constexpr int CW = 64, OW = D / 2;   // a thread's columns of S and of O
    const int quarter = warp & 3, ch = warp >> 2, r = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const int pair_bar = 1 + quarter;
    float* const red = reinterpret_cast<float*>(smem + C::kRedOff);  // [parity][half][row]
    auto valid_rows = [&](int t) { return min(a.seqs, max(0, a.batch - (b0 + t * a.seqs))) * a.group; };
    float m_ref0 = -INFINITY, m_ref1 = -INFINITY, l_part0 = 0.f, l_part1 = 0.f;
    bool ok = true;
#pragma unroll 1
    for (int i = 0; ok && i < steps; ++i) {
      const int t = i & 1;
      const float m_ref_t = t ? m_ref1 : m_ref0;
      const uint32_t s_tm = tmem + lane_off + t * 128;
      const uint32_t o_tm = tmem + lane_off + 256 + t * 128 + ch * OW;
      if (!__all_sync(0xffffffffu, wait_or_abort(&bars->s_full[t], (i >> 1) & 1, abort))) {
        ok = false;
        break;
      }
      if (quarter * 32 >= valid_rows(kPair ? t : 0)) {  // no row of these warps counts
        mbar_arrive(&bars->p_full[t]);
        continue;
      }
      tc_fence_after();
      float sv[CW];
#pragma unroll
      for (int c = 0; c < CW; c += 32) tmem_ld32(s_tm + ch * CW + c, sv + c);
      tmem_wait_ld();
      const int left = a.tokens - (j0 + tile_of(i)) * kTileN;  // of the prefix, from this tile on
      if (left < kTileN) {
#pragma unroll
        for (int c = 0; c < CW; ++c)
          if (ch * CW + c >= left) sv[c] = -INFINITY;
      }
      float mx4[4] = {sv[0], sv[1], sv[2], sv[3]};
#pragma unroll
      for (int c = 4; c < CW; c += 2)
        asm("max.f32 %0, %0, %1, %2;" : "+f"(mx4[(c >> 1) & 3]) : "f"(sv[c]), "f"(sv[c + 1]));
      float* const rbuf = red + (i & 1) * 2 * kTileM;
      rbuf[ch * kTileM + r] = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
      asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
      const float m_tile = fmaxf(rbuf[r], rbuf[kTileM + r]) * a.scale_log2;  // scale > 0 keeps the order
      const bool move = m_tile > m_ref_t + kRescaleThreshold;
      const float m_new = move ? m_tile : m_ref_t;
      const float corr = move ? ex2_ftz(m_ref_t - m_new) : 1.f;
      float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      const float2 sc2 = make_float2(a.scale_log2, a.scale_log2), nm2 = make_float2(-m_new, -m_new);
#pragma unroll
      for (int c = 0; c < CW; c += 32) {
        uint32_t pw[16], lw[16];
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          const float2 x = __ffma2_rn(make_float2(sv[c + k], sv[c + k + 1]), sc2, nm2);
          float2 pp;
          pp.x = ex2_ftz(x.x);
          pp.y = ex2_ftz(x.y);
          sum2[(k >> 1) & 1] = __fadd2_rn(sum2[(k >> 1) & 1], pp);
          const __nv_bfloat162 pb = __floats2bfloat162_rn(pp.x, pp.y);
          const uint32_t hw = *reinterpret_cast<const uint32_t*>(&pb);
          pw[k / 2] = hw;
          // what bf16 leaves of a weight is exact in fp32; its own rounding carries the next 8 bits
          const float2 hi = make_float2(__uint_as_float(hw << 16), __uint_as_float(hw & 0xFFFF0000u));
          const float2 d = __fadd2_rn(pp, make_float2(-hi.x, -hi.y));
          const __nv_bfloat162 lb = __floats2bfloat162_rn(d.x, d.y);
          lw[k / 2] = *reinterpret_cast<const uint32_t*>(&lb);
        }
        // P as bf16 pairs along the tokens: the first numbers in columns [0, 64), the second in [64, 128)
        tmem_st16(s_tm + ch * (CW / 2) + c / 2, pw);
        tmem_st16(s_tm + 64 + ch * (CW / 2) + c / 2, lw);
      }
      const float l_new = (t ? l_part1 : l_part0) * corr + ((sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y));
      if (t) l_part1 = l_new; else l_part0 = l_new;
      tmem_wait_st();
      if (i > 1 && __any_sync(0xffffffffu, corr != 1.f)) {
        // O must hold the stream's last PV before it is rescaled
        if (!__all_sync(0xffffffffu, wait_or_abort(&bars->o_full[t], ((i >> 1) - 1) & 1, abort))) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < OW; c += 32) {
          float ov[32];
          tmem_ld32(o_tm + c, ov);
          tmem_wait_ld();
          uint32_t ow[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) ow[k] = __float_as_uint(ov[k] * corr);
          tmem_st32(o_tm + c, ow);
        }
        tmem_wait_st();
      }
      if (t) m_ref1 = m_new; else m_ref0 = m_new;
      tc_fence_before();
      mbar_arrive(&bars->p_full[t]);
    }
    // ---- the rows' partial results ----
    const long long rows = (long long)a.batch * a.n_q_heads;
#pragma unroll 1
    for (int t = 0; ok && t < 2; ++t) {
      const int n_t = (steps + 1 - t) / 2;  // steps of the stream
      if (n_t && !__all_sync(0xffffffffu, wait_or_abort(&bars->o_full[t], (n_t - 1) & 1, abort))) break;
      if (!kPair && t == 0) continue;  // both streams' at once
      tc_fence_after();
      if (quarter * 32 >= valid_rows(kPair ? t : 0)) continue;
      float m = t ? m_ref1 : m_ref0, l = t ? l_part1 : l_part0, f0 = 1.f, f1 = 1.f;
      if constexpr (!kPair) {
        m = fmaxf(m_ref0, m_ref1);
        f0 = m_ref0 == m ? 1.f : ex2_ftz(m_ref0 - m);
        f1 = m_ref1 == m ? 1.f : ex2_ftz(m_ref1 - m);
        l = l_part0 * f0 + l_part1 * f1;
      }
      float* const lbuf = red + ((steps + t) & 1) * 2 * kTileM;
      lbuf[ch * kTileM + r] = l;
      asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
      l = lbuf[r] + lbuf[kTileM + r];
      const bool there = r < valid_rows(kPair ? t : 0);
      const int b = b0 + (kPair ? t : 0) * a.seqs + r / a.group;
      const long long row = split * rows + (there ? (long long)b * a.n_q_heads + kvh * a.group + r % a.group : 0);
      if (there && ch == 0) a.ml[row] = make_float2(m, l);
      float* const dst = a.acc + row * D + ch * OW;
#pragma unroll
      for (int c = 0; c < OW; c += 32) {
        float ov[32];
        tmem_ld32(tmem + lane_off + 256 + (kPair ? t : 0) * 128 + ch * OW + c, ov);
        tmem_wait_ld();
        if constexpr (!kPair) {
          if (steps > 1) {
            float ow[32];
            tmem_ld32(tmem + lane_off + 256 + 128 + ch * OW + c, ow);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) ov[k] = ov[k] * f0 + ow[k] * f1;
          }
        }
        if (there) {
#pragma unroll
          for (int k = 0; k < 32; k += 4)
            *reinterpret_cast<float4*>(dst + c + k) = make_float4(ov[k], ov[k + 1], ov[k + 2], ov[k + 3]);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort) {
    if (threadIdx.x == 0) atomicOr(a.status, kDevWaitTimeout);
    if (threadIdx.x == kTmaWarp * 32) {
      (void)mbar_wait_bounded(&bars->q_full, 0);
      for (int j = max(0, bars->k_issued - C::kKStages); j < bars->k_issued; ++j)
        (void)mbar_wait_bounded(&bars->k_full[j % C::kKStages], (j / C::kKStages) & 1);
      for (int j = max(0, bars->v_issued - C::kVStages); j < bars->v_issued; ++j)
        (void)mbar_wait_bounded(&bars->v_full[j % C::kVStages], (j / C::kVStages) & 1);
    }
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

template <int D, bool kPair>
cudaError_t launch(const PrefixArgs& a, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                   cudaStream_t stream) {
  using C = Cfg<D, kPair>;
  const void* fn = reinterpret_cast<const void*>(&prefix_kernel<D, kPair>);
  {
    static std::mutex mu;
    static uint64_t done = 0;  // the shared-memory opt-in is per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    std::lock_guard<std::mutex> lock(mu);
    if (dev > 63 || !(done >> dev & 1)) {
      e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
      if (e != cudaSuccess) return e;
      if (dev <= 63) done |= 1ull << dev;
    }
  }
  void* p[] = {const_cast<CUtensorMap*>(&mq), const_cast<CUtensorMap*>(&mk), const_cast<CUtensorMap*>(&mv),
               const_cast<PrefixArgs*>(&a)};
  return launch_with_pdl(fn, dim3((unsigned)(a.n_kv_heads * a.units * a.splits)), dim3(kThreads), p, C::kSmem, stream);
}

}  // namespace

namespace paged {

PrefixPlan prefix_plan(int batch, int n_kv_heads, int group, int tokens) {
  PrefixPlan p{};
  p.seqs = kTileM / group;
  const int row_tiles = (batch + p.seqs - 1) / p.seqs;
  p.pair = row_tiles > 1;
  p.units = p.pair ? (row_tiles + 1) / 2 : 1;
  const int tiles = (tokens + kTileN - 1) / kTileN;
  const long long units = (long long)p.units * n_kv_heads, sms = std::max(1, device_sm_count());
  // the CTAs of one wave, as far as there are tiles
  p.splits = (int)std::max(1ll, std::min<long long>(tiles, sms / units));
  return p;
}

cudaError_t prefix_launch(const PrefixPlan& plan, const uint16_t* q, const uint16_t* k, const uint16_t* v,
                          const PoolIndex& index, int tokens, int batch, int n_q_heads, int head_dim, float scale_log2,
                          float2* ml, float* acc, int* status, cudaStream_t stream) {
  const int group = n_q_heads / index.n_kv_heads, page = 1 << index.page_log2;
  CUtensorMap mq, mk, mv;
  // Q: (d, head of the group, kv head, sequence); K/V: (d, row in page, kv head, page)
  const cuuint64_t D = (cuuint64_t)head_dim, hkv = (cuuint64_t)index.n_kv_heads;
  const cuuint64_t qd[4] = {D, (cuuint64_t)group, hkv, (cuuint64_t)batch};
  const cuuint64_t qs[3] = {D * 2, D * 2 * group, D * 2 * n_q_heads};
  const cuuint32_t qbox[4] = {64, (cuuint32_t)group, 1, (cuuint32_t)plan.seqs};
  const cuuint64_t kd[4] = {D, (cuuint64_t)page, hkv, (cuuint64_t)index.num_pages};
  const cuuint64_t ks[3] = {D * 2, D * 2 * page, D * 2 * page * hkv};
  const cuuint32_t kbox[4] = {64, (cuuint32_t)std::min(page, kTileN), 1, 1};
  if (!make_tensor_map_bf16(&mq, q, 4, qd, qs, qbox) || !make_tensor_map_bf16(&mk, k, 4, kd, ks, kbox) ||
      !make_tensor_map_bf16(&mv, v, 4, kd, ks, kbox))
    return cudaErrorInvalidValue;
  PrefixArgs a{};
  a.table = index.block_table;
  a.tokens = tokens;
  a.batch = batch;
  a.n_q_heads = n_q_heads;
  a.n_kv_heads = index.n_kv_heads;
  a.group = group;
  a.seqs = plan.seqs;
  a.units = plan.units;
  a.splits = plan.splits;
  a.page_log2 = index.page_log2;
  a.num_pages = index.num_pages;
  a.scale_log2 = scale_log2;
  a.ml = ml;
  a.acc = acc;
  a.status = status;
  if (head_dim == 128) return plan.pair ? launch<128, true>(a, mq, mk, mv, stream) : launch<128, false>(a, mq, mk, mv, stream);
  return plan.pair ? launch<64, true>(a, mq, mk, mv, stream) : launch<64, false>(a, mq, mk, mv, stream);
}

}  // namespace paged

}  // namespace lara
