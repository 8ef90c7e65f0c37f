// The first launch of a decode behind a prefix that the batch has in common
// (lara_gqa_decode_shared): some CTAs take the prefix, once for the batch, on the
// 5th-generation tensor cores, the others the tokens that sequences have for
// themselves (paged_own.cuh).  The first is bound by the tensor cores or the
// softmax, the second by HBM, so they run side by side; how many CTAs do which
// follows from the lengths, on the device.
//
// The prefix: for each kv head the G query heads of all sequences are the rows
// of one attention.  Tiles of floor(128 / G) sequences (rows = TMEM lanes) meet
// tiles of 128 tokens as two streams in ping-pong, so that the tensor core works
// on one while the other's softmax runs.  kPair: the streams are two row tiles and
// share every K/V tile; otherwise (one row tile) they are the even and the odd
// token tiles of the same rows, joined at the end.
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
// All token tiles of all units, (kv head, row tiles), laid end to end, are shared
// out equally; a CTA leaves (reference, sum, unnormalised output) of its rows for
// each unit that it has a part of.
//
// Measured (32 heads on 8, head_dim 128), one state replayed in a graph and, in
// brackets, inputs that change from pass to pass: 64 sequences behind 8192 tokens, with
// up to 512 of their own, 38 us (41), 132 with shared_pages = 0; 256 (64 heads) behind
// 16384 231 to 260 us (263 to 277; 1127 to 1235 with 0), 545 to 615 TFLOP/s at 4 head_dim
// operations a head and token, half as many again on the tensor cores (P in two
// numbers).  That is bound by the softmax: 2287 cycles a step, of which 1430 are
// exponentials and the two bf16 numbers, while the products take 1536.  4 sequences
// behind 1024 12.9 us (13.0; 12.2 with 0), and 37 behind 2000 (head_dim 64) 17.2 (17.1;
// 15.9 with 0): latency, and sharing gains nothing yet.
// Every wait is bounded; on a timeout the CTA
// flags the status word, drains its own work and returns.
#include <cuda.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "paged_own.cuh"
#include "tcgen05.cuh"

namespace lara {

using namespace tc;
using namespace paged;

namespace {

constexpr int kTileM = 128, kTileN = 128;
constexpr int kSoftmaxWarps = 8, kMmaWarp = 8, kTmaWarp = 9;
constexpr int kOwnWarps = 12, kThreads = kOwnWarps * 32;  // two warps of the prefix's CTAs idle
constexpr float kRescaleThreshold = 8.0f;
constexpr uint32_t kTmemCols = 512;  // S_0 | S_1 | O_0 | O_1, 128 columns each

template <int D, bool kPair>
struct Prefix {
  static constexpr int kHalves = D / 64;            // 128-byte-swizzled parts of a row
  static constexpr int kHalfBytes = 128 * 128;      // [128 rows][64 bf16]
  static constexpr int kTileBytes = kHalves * kHalfBytes;
  static constexpr int kQTiles = kPair ? 2 : 1;
  static constexpr int kKStages = D == 128 ? (kPair ? 2 : 3) : 4;
  static constexpr int kVStages = D == 128 ? 2 : 4;
  static constexpr int kKOff = kQTiles * kTileBytes;
  static constexpr int kVOff = kKOff + kKStages * kTileBytes;
  // exchange of the pairs: per stream, row maxima, then sums, [2][2][2][128] floats
  static constexpr int kRedOff = kVOff + kVStages * kTileBytes;
  static constexpr int kSmem = kRedOff + 2 * 2 * 2 * kTileM * 4 + 1024;
  static constexpr int kRows = kQTiles * kTileM;
};

struct Bars {
  uint64_t q_full, q_empty;
  uint64_t k_full[4], k_empty[4];
  uint64_t v_full[4], v_empty[4];
  uint64_t s_full[2], p_full[2], o_full[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
  int k_issued, v_issued, q_issued;
};
// What one lane of a whole warp issues.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one;
}
__device__ __forceinline__ void mma_ss_one(uint32_t one, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                           uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(one)
      : "memory");
}
__device__ __forceinline__ void mma_ts_one(uint32_t one, uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                           uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(one)
      : "memory");
}
__device__ __forceinline__ void mma_commit_one(uint32_t one, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)),
      "r"(one)
      : "memory");
}
__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return __all_sync(0xffffffffu, wait_or_abort(bar, parity, abort));
}

struct PrefixArgs {
  int units;  // of all kv heads
  int tiles;  // of 128 tokens
  int brought;  // of a CTA's: all, but in the self-test of waits that run out
};

// The part of a unit that a CTA takes: token tiles [j0, j0 + n).
struct Segment {
  int unit, j0, n;
};

template <int D, bool kPair>
__device__ __forceinline__ void prefix_pass(const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                                            const DecodeArgs& a, const PrefixArgs& p, int seq, int me, int ctas,
                                            uint8_t* smem_raw, Bars* bars, uint32_t tmem) {
  using C = Prefix<D, kPair>;
  uint8_t* const smem = smem_raw + (-smem_addr(smem_raw) & 1023);
  volatile int* const abort = &bars->abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long all = (long long)p.units * p.tiles;
  const int workers = (int)min((long long)ctas, all);
  if (me >= workers) return;
  const Shares sh{quotient(all, workers), all - quotient(all, workers) * workers};
  const long long begin = sh.start(me), end = sh.start(me + 1);
  // segment after segment: at is advanced
  auto next_segment = [&](long long& at) {
    const int unit = (int)quotient(at, p.tiles), j0 = (int)(at - (long long)unit * p.tiles);
    const int n = (int)min((long long)(p.tiles - j0), end - at);
    at += n;
    return Segment{unit, j0, n};
  };
  auto head_of = [&](const Segment& g) { return g.unit / a.prefix.units; };
  auto seq_of = [&](const Segment& g) { return g.unit % a.prefix.units * (C::kQTiles * a.prefix.seqs); };
  // step i of a segment: stream i & 1, tile i / 2 (pair) or i
  auto steps_of = [](const Segment& g) { return kPair ? 2 * g.n : g.n; };

  if (warp == kTmaWarp) {
    // ---------------------------------------------------------------- TMA
    const int log2 = a.index.page_log2, piece = min(kTileN, 1 << log2), pieces = kTileN / piece;
    const int32_t* const table = a.index.block_table + (long long)seq * a.index.pages_per_seq;
    // lane i copies piece i of every tile; its page is looked up a tile ahead.  Behind the
    // prefix's end a page that is not there: the copy writes zeros
    auto page_of = [&](int j) {
      const int tok = j * kTileN + lane * piece;
      if (lane >= pieces || tok >= a.shared_tokens) return a.index.num_pages;
      int pg = __ldg(table + (tok >> log2));
      if ((unsigned)pg >= (unsigned)a.index.num_pages) {
        atomicOr(a.status, kDevBadPage);
        pg = 0;
      }
      return pg;
    };
    auto load = [&](const CUtensorMap* map, uint8_t* to, uint64_t* full, uint64_t* empty, int count, int stages, int j,
                    int kvh, int pg) {
      int good = 1;
      if (lane == 0) {
        if (count >= stages && !wait_or_abort(empty, ((count / stages) - 1) & 1, abort)) good = 0;
        if (good) mbar_arrive_expect_tx(full, C::kTileBytes);
      }
      if (!__shfl_sync(0xffffffffu, good, 0)) return false;
      if (lane < pieces) {
        const int row = j * kTileN & ((1 << log2) - 1);  // 0 where pages are smaller than a tile
        for (int x = 0; x < C::kHalves; ++x)
          tma_load_4d(to + x * C::kHalfBytes + lane * piece * 128, map, 64 * x, row, kvh, pg, full);
      }
      return true;
    };
    int count = 0, segments = 0;  // tiles so far
    int pg = page_of((int)(begin - quotient(begin, p.tiles) * p.tiles));
    bool ok = true;
    for (long long at = begin; ok && at < end; ++segments) {
      const Segment g = next_segment(at);
      const int kvh = head_of(g), b0 = seq_of(g);
      int good = 1;
      if (lane == 0) {  // the queries, when the scores of the segment before are there
        if (segments && !wait_or_abort(&bars->q_empty, (segments - 1) & 1, abort)) good = 0;
        if (good) {
          mbar_arrive_expect_tx(&bars->q_full, (uint32_t)(C::kQTiles * C::kHalves * a.prefix.seqs * a.group * 128));
          for (int t = 0; t < C::kQTiles; ++t)
            for (int x = 0; x < C::kHalves; ++x)
              tma_load_4d(smem + t * C::kTileBytes + x * C::kHalfBytes, &tm_q, 64 * x, 0, kvh, b0 + t * a.prefix.seqs,
                          &bars->q_full);
          bars->q_issued = segments + 1;
        }
      }
      ok = __shfl_sync(0xffffffffu, good, 0);
      for (int j = 0; ok && j < g.n; ++j, ++count) {
        if (count >= p.brought) {
          ok = false;
          break;
        }
        // the tile after this one: of this segment, or the next unit's first
        const int next = page_of(j + 1 < g.n ? g.j0 + j + 1 : 0);
        const int ks = count % C::kKStages, vs = count % C::kVStages;
        ok = load(&tm_k, smem + C::kKOff + ks * C::kTileBytes, &bars->k_full[ks], &bars->k_empty[ks], count,
                  C::kKStages, g.j0 + j, kvh, pg);
        if (ok && lane == 0) bars->k_issued = count + 1;
        ok = ok && load(&tm_v, smem + C::kVOff + vs * C::kTileBytes, &bars->v_full[vs], &bars->v_empty[vs], count,
                        C::kVStages, g.j0 + j, kvh, pg);
        if (ok && lane == 0) bars->v_issued = count + 1;
        pg = next;
      }
    }
  } else if (warp == kMmaWarp) {
    // ---------------------------------------------------------------- MMA
    // The whole warp goes through the steps and one lane issues, so that what a product needs is made
    // in uniform registers: made by one thread alone, it took longer than the product takes.
    {
      const uint32_t one = elect_one();
      const uint32_t id_s = idesc_bf16(kTileM, kTileN, 0), id_pv = idesc_bf16(kTileM, D, 1);
      // descriptors differ in their address field alone, whose unit is 16 bytes
      const uint64_t q_desc0 = desc_sw128(smem_addr(smem), 16, 1024);
      const uint64_t k_desc0 = desc_sw128(smem_addr(smem + C::kKOff), 16, 1024);
      const uint64_t v_desc0 = desc_sw128(smem_addr(smem + C::kVOff), C::kHalfBytes, 1024);
      int tiles = 0;             // before this segment
      int done0 = 0, done1 = 0;  // steps of each stream before it
      auto tile_of = [&](int i) { return tiles + (kPair ? i >> 1 : i); };
      auto issue_s = [&](int i) {
        const int t = i & 1, j = tile_of(i), st = j % C::kKStages;
        if (!wait_all(&bars->k_full[st], (j / C::kKStages) & 1, abort)) return false;
        tc_fence_after();
        const uint64_t k_desc = k_desc0 + st * (C::kTileBytes >> 4);
        const uint64_t q_desc = q_desc0 + (kPair ? t : 0) * (C::kTileBytes >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * C::kHalfBytes + (kk & 3) * 32;
          mma_ss_one(one, tmem + t * 128, q_desc + (off >> 4), k_desc + (off >> 4), id_s, kk > 0);
        }
        mma_commit_one(one, &bars->s_full[t]);
        if (!kPair || t == 1) mma_commit_one(one, &bars->k_empty[st]);
        return true;
      };
      auto issue_pv = [&](int i) {
        const int t = i & 1, j = tile_of(i), st = j % C::kVStages;
        if (!wait_all(&bars->v_full[st], (j / C::kVStages) & 1, abort)) return false;
        tc_fence_after();
        const uint64_t v_desc = v_desc0 + st * (C::kTileBytes >> 4);
        const uint32_t p_tmem = tmem + t * 128, o_tmem = tmem + 256 + t * 128;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          mma_ts_one(one, o_tmem, p_tmem + kk * 8, v_desc + (kk * 16 * 128 >> 4), id_pv,
                 (i > 1 || kk > 0) ? 1u : 0u);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          mma_ts_one(one, o_tmem, p_tmem + 64 + kk * 8, v_desc + (kk * 16 * 128 >> 4), id_pv, 1u);
        mma_commit_one(one, &bars->o_full[t]);
        if (!kPair || t == 1) mma_commit_one(one, &bars->v_empty[st]);
        return true;
      };
      bool ok = true;
      int segments = 0;
      for (long long at = begin; ok && at < end; ++segments) {
        const Segment g = next_segment(at);
        const int steps = steps_of(g);
        ok = wait_all(&bars->q_full, segments & 1, abort) && issue_s(0) && (steps < 2 || issue_s(1));
        for (int i = 0; ok && i < steps; ++i) {
          const int t = i & 1;
          if (!wait_all(&bars->p_full[t], ((t ? done1 : done0) + (i >> 1)) & 1, abort)) {
            ok = false;
            break;
          }
          tc_fence_after();
          ok = issue_pv(i) && (i + 2 >= steps || issue_s(i + 2));  // in order: P(i) is read before S(i + 2) replaces it
        }
        mma_commit_one(one, &bars->q_empty);  // every score of the segment is there
        tiles += g.n;
        done0 += (steps + 1) / 2;
        done1 += steps / 2;
      }
      mma_commit_one(one, &bars->drain);
      (void)mbar_wait_bounded(&bars->drain, 0);
    }
  } else if (warp < kSoftmaxWarps) {
    // ------------------------------------------------------------ softmax
    constexpr int CW = 64, OW = D / 2;   // a thread's columns of S and of O
    const int quarter = warp & 3, ch = warp >> 2, r = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const int pair_bar = 1 + quarter;
    float* const red = reinterpret_cast<float*>(smem + C::kRedOff);  // [maxima, sums][stream][half][row]
    int done0 = 0, done1 = 0;  // steps of each stream before this segment
    // A wait that ran out leaves the order as it is: each warp goes on through all steps, without further
    // waits and with results that are not written.  So no warp stands alone at its pair's barrier, which has
    // no limit, and every unit's parts are entered, by which the join finds its way.
    bool ok = true;
    auto wait = [&](uint64_t* bar, int phase) {
      if (!wait_all(bar, phase & 1, abort)) ok = false;
    };
    for (long long at = begin; at < end;) {
      const Segment g = next_segment(at);
      const int steps = steps_of(g), kvh = head_of(g), b0 = seq_of(g);
      auto valid_rows = [&](int t) { return min(a.prefix.seqs, max(0, a.batch - (b0 + t * a.prefix.seqs))) * a.group; };
      float m_ref0 = -INFINITY, m_ref1 = -INFINITY, l_part0 = 0.f, l_part1 = 0.f;
#pragma unroll 1
      for (int i = 0; i < steps; ++i) {
        const int t = i & 1;
        const float m_ref_t = t ? m_ref1 : m_ref0;
        const uint32_t s_tm = tmem + lane_off + t * 128;
        const uint32_t o_tm = tmem + lane_off + 256 + t * 128 + ch * OW;
        wait(&bars->s_full[t], (t ? done1 : done0) + (i >> 1));
        if (quarter * 32 >= valid_rows(kPair ? t : 0)) {  // no row of these warps counts
          mbar_arrive(&bars->p_full[t]);
          continue;
        }
        tc_fence_after();
        float sv[CW];
#pragma unroll
        for (int c = 0; c < CW; c += 32) tmem_ld32(s_tm + ch * CW + c, sv + c);
        tmem_wait_ld();
        const int left = a.shared_tokens - (g.j0 + (kPair ? i >> 1 : i)) * kTileN;  // of the prefix, from this tile on
        if (left < kTileN) {
#pragma unroll
          for (int c = 0; c < CW; ++c)
            if (ch * CW + c >= left) sv[c] = -INFINITY;
        }
        float mx4[4] = {sv[0], sv[1], sv[2], sv[3]};
#pragma unroll
        for (int c = 4; c < CW; c += 2)
          asm("max.f32 %0, %0, %1, %2;" : "+f"(mx4[(c >> 1) & 3]) : "f"(sv[c]), "f"(sv[c + 1]));
        float* const rbuf = red + t * 2 * kTileM;  // its last readers have let this step's scores come
        const float top = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * a.scale_log2;  // scale > 0 keeps the order
        rbuf[ch * kTileM + r] = top;
        const float unit = score_unit(sv, top, a.scale_log2);
        asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
        const float m_tile = fmaxf(rbuf[r], rbuf[kTileM + r]);
        const bool move = m_tile > m_ref_t + kRescaleThreshold;
        const float m_new = move ? m_tile : m_ref_t;
        const float corr = move ? ex2_ftz(m_ref_t - m_new) : 1.f;
        float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        const float m_use = m_new == -INFINITY ? 0.f : m_new;  // while all scores were -inf they weigh nothing
        const float2 sc2 = make_float2(unit, unit), nm2 = make_float2(-m_use, -m_use);
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
          wait(&bars->o_full[t], (t ? done1 : done0) + (i >> 1) - 1);
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
      const int slot = g.unit + me;
      if (threadIdx.x == 0 && g.j0 == 0)  // the unit starts here
        a.prefix_units[g.unit] = UnitParts{slot, sh.cta((long long)(g.unit + 1) * p.tiles - 1) - me + 1};
#pragma unroll 1
      for (int t = 0; t < 2; ++t) {
        const int n_t = (steps + 1 - t) / 2;  // steps of the stream
        if (n_t) wait(&bars->o_full[t], (t ? done1 : done0) + n_t - 1);
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
        float* const lbuf = red + (2 + t) * 2 * kTileM;
        lbuf[ch * kTileM + r] = l;
        asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
        l = lbuf[r] + lbuf[kTileM + r];
        const bool there = ok && r < valid_rows(kPair ? t : 0);
        const long long row = (long long)slot * C::kRows + (kPair ? t : 0) * kTileM + r;
        if (there && ch == 0) a.prefix_ml[row] = make_float2(m, l);
        float* const dst = a.prefix_acc + row * D + ch * OW;
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
      tc_fence_before();  // before the next segment's first products replace O
      done0 += (steps + 1) / 2;
      done1 += steps / 2;
    }
  }

  __syncthreads();
  if (*abort) {
    if (threadIdx.x == 0) atomicOr(a.status, kDevWaitTimeout);
    if (threadIdx.x == kTmaWarp * 32) {
      if (bars->q_issued) (void)mbar_wait_bounded(&bars->q_full, (bars->q_issued - 1) & 1);
      for (int j = max(0, bars->k_issued - C::kKStages); j < bars->k_issued; ++j)
        (void)mbar_wait_bounded(&bars->k_full[j % C::kKStages], (j / C::kKStages) & 1);
      for (int j = max(0, bars->v_issued - C::kVStages); j < bars->v_issued; ++j)
        (void)mbar_wait_bounded(&bars->v_full[j % C::kVStages], (j / C::kVStages) & 1);
    }
  }
}

// What the passes cost, in nanoseconds of one SM, as measured (head_dim 64: half as much): a tile of
// 128 tokens for a pair of row tiles or for one, what a CTA spends beside its tiles; 16 own tokens, and
// a unit of them beside, where CTAs or warps take them.  With 85 or 115 for an own tile the times
// differ by 1 %; with 3000 for a unit 37 sequences of 20 tiles took 19.7 us in place of 17.4.
constexpr int kPairTileNs = 2800, kTileNs = 1600, kPassNs = 8000, kOwnTileNs = 100, kUnitNs = 6000,
              kSoloUnitNs = 500;

template <int D, int NG, bool kPair>
using OwnOf = OwnTokens<D, NG, kOwnWarps, D == 128 ? 2 : 4, false>;

template <int D, int NG, bool kPair>
__global__ void __launch_bounds__(kThreads, 1)
    shared_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ DecodeArgs a,
                  const __grid_constant__ PrefixArgs p) {
  using Own = OwnOf<D, NG, kPair>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ typename Own::Shared shared;
  __shared__ Bars bars;
  __shared__ int covering;  // the first sequence that is as long as the prefix
  // what the prefix needs is set up while the kernel before this one ends
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    mbar_init(&bars.q_full, 1);
    mbar_init(&bars.q_empty, 1);
    for (int s = 0; s < 4; ++s) {
      mbar_init(&bars.k_full[s], 1);
      mbar_init(&bars.k_empty[s], 1);
      mbar_init(&bars.v_full[s], 1);
      mbar_init(&bars.v_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars.s_full[t], 1);
      mbar_init(&bars.p_full[t], kSoftmaxWarps * 32);
      mbar_init(&bars.o_full[t], 1);
    }
    mbar_init(&bars.drain, 1);
    bars.abort = 0;
    bars.k_issued = bars.v_issued = bars.q_issued = 0;
    covering = 0x7fffffff;
    mbar_fence_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&bars.tmem_base)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  grid_dependency_wait();
  Own own(a, shared);
  own.totals();
  if (own.covering != 0x7fffffff) atomicMin(&covering, own.covering);
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem_base;
  // CTAs for the own tokens: as many as make both passes end together
  const long long own_ns =
      own.total * (kOwnTileNs * D / 128) + own.units * (own.solo_units(gridDim.x / 4) ? kSoloUnitNs : kUnitNs);
  const long long prefix_tiles = covering < a.batch ? (long long)p.units * p.tiles : 0;
  const long long prefix_ns = prefix_tiles * ((kPair ? kPairTileNs : kTileNs) * D / 128) +
                              kPassNs * min(prefix_tiles, (long long)gridDim.x);
  int ctas = (int)gridDim.x;
  if (prefix_ns > 0) {
    // at least as many as keep a share below 2^30 tiles
    const int least = own_ns == 0 ? 0 : 1 + (int)((own.total + own.units * kUnitCost) >> 30);
    ctas = max(least, min(ctas - 1, (int)((float)own_ns / (float)(own_ns + prefix_ns) * ctas + 0.5f)));
  }
  if ((int)blockIdx.x < ctas) {
    own.run(blockIdx.x, ctas, smem_raw + (-smem_addr(smem_raw) & 127));
  } else {
    prefix_pass<D, kPair>(tm_q, tm_k, tm_v, a, p, covering, blockIdx.x - ctas, gridDim.x - ctas, smem_raw,
                          &bars, tmem);
  }
  allow_dependent_launch();
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

template <int D, int NG, bool kPair>
cudaError_t launch(const DecodeArgs& a, const PrefixArgs& pa, const CUtensorMap& mq, const CUtensorMap& mk,
                   const CUtensorMap& mv, cudaStream_t stream) {
  using Own = OwnOf<D, NG, kPair>;
  constexpr int kSmem = std::max(Prefix<D, kPair>::kSmem, Own::C::kSmemBytes);
  const void* fn = reinterpret_cast<const void*>(&shared_kernel<D, NG, kPair>);
  {
    static std::mutex mu;
    static uint64_t done = 0;  // the shared-memory opt-in is per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    std::lock_guard<std::mutex> lock(mu);
    if (dev > 63 || !(done >> dev & 1)) {
      e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
      if (e != cudaSuccess) return e;
      if (dev <= 63) done |= 1ull << dev;
    }
  }
  void* p[] = {const_cast<CUtensorMap*>(&mq), const_cast<CUtensorMap*>(&mk), const_cast<CUtensorMap*>(&mv),
               const_cast<DecodeArgs*>(&a), const_cast<PrefixArgs*>(&pa)};
  return launch_with_pdl(fn, dim3((unsigned)std::max(2, device_sm_count())), dim3(kThreads), p, kSmem, stream);
}

}  // namespace

namespace paged {

PrefixPlan prefix_plan(int batch, int group) {
  PrefixPlan p;
  p.seqs = kTileM / group;
  const int row_tiles = (batch + p.seqs - 1) / p.seqs;
  p.units = (row_tiles + 1) / 2;
  p.rows = row_tiles > 1 ? 2 * kTileM : kTileM;
  return p;
}

cudaError_t shared_launch(const DecodeArgs& a, int head_dim, cudaStream_t stream) {
  const int page = 1 << a.index.page_log2;
  CUtensorMap mq, mk, mv;
  // Q: (d, head of the group, kv head, sequence); K/V: (d, row in page, kv head, page)
  const cuuint64_t D = (cuuint64_t)head_dim, hkv = (cuuint64_t)a.index.n_kv_heads, group = (cuuint64_t)a.group;
  const cuuint64_t qd[4] = {D, group, hkv, (cuuint64_t)a.batch};
  const cuuint64_t qs[3] = {D * 2, D * 2 * group, D * 2 * a.n_q_heads};
  const cuuint32_t qbox[4] = {64, (cuuint32_t)group, 1, (cuuint32_t)a.prefix.seqs};
  const cuuint64_t kd[4] = {D, (cuuint64_t)page, hkv, (cuuint64_t)a.index.num_pages};
  const cuuint64_t ks[3] = {D * 2, D * 2 * page, D * 2 * page * hkv};
  const cuuint32_t kbox[4] = {64, (cuuint32_t)std::min(page, kTileN), 1, 1};
  if (!make_tensor_map_bf16(&mq, a.q, 4, qd, qs, qbox) || !make_tensor_map_bf16(&mk, a.k, 4, kd, ks, kbox) ||
      !make_tensor_map_bf16(&mv, a.v, 4, kd, ks, kbox))
    return cudaErrorInvalidValue;
  PrefixArgs p;
  p.tiles = (a.shared_tokens + kTileN - 1) / kTileN;
  p.units = p.tiles ? a.prefix.units * a.index.n_kv_heads : 0;
  p.brought = selftest_tiles_brought();
  const bool pair = a.prefix.rows > kTileM;
#define LARA_CASE(d, ng)         \
  if (head_dim == d && (a.group > 8 ? 2 : 1) == ng) \
    return pair ? launch<d, ng, true>(a, p, mq, mk, mv, stream) : launch<d, ng, false>(a, p, mq, mk, mv, stream);
  LARA_CASE(128, 1) LARA_CASE(128, 2) LARA_CASE(64, 1) LARA_CASE(64, 2)
#undef LARA_CASE
  return cudaErrorInvalidValue;
}

}  // namespace paged

}  // namespace lara
