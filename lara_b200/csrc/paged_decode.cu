// Decode over the paged bf16 cache, with each slot's attention weight gathered
// (lara_gqa_decode_scored) or behind a prefix that the batch shares
// (lara_gqa_decode_shared); declared in include/lara_b200.h.
//
//   s_t = scale log2(e) q.k_t,  o = sum_t 2^(s_t - R) v_t / sum_t 2^(s_t - R)
//   w_t += sum over the group's heads of 2^(s_t - M) / L   (M, L: the whole row's R and sum)
//
// Two launches.  The first reads every cached row once and leaves partial
// results (R, l, acc) of each unit, a (sequence, kv head), or of the parts that
// several CTAs take of it; the second joins them, and, scoring, turns the
// scores that the first left into weights (G fp32 numbers per token and kv head
// written and read beside the 4 D bytes of its rows: at G = 4, D = 128 6 % of
// them, against 50 % for reading K twice).
#include <algorithm>
#include <cmath>
#include <mutex>

#include "paged.cuh"

namespace lara {

using namespace paged;

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 16;            // tokens per warp and stage: never across pages
constexpr int kGroup = 32;           // tokens whose scores lie together, head by head (a line of 128 bytes)
constexpr int kMinTiles = kWarps;    // tiles per CTA below which fewer CTAs run
constexpr int kUnitCost = 8;         // what a unit costs beside its tiles, in tiles
constexpr int kMostCtasPerSm = 4;
constexpr int kLensCached = 1024;    // lengths kept in shared memory
// R moves only when a score passes it by this much (log2): weights stay below 2^8.
constexpr float kSlack = 8.f;

template <int D, int NG>
struct Cfg {
  static constexpr int kStages = D == 64 ? 4 : NG == 1 ? 2 : 3;
  static constexpr int kCtasPerSm = NG == 1 ? 3 : 2;
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kRowsBytes = kTile * kRowBytes;  // K (or V) of a stage
  static constexpr int kStageBytes = 2 * kRowsBytes;
  static constexpr int kWarpBytes = kStages * kStageBytes;
  static constexpr int kSmemBytes = kWarps * kWarpBytes + 128;
  static_assert(kCtasPerSm <= kMostCtasPerSm);
  static constexpr int kPitch = D + 4;  // floats per head in the join (lanes of a store hit distinct banks)
  static_assert(8 * kPitch * 4 <= kStageBytes, "a stage holds the sums of eight heads");
};

struct Args {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  PoolIndex index;
  const int32_t* lens;
  uint16_t* o;
  int batch, n_q_heads, group;
  float scale_log2;
  int* status;
  UnitParts* units;  // [batch * kv heads]; of sequences without tokens, undefined
  long long* seq_groups;  // [batch + 1] groups of one kv head of the sequences before this one
  float2* part_ml;   // [units + CTAs][group] (R, l)
  float* part_acc;   // [units + CTAs][group][D]
  // behind a shared prefix: its tokens, and what the pass over it leaves of each row
  int shared_tokens;
  int splits;
  const float2* prefix_ml;  // [splits][rows]
  const float* prefix_acc;  // [splits][rows][D]
  // scoring
  float* scores;           // [groups][group][kGroup], in the order of the units
  long long score_groups;  // that there is room for
  const float* w_in;      // [pages][kv heads][page]
  float* w_out;
};

template <int kDst>
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0+%2], [%1], 16, %3;" ::"r"(dst), "l"(src), "n"(kDst),
               "l"(policy)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma_bf16(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix(uint32_t v[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_trans(uint32_t v[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ int tiles_of(int len) { return (len + kTile - 1) / kTile; }
__device__ __forceinline__ int groups_of(int tiles) { return (tiles + kGroup / kTile - 1) / (kGroup / kTile); }

__device__ __forceinline__ long long quotient(long long a, long long b) {
  if (((a | b) >> 31) == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}

// A unit (b, kvh); `base` is the place of its first tile, counted from the
// start of the CTA's share, `group0` that of its first group of scores.  Its
// tokens are `start` .. `start` + `len` - 1.
struct Unit {
  long long group0;
  int base, tiles, len, start, b, kvh;
};

// The tokens that a sequence has for itself: a sequence that covers the shared
// prefix starts behind it.
struct Own {
  int start, len;
};
__device__ __forceinline__ Own own_tokens(const Args& a, int len) {
  const int start = a.shared_tokens > 0 && len >= a.shared_tokens ? a.shared_tokens : 0;
  return {start, len - start};
}

// Equal shares of the span: the first `rem` take one more.
struct Shares {
  long long per, rem;
  __device__ __forceinline__ long long start(long long c) const { return c * per + min(c, rem); }
  __device__ __forceinline__ int cta(long long at) const {
    return (int)(at < rem * (per + 1) ? quotient(at, per + 1) : rem + quotient(at - rem * (per + 1), per));
  }
};

// The products run as warp-wide mma with the cache as the 16-row operand and
// the group's heads as the 8 columns: S^T[token][head] = K q^T, O^T[dim][head]
// = V^T P^T.  The columns of both lie in the same lanes, so rescaling needs no
// exchange, and movmatrix turns a tile of P into the second operand.  P is the
// sum of two bf16 numbers (what both leave is 2^-17 of it), since one alone
// would show wherever values nearly cancel in an output.
template <int D, int NG, bool kScored>
__global__ void __launch_bounds__(kThreads, Cfg<D, NG>::kCtasPerSm) own_tokens_kernel(const __grid_constant__ Args a) {
  using C = Cfg<D, NG>;
  constexpr int KS = D / 16;
  extern __shared__ uint8_t smem_raw[];
  __shared__ long long s_sum[2][kWarps];
  __shared__ Unit s_first;
  __shared__ float2 s_ml[kWarps][NG * 8];
  __shared__ int s_idle[kWarps];
  __shared__ int s_lens[kLensCached];
  uint8_t* const smem = smem_raw + (-smem_addr(smem_raw) & 127);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int G = a.group, hkv = a.index.n_kv_heads;
  const long long cap = a.index.capacity();

  // The pass over a prefix has waited for what was before it when this one starts, and nothing
  // here needs what it leaves; the join does, so that this grid ends after that one.
  if (a.shared_tokens == 0) grid_dependency_wait();

  // ---- this CTA's share of all tiles, and the unit in which it starts ----
  auto load_len = [&](int b) { return (int)min((long long)max(__ldcg(a.lens + b), 0), cap); };
  auto len_of = [&](int b) { return b < kLensCached ? s_lens[b] : load_len(b); };
  auto next_unit = [&](Unit& u) {
    u.base += u.tiles + kUnitCost;
    u.group0 += groups_of(u.tiles);
    if (++u.kvh == hkv) {
      u.kvh = 0;
      do {
        ++u.b;
        const Own own = own_tokens(a, u.b < a.batch ? len_of(u.b) : 0);
        u.start = own.start;
        u.len = own.len;
        u.tiles = u.b < a.batch ? tiles_of(u.len) : 0x3fffffff;
      } while (u.tiles == 0);
    }
  };
  const int per_thread = (a.batch + kThreads - 1) / kThreads;
  const int b_lo = min(a.batch, (int)threadIdx.x * per_thread), b_hi = min(a.batch, b_lo + per_thread);
  long long mine = 0;    // tiles in the low 40 bits, sequences that have some above
  long long groups = 0;  // scoring: of scores
  for (int b = b_lo; b < b_hi; ++b) {
    const int raw = __ldcg(a.lens + b);
    const int len = (int)min((long long)max(raw, 0), cap);
    if (raw != len) atomicOr(a.status, kDevBadLength);
    if (b < kLensCached) s_lens[b] = len;
    const int own = own_tokens(a, len).len;
    mine += tiles_of(own) + (own > 0 ? 1ll << 40 : 0);
    groups += groups_of(tiles_of(own));
  }
  // exclusive prefix over the threads, and the sum of all
  auto prefix = [&](long long x, long long* s_sum, long long& all) {
    long long ahead = x;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, ahead, off);
      if (lane >= off) ahead += y;
    }
    if (lane == 31) s_sum[warp] = ahead;
    __syncthreads();
    ahead -= x;
    all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) ahead += s_sum[w];
      all += s_sum[w];
    }
    return ahead;
  };
  long long all, groups_ahead = 0;
  const long long ahead = prefix(mine, s_sum[0], all);
  if constexpr (kScored) {
    long long all_groups;
    groups_ahead = prefix(groups, s_sum[1], all_groups);
    if (blockIdx.x == 0) {
      long long at = groups_ahead;
      for (int b = b_lo; b < b_hi; ++b) {
        a.seq_groups[b] = at;
        at += groups_of(tiles_of(len_of(b)));
      }
      if (threadIdx.x == 0) a.seq_groups[a.batch] = all_groups;
    }
  }
  constexpr long long kLow = (1ll << 40) - 1;
  const long long total = (all & kLow) * hkv, units = (all >> 40) * hkv;
  if (total == 0) {
    grid_dependency_wait();
    return;
  }
  const long long span = total + units * kUnitCost;
  const int workers = (int)min((long long)gridDim.x, max((total + kMinTiles - 1) / kMinTiles, units));
  const int me = blockIdx.x;
  if (me >= workers) {
    grid_dependency_wait();
    return;
  }
  const Shares sh{quotient(span, workers), span - quotient(span, workers) * workers};
  const int share = (int)(sh.start(me + 1) - sh.start(me));
  {
    // found by the thread that counted the sequence in which the share starts
    const long long begin = ((ahead & kLow) + (ahead >> 40) * kUnitCost) * hkv;
    const long long stop = begin + ((mine & kLow) + (mine >> 40) * kUnitCost) * hkv;
    const long long x = sh.start(me);
    if (x >= begin && x < stop) {
      long long at = begin, group0 = groups_ahead * hkv;
      Unit u{0, 0, 0, 0, 0, b_lo, 0};
      for (;; ++u.b) {  // by whole sequences
        const Own own = own_tokens(a, len_of(u.b));
        u.start = own.start;
        u.len = own.len;
        u.tiles = tiles_of(u.len);
        const long long span_b = u.tiles ? (long long)(u.tiles + kUnitCost) * hkv : 0;
        if (x < at + span_b) break;
        at += span_b;
        group0 += (long long)groups_of(u.tiles) * hkv;
      }
      u.kvh = (int)quotient(x - at, u.tiles + kUnitCost);
      u.base = (int)(at + (long long)u.kvh * (u.tiles + kUnitCost) + kUnitCost - x);
      u.group0 = group0 + (long long)u.kvh * groups_of(u.tiles);
      s_first = u;
    }
  }
  __syncthreads();
  const Unit u0 = s_first;
  auto in_share = [&](const Unit& u) { return u.base < share; };
  auto tiles_end = [&](const Unit& u) { return min(share, u.base + u.tiles); };

  // ---- the warp's ring.  Rows are read once: they leave L2 before the scores do ----
  const uint64_t policy = make_evict_first_policy();
  uint8_t* const ring = smem + warp * C::kWarpBytes;
  constexpr int kChunks = D / 8, kRowsPer = 32 / kChunks;  // a warp copies kRowsPer rows (512 bytes) at a time
  // chunk c of row r lies at r kRowBytes + ((c ^ (r & 7)) << 4): eight rows of a matrix hit distinct banks
  const int c_row = lane / kChunks;
  const uint32_t copy_at = c_row * C::kRowBytes + (((lane % kChunks) ^ c_row) << 4);
  Unit pu = u0;                           // where the next tile to fetch lies
  int pid = max(pu.base, 0) + warp;       // its number
  int page = 0;                           // its page, fetched a tile ahead
  bool more = in_share(pu);
  const int log2 = a.index.page_log2;
  auto fetch_page = [&] {
    while (more && pid >= tiles_end(pu)) {
      next_unit(pu);
      pid = pu.base + warp;
      more = in_share(pu);
    }
    if (!more) return;
    const int pos = pu.start + (pid - pu.base) * kTile;
    page = __ldcg(a.index.block_table + (long long)pu.b * a.index.pages_per_seq + (pos >> log2));
  };
  auto fetch_tile = [&](int stage) {
    if (more) {
      const uint32_t st = smem_addr(ring) + stage * C::kStageBytes + copy_at;
      const int pos = pu.start + (pid - pu.base) * kTile;
      if ((unsigned)page >= (unsigned)a.index.num_pages) {
        atomicOr(a.status, kDevBadPage);
        page = 0;
      }
      const long long row0 = (((long long)page * hkv + pu.kvh) << log2) + (pos & ((1 << log2) - 1));
      const char* ks = reinterpret_cast<const char*>(a.k + row0 * D) + lane * 16;
      const char* vs = reinterpret_cast<const char*>(a.v + row0 * D) + lane * 16;
#pragma unroll
      for (int i = 0; i < kTile / kRowsPer; ++i) {
        const uint32_t to = (st ^ ((i * kRowsPer & 7) << 4)) + i * 512;
        cp_async16<0>(to, ks + i * 512, policy);
        cp_async16<C::kRowsBytes>(to, vs + i * 512, policy);
      }
      pid += kWarps;
      fetch_page();
    }
    cp_async_commit();
  };
  fetch_page();
#pragma unroll
  for (int s = 0; s < C::kStages - 1; ++s) fetch_tile(s);

  // ldmatrix addresses: K rows as they are (tokens), V's transposed (dims)
  const uint32_t k_row = (lane & 7) + (lane & 8), v_row = (lane & 7) + (lane >> 4 << 3);
  const uint32_t k_at = k_row * C::kRowBytes + (((lane >> 4) ^ (lane & 7)) << 4);
  const uint32_t v_at = C::kRowsBytes + v_row * C::kRowBytes + ((((lane >> 3) & 1) ^ (lane & 7)) << 4);

  // ---- units of this CTA ----
  int stage = 0;
  for (Unit u = u0; in_share(u); next_unit(u)) {
    const int end = tiles_end(u);
    uint32_t qf[NG][KS][2];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const int h = n * 8 + g;
      const uint32_t* src =
          reinterpret_cast<const uint32_t*>(a.q + ((long long)u.b * a.n_q_heads + u.kvh * G + h) * D) + t4;
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        qf[n][j][0] = h < G ? __ldcg(src + 8 * j) : 0;
        qf[n][j][1] = h < G ? __ldcg(src + 8 * j + 4) : 0;
      }
    }
    float R[NG][2], l[NG][2], o[NG][KS][4];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      R[n][0] = R[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }

    for (int id = max(u.base, 0) + warp; id < end; id += kWarps) {
      cp_async_wait<C::kStages - 2>();
      __syncwarp();
      fetch_tile(stage == 0 ? C::kStages - 1 : stage - 1);
      uint8_t* const st = ring + stage * C::kStageBytes;
      const uint32_t sa = smem_addr(st);
      stage = stage + 1 == C::kStages ? 0 : stage + 1;

      // ---- scores of tokens g (0, 1) and g + 8 (2, 3), heads 2 t4 and 2 t4 + 1 ----
      float s[NG][4];
#pragma unroll
      for (int n = 0; n < NG; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        uint32_t k[4];
        ldmatrix(k, sa + (k_at ^ (j << 5)));
#pragma unroll
        for (int n = 0; n < NG; ++n) mma_bf16(s[n], k, qf[n][j][0], qf[n][j][1]);
      }
      const int first = (id - u.base) * kTile, valid = u.len - first;
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] *= a.scale_log2;
      if (valid < kTile) {  // the sequence's last tile: nothing past its end counts, whatever lies there
        for (int i = max(valid, 0) * kChunks + lane; i < kTile * kChunks; i += 32)
          reinterpret_cast<uint4*>(st + C::kRowsBytes)[i] = make_uint4(0, 0, 0, 0);
        __syncwarp();
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (g + 8 * (i >> 1) >= valid) s[n][i] = -INFINITY;
      }
      if constexpr (kScored) {
        const int tile = id - u.base;
        const long long group = u.group0 + tile / 2;
        if (group < a.score_groups) {
          float* const dst = a.scores + (group * G + 2 * t4) * kGroup + tile % 2 * kTile + g;
#pragma unroll
          for (int n = 0; n < NG; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (8 * n + 2 * t4 + (i & 1) < G) dst[(8 * n + (i & 1)) * kGroup + 8 * (i >> 1)] = s[n][i];
        }
      }

      // ---- move R where a score passes it by far ----
      bool over = false;
#pragma unroll
      for (int n = 0; n < NG; ++n)
        over |= fmaxf(s[n][0], s[n][2]) > R[n][0] + kSlack || fmaxf(s[n][1], s[n][3]) > R[n][1] + kSlack;
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float m = fmaxf(s[n][c], s[n][2 + c]);
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
            if (m > R[n][c] + kSlack) {
              const float f = ex2_ftz(R[n][c] - m);
              R[n][c] = m;
              l[n][c] *= f;
#pragma unroll
              for (int i = 0; i < KS; ++i) {
                o[n][i][c] *= f;
                o[n][i][2 + c] *= f;
              }
            }
          }
      }

      // ---- weights as the second operand: tokens 2 t4, 2 t4 + 1 (and + 8) of column g ----
      uint32_t pf[NG][2], pr[NG][2];
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float p0 = ex2_ftz(s[n][2 * i] - R[n][0]), p1 = ex2_ftz(s[n][2 * i + 1] - R[n][1]);
          l[n][0] += p0;
          l[n][1] += p1;
          const uint32_t hi = pack2_rn(p0, p1);
          pf[n][i] = transpose8x8(hi);
          pr[n][i] = transpose8x8(pack2_rn(p0 - bf16lo(hi), p1 - bf16hi(hi)));
        }

      // ---- O^T += V^T P^T: block c holds dims 16 c + g and 16 c + g + 8 ----
#pragma unroll
      for (int c = 0; c < KS; ++c) {
        uint32_t v[4];
        ldmatrix_trans(v, sa + (v_at ^ (c << 5)));
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          mma_bf16(o[n][c], v, pf[n][0], pf[n][1]);
          mma_bf16(o[n][c], v, pr[n][0], pr[n][1]);
        }
      }
      __syncwarp();
    }

    // ---- the unit's end: the warps join through the stages that held their last tiles ----
    const int idle = (stage == 0 ? C::kStages : stage) - 1;
    float* const sums = reinterpret_cast<float*>(ring + idle * C::kStageBytes);
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], off);
        if (g == 0) s_ml[warp][n * 8 + 2 * t4 + c] = make_float2(R[n][c], l[n][c]);
      }
    if (lane == 0) s_idle[warp] = warp * C::kWarpBytes + idle * C::kStageBytes;
    const long long at0 = sh.start(me) + u.base;
    const int index = u.b * hkv + u.kvh, slot = index + me;
    if (threadIdx.x == 0 && u.base >= 0)  // the unit starts here
      a.units[index] = UnitParts{slot, sh.cta(at0 + u.tiles - 1) - me + 1};
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NG; ++n) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_ml[w][n * 8 + 2 * t4 + c].x);
        const float f = R[n][c] == top ? 1.f : ex2_ftz(R[n][c] - top);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          sums[(2 * t4 + c) * C::kPitch + 16 * i + g] = o[n][i][c] * f;
          sums[(2 * t4 + c) * C::kPitch + 16 * i + g + 8] = o[n][i][2 + c] * f;
        }
      }
      __syncthreads();
      const int heads = min(8, G - 8 * n);
      for (int item = threadIdx.x; item < heads * (D / 4); item += kThreads) {
        const int hl = item / (D / 4), d = item % (D / 4) * 4, h = 8 * n + hl;
        float top = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_ml[w][h].x);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float2 ml = s_ml[w][h];
          L = fmaf(ml.y, ml.x == top ? 1.f : ex2_ftz(ml.x - top), L);
          const float4 y = *reinterpret_cast<const float4*>(
              reinterpret_cast<const float*>(smem + s_idle[w]) + hl * C::kPitch + d);
          x.x += y.x;
          x.y += y.y;
          x.z += y.z;
          x.w += y.w;
        }
        *reinterpret_cast<float4*>(a.part_acc + ((long long)slot * G + h) * D + d) = x;
        if (d == 0) a.part_ml[(long long)slot * G + h] = make_float2(top, L);
      }
      __syncthreads();  // the idle stages may be filled again
    }
  }
  cp_async_wait<0>();
  allow_dependent_launch();  // not before: the join's blocks would take the room of this grid's
  grid_dependency_wait();
}

// ---- the second launch ----
constexpr int kJoinThreads = 256;
constexpr int kJoinWarps = kJoinThreads / 32;
constexpr int kAhead = 2;      // times four tokens of a thread whose scores are in flight
constexpr int kFewParts = 32;  // parts of a row that one warp joins

// What a row's result is joined from.
struct Parts {
  long long row;
  int h, slot0, prefix, all;
};

// Joins the parts of kJoinWarps output rows: a warp to a row, and the rows of many
// parts by the whole block, one after the other.
template <int D>
__device__ __forceinline__ void join_rows(const Args& a, int block) {
  constexpr int kLanes = D / 4, kSub = kJoinThreads / kLanes;  // lanes of a row, parts in flight
  __shared__ float4 s_x[kSub][kLanes];
  __shared__ float s_l[kSub];
  __shared__ Parts s_many[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.group;
  const long long rows = (long long)a.batch * a.n_q_heads, row0 = (long long)block * kJoinWarps;
  // part i of a row: of the prefix, then of the unit
  auto ml_of = [&](const Parts& up, int i) {
    return i < up.prefix ? a.prefix_ml + i * rows + up.row
                         : a.part_ml + (long long)(up.slot0 + i - up.prefix) * G + up.h;
  };
  auto acc_of = [&](const Parts& up, int i) {
    return i < up.prefix ? a.prefix_acc + (i * rows + up.row) * D
                         : a.part_acc + ((long long)(up.slot0 + i - up.prefix) * G + up.h) * D;
  };
  auto largest = [&](const Parts& up) {
    float M = -INFINITY;
    for (int i = lane; i < up.all; i += 32) M = fmaxf(M, __ldcg(ml_of(up, i)).x);
#pragma unroll
    for (int off = 16; off; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
    return M;
  };
  // parts i0, i0 + step, ..
  auto sum = [&](const Parts& up, float M, int i0, int step, int at, float& L) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = i0; i < up.all; i += step) {
      const float2 ml = __ldcg(ml_of(up, i));
      const float4 y = __ldcg(reinterpret_cast<const float4*>(acc_of(up, i)) + at);
      const float f = ml.x == M ? 1.f : ex2_ftz(ml.x - M);
      L = fmaf(ml.y, f, L);
      x.x = fmaf(y.x, f, x.x);
      x.y = fmaf(y.y, f, x.y);
      x.z = fmaf(y.z, f, x.z);
      x.w = fmaf(y.w, f, x.w);
    }
    return x;
  };
  auto store = [&](long long row, int at, const float4& x, float L) {
    const float inv = 1.f / L;
    reinterpret_cast<uint2*>(a.o + row * D)[at] =
        make_uint2(pack2_rn(x.x * inv, x.y * inv), pack2_rn(x.z * inv, x.w * inv));
  };
  {
    const long long row = row0 + warp;
    Parts up{row, 0, 0, 0, 0};
    if (row < rows) {
      const int b = (int)(row / a.n_q_heads), hq = (int)(row % a.n_q_heads);
      up.h = hq % G;
      const int len = (int)min((long long)__ldcg(a.lens + b), a.index.capacity());
      const Own own = own_tokens(a, len);
      if (own.start > 0) up.prefix = up.all = a.splits;
      if (own.len > 0) {
        const UnitParts unit = a.units[b * a.index.n_kv_heads + hq / G];
        up.slot0 = unit.slot0;
        up.all += unit.parts;
      }
      const int at = lane % kLanes;
      if (len <= 0) {
        if (lane < kLanes) reinterpret_cast<uint2*>(a.o + row * D)[at] = make_uint2(0, 0);
      } else if (up.all <= kFewParts) {
        float L = 0.f;
        const float4 x = sum(up, largest(up), 0, 1, at, L);
        if (lane < kLanes) store(row, at, x, L);
      }
    }
    if (lane == 0) s_many[warp] = up;
  }
  __syncthreads();
  for (int r = 0; r < kJoinWarps; ++r) {
    const Parts up = s_many[r];
    if (up.all <= kFewParts) continue;
    const int sub = threadIdx.x / kLanes, at = threadIdx.x % kLanes;
    float L = 0.f;
    const float4 part = sum(up, largest(up), sub, kSub, at, L);
    s_x[sub][at] = part;
    if (at == 0) s_l[sub] = L;
    __syncthreads();
    if (threadIdx.x < kLanes) {
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      L = 0.f;
#pragma unroll
      for (int i = 0; i < kSub; ++i) {
        const float4 y = s_x[i][at];
        L += s_l[i];
        x.x += y.x;
        x.y += y.y;
        x.z += y.z;
        x.w += y.w;
      }
      store(row0 + r, at, x, L);
    }
    __syncthreads();
  }
}

// Adds the weights of an equal run of all groups, four tokens to a thread.
__device__ __forceinline__ void add_weights(const Args& a, int block, int blocks) {
  __shared__ float2 s_ml[16];  // each head's (M, 1 / L)
  __shared__ int s_seq;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.group, hkv = a.index.n_kv_heads, log2 = a.index.page_log2;
  const long long total = __ldcg(a.seq_groups + a.batch) * hkv;
  const long long room = min(total, a.score_groups);
  if (room < total && block == 0 && threadIdx.x == 0) atomicOr(a.status, kDevScoreRoom);
  const long long per = (room + blocks - 1) / blocks;
  const long long lo = block * per, hi = min(room, lo + per);
  if (lo >= hi) return;
  for (int b = threadIdx.x; b < a.batch; b += kJoinThreads)  // the sequence with group lo
    if (__ldcg(a.seq_groups + b) * hkv <= lo && lo < __ldcg(a.seq_groups + b + 1) * hkv) s_seq = b;
  __syncthreads();
  int b = s_seq;
  long long first = __ldcg(a.seq_groups + b);
  int groups = (int)(__ldcg(a.seq_groups + b + 1) - first);
  int kvh = (int)quotient(lo - first * hkv, groups);
  long long at = first * hkv + (long long)kvh * groups;  // the unit's first group
  while (true) {
    const UnitParts up = a.units[b * hkv + kvh];
    const int len = (int)min((long long)__ldcg(a.lens + b), a.index.capacity());
    const int t0 = (int)(max(lo, at) - at) * kGroup, t1 = min((int)(min(hi, at + groups) - at) * kGroup, len);
    const int32_t* const pages = a.index.block_table + (long long)b * a.index.pages_per_seq;
    auto page_of = [&](int t) { return t < t1 ? __ldg(pages + (t >> log2)) : -1; };
    constexpr int kStep = 4 * kJoinThreads;
    int page[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) page[j] = page_of(t0 + kStep * j + 4 * threadIdx.x);
    for (int h = warp; h < G; h += kJoinWarps) {
      float M = -INFINITY, L = 0.f;
      auto join = [&](float m, float l) {
        const float to = fmaxf(M, m);
        L = L * (M == to ? 1.f : ex2_ftz(M - to)) + l * (m == to ? 1.f : ex2_ftz(m - to));
        M = to;
      };
      for (int p = lane; p < up.parts; p += 32) {
        const float2 x = __ldcg(a.part_ml + (long long)(up.slot0 + p) * G + h);
        join(x.x, x.y);
      }
#pragma unroll
      for (int off = 16; off; off >>= 1)
        join(__shfl_xor_sync(0xffffffffu, M, off), __shfl_xor_sync(0xffffffffu, L, off));
      if (lane == 0) s_ml[h] = make_float2(M, 1.f / L);
    }
    __syncthreads();
    for (int t = t0 + 4 * threadIdx.x; t < t1; t += kStep * kAhead) {
      const float4* s[kAhead];
      long long row[kAhead];
      float4 w[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int x = t + kStep * j;
        const bool there = x < t1 && (unsigned)page[j] < (unsigned)a.index.num_pages;  // else flagged before
        row[j] = there ? (((long long)page[j] * hkv + kvh) << log2) + (x & ((1 << log2) - 1)) : -1;
        s[j] = reinterpret_cast<const float4*>(
            a.scores + (there ? (at + x / kGroup) * (G * kGroup) + x % kGroup : 0));
        w[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (there) w[j] = __ldcg(reinterpret_cast<const float4*>(a.w_in + row[j]));
        page[j] = page_of(x + kStep * kAhead);
      }
      float4 sum[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) sum[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int i = 0; i < G; ++i) {
        const float2 x = s_ml[i];
        float4 y[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) y[j] = __ldcg(s[j] + i * (kGroup / 4));
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          sum[j].x = fmaf(ex2_ftz(y[j].x - x.x), x.y, sum[j].x);
          sum[j].y = fmaf(ex2_ftz(y[j].y - x.x), x.y, sum[j].y);
          sum[j].z = fmaf(ex2_ftz(y[j].z - x.x), x.y, sum[j].z);
          sum[j].w = fmaf(ex2_ftz(y[j].w - x.x), x.y, sum[j].w);
        }
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (row[j] < 0) continue;
        const int left = t1 - (t + kStep * j);
        const float4 v =
            make_float4(w[j].x + sum[j].x, w[j].y + sum[j].y, w[j].z + sum[j].z, w[j].w + sum[j].w);
        float* const to = a.w_out + row[j];
        if (left >= 4) {
          *reinterpret_cast<float4*>(to) = v;
        } else {
          to[0] = v.x;
          if (left > 1) to[1] = v.y;
          if (left > 2) to[2] = v.z;
        }
      }
    }
    at += groups;
    if (at >= hi) return;
    if (++kvh == hkv) {
      kvh = 0;
      do {
        ++b;
        first = __ldcg(a.seq_groups + b);
        groups = (int)(__ldcg(a.seq_groups + b + 1) - first);
      } while (groups == 0);
    }
    __syncthreads();  // s_ml is free again
  }
}

// The blocks of weights, of one wave, come first: they take longer than the others.
template <int D, bool kScored>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ Args a, int weight_blocks) {
  allow_dependent_launch();
  grid_dependency_wait();
  if constexpr (kScored) {
    if ((int)blockIdx.x < weight_blocks) {
      add_weights(a, blockIdx.x, weight_blocks);
      return;
    }
  }
  join_rows<D>(a, blockIdx.x - weight_blocks);
}

// Workspace: status word | units | partial results | scores, or the prefix's results.
struct Layout {
  size_t units_off, seq_off, ml_off, acc_off, scores_off, prefix_ml_off, prefix_acc_off, total;
  long long score_groups;
};

Layout layout(int batch, int n_kv_heads, int group, int head_dim, long long score_tokens, size_t prefix_rows) {
  const size_t units = (size_t)batch * n_kv_heads, slots = units + kMostCtasPerSm * (size_t)std::max(1, device_sm_count());
  Layout w;
  w.units_off = kStatusBytes;
  w.seq_off = w.units_off + up256(units * sizeof(UnitParts));
  w.ml_off = w.seq_off + up256(((size_t)batch + 1) * sizeof(long long));
  w.acc_off = w.ml_off + up256(slots * group * sizeof(float2));
  w.scores_off = w.acc_off + up256(slots * group * head_dim * sizeof(float));
  // every sequence's scores start in a group of their own
  w.score_groups = score_tokens ? (score_tokens / kGroup + batch) * n_kv_heads : 0;
  w.prefix_ml_off = w.scores_off + up256((size_t)w.score_groups * kGroup * group * sizeof(float));
  w.prefix_acc_off = w.prefix_ml_off + up256(prefix_rows * sizeof(float2));
  w.total = w.prefix_acc_off + up256(prefix_rows * head_dim * sizeof(float));
  return w;
}

template <int D, int NG, bool kScored>
cudaError_t launch(const Args& a, cudaStream_t stream) {
  using C = Cfg<D, NG>;
  const void* fn = reinterpret_cast<const void*>(&own_tokens_kernel<D, NG, kScored>);
  {
    static std::mutex mu;
    static uint64_t done = 0;  // the shared-memory opt-in is per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    std::lock_guard<std::mutex> lock(mu);
    if (dev > 63 || !(done >> dev & 1)) {
      e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
      if (e != cudaSuccess) return e;
      if (dev <= 63) done |= 1ull << dev;
    }
  }
  // no more CTAs than a full cache could feed, one for each unit at least
  const long long units = (long long)a.batch * a.index.n_kv_heads;
  const long long tiles = units * ((a.index.capacity() + kTile - 1) / kTile);
  const long long ctas = std::min<long long>(device_sm_count() * C::kCtasPerSm, std::max(units, (tiles + kMinTiles - 1) / kMinTiles));
  Args args = a;
  void* p[] = {&args};
  cudaError_t e = launch_with_pdl(fn, dim3((unsigned)ctas), dim3(kThreads), p, C::kSmemBytes, stream);
  if (e != cudaSuccess) return e;
  const long long rows = (long long)a.batch * a.n_q_heads;
  int weight_blocks = 0;
  if (kScored) weight_blocks = (int)std::min<long long>(device_sm_count() * 3, (tiles + 31) / 32);
  const int blocks = weight_blocks + (int)((rows + kJoinWarps - 1) / kJoinWarps);
  void* p2[] = {&args, &weight_blocks};
  return launch_with_pdl(reinterpret_cast<const void*>(&join_kernel<D, kScored>), dim3((unsigned)blocks),
                         dim3(kJoinThreads), p2, 0, stream);
}

}  // namespace

namespace paged {

int check_paged_pool(const void* k_pages, const void* v_pages, const void* block_table, int n_kv_heads, int head_dim,
                     int page_size, int pages_per_seq, int num_pages, int batch, PoolIndex* index) {
  if (head_dim != 64 && head_dim != 128) return set_last_error(LARA_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  if (page_size < 16 || page_size > 65536 || (page_size & (page_size - 1)))
    return set_last_error(LARA_ERR_BAD_CFG, "page_size must be a power of two in [16, 65536]");
  if (batch < 0 || batch > 65535) return set_last_error(LARA_ERR_BAD_CFG, "batch must be in [0, 65535]");
  if (n_kv_heads < 1 || n_kv_heads > 65535 || num_pages < 1 || pages_per_seq < 1 ||
      (long long)pages_per_seq * page_size > 0x3fffffffll || (long long)batch * n_kv_heads > 0x3fffffffll ||
      (double)batch * n_kv_heads * pages_per_seq * page_size > 0x1p40)
    return set_last_error(LARA_ERR_BAD_CFG,
                          "bad paged-cache geometry (at most 2^30 - 1 tokens a sequence, 2^40 rows in all)");
  if (batch == 0) return LARA_OK;
  if (!k_pages || !v_pages || !block_table) return set_last_error(LARA_ERR_STREAM_DEST, "null pointer");
  if (!aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(block_table, 4))
    return set_last_error(LARA_ERR_STREAM_DEST, "k_pages and v_pages must be 16-byte aligned");
  index->block_table = static_cast<const int32_t*>(block_table);
  index->pages_per_seq = pages_per_seq;
  index->page_log2 = __builtin_ctz(page_size);
  index->num_pages = num_pages;
  index->n_kv_heads = n_kv_heads;
  return LARA_OK;
}

int check_weights(const float* in, const float* out, int n_kv_heads, int page_size, int num_pages) {
  if (!in || !out) return set_last_error(LARA_ERR_STREAM_DEST, "null pointer");
  if (!aligned(in, 16) || !aligned(out, 16))
    return set_last_error(LARA_ERR_STREAM_DEST, "weights must be 16-byte aligned");
  if (in != out && kvq::overlap(in, out, (size_t)num_pages * n_kv_heads * page_size * 4))
    return set_last_error(LARA_ERR_STREAM_DEST, "weights_out must be weights or lie apart from them");
  return LARA_OK;
}

}  // namespace paged

}  // namespace lara

using namespace lara;

namespace {

// The checks and arguments that the two decodes have in common.
int decode_args(Args& a, const uint16_t* q, const uint16_t* k_pages, const uint16_t* v_pages,
                const int32_t* block_table, const int32_t* seq_lens, uint16_t* o, int batch, int n_q_heads,
                int n_kv_heads, int head_dim, int page_size, int pages_per_seq, int num_pages, float scale,
                const void* workspace) {
  if (const int rc = check_paged_pool(k_pages, v_pages, block_table, n_kv_heads, head_dim, page_size, pages_per_seq,
                                      num_pages, batch, &a.index))
    return rc;
  if (n_q_heads < 1 || n_q_heads % n_kv_heads)
    return set_last_error(LARA_ERR_BAD_CFG, "n_q_heads must be a multiple of n_kv_heads");
  if (n_q_heads / n_kv_heads > 16)
    return set_last_error(LARA_ERR_UNSUPPORTED, "groups of at most 16 query heads per kv head");
  if (!(scale > 0.f) || !std::isfinite(scale))
    return set_last_error(LARA_ERR_BAD_CFG, "scale must be positive and finite");
  if (batch == 0) return LARA_OK;
  if (!q || !seq_lens || !o || !workspace) return set_last_error(LARA_ERR_STREAM_DEST, "null pointer");
  if (!aligned(q, 16) || !aligned(o, 16) || !aligned(seq_lens, 4) || !aligned(workspace, 256))
    return set_last_error(LARA_ERR_STREAM_DEST, "q and o must be 16-byte aligned, the workspace 256-byte");
  a.q = q;
  a.k = k_pages;
  a.v = v_pages;
  a.lens = seq_lens;
  a.o = o;
  a.batch = batch;
  a.n_q_heads = n_q_heads;
  a.group = n_q_heads / n_kv_heads;
  a.scale_log2 = scale * 1.4426950408889634f;
  return LARA_OK;
}

void place(Args& a, const Layout& w, void* workspace) {
  char* base = static_cast<char*>(workspace);
  a.status = reinterpret_cast<int*>(base);
  a.units = reinterpret_cast<UnitParts*>(base + w.units_off);
  a.seq_groups = reinterpret_cast<long long*>(base + w.seq_off);
  a.part_ml = reinterpret_cast<float2*>(base + w.ml_off);
  a.part_acc = reinterpret_cast<float*>(base + w.acc_off);
  a.scores = reinterpret_cast<float*>(base + w.scores_off);
  a.score_groups = w.score_groups;
}

template <bool kScored>
cudaError_t launch_any(const Args& a, int head_dim, cudaStream_t st) {
  if (head_dim == 128) return a.group <= 8 ? launch<128, 1, kScored>(a, st) : launch<128, 2, kScored>(a, st);
  return a.group <= 8 ? launch<64, 1, kScored>(a, st) : launch<64, 2, kScored>(a, st);
}

// Tokens whose scores a call can leave: those of every page its tables can name.
long long score_tokens(int batch, int page_size, int pages_per_seq, int num_pages) {
  return std::min<long long>((long long)batch * pages_per_seq, num_pages) * page_size;
}

}  // namespace

extern "C" size_t lara_decode_scored_workspace_bytes(int batch, int n_q_heads, int n_kv_heads, int head_dim,
                                                     int page_size, int pages_per_seq, int num_pages) {
  if (batch < 1 || n_q_heads < 1 || n_kv_heads < 1 || head_dim < 1 || page_size < 1 || pages_per_seq < 1 ||
      num_pages < 1)
    return 0;
  return layout(batch, n_kv_heads, (n_q_heads + n_kv_heads - 1) / n_kv_heads, head_dim,
                score_tokens(batch, page_size, pages_per_seq, num_pages), 0)
      .total;
}

extern "C" int lara_gqa_decode_scored(const uint16_t* q, const uint16_t* k_pages, const uint16_t* v_pages,
                                      const float* weights, float* weights_out, const int32_t* block_table,
                                      const int32_t* seq_lens, uint16_t* o, int batch, int n_q_heads, int n_kv_heads,
                                      int head_dim, int page_size, int pages_per_seq, int num_pages, float scale,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  LARA_NVTX("lara_gqa_decode_scored");
  Args a{};
  if (const int rc = decode_args(a, q, k_pages, v_pages, block_table, seq_lens, o, batch, n_q_heads, n_kv_heads,
                                 head_dim, page_size, pages_per_seq, num_pages, scale, workspace))
    return rc;
  if (batch == 0) return LARA_OK;
  if (const int rc = check_weights(weights, weights_out, n_kv_heads, page_size, num_pages)) return rc;
  const Layout w = layout(batch, n_kv_heads, a.group, head_dim,
                          score_tokens(batch, page_size, pages_per_seq, num_pages), 0);
  if (workspace_bytes < w.total) return set_last_error(LARA_ERR_RESULT_LEN, "scored decode workspace too small");
  place(a, w, workspace);
  a.w_in = weights;
  a.w_out = weights_out;
  const cudaError_t e = launch_any<true>(a, head_dim, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess)
    return set_last_error(LARA_ERR_CUDA, std::string("scored decode launch: ") + cudaGetErrorString(e));
  return LARA_OK;
}

extern "C" size_t lara_decode_shared_workspace_bytes(int batch, int n_q_heads, int n_kv_heads, int head_dim) {
  if (batch < 1 || n_q_heads < 1 || n_kv_heads < 1 || head_dim < 1) return 0;
  const int group = std::min(16, (n_q_heads + n_kv_heads - 1) / n_kv_heads);
  // a wave of CTAs, of two row tiles each, or one split of all rows; of this or any smaller batch
  const size_t rows = (size_t)batch * n_kv_heads * group, sms = std::max(1, device_sm_count());
  const size_t most = std::min(rows * std::max<size_t>(1, sms / n_kv_heads), std::max(rows, 256 * sms));
  return layout(batch, n_kv_heads, group, head_dim, 0, most).total;
}

extern "C" int lara_gqa_decode_shared(const uint16_t* q, const uint16_t* k_pages, const uint16_t* v_pages,
                                      const int32_t* block_table, const int32_t* seq_lens, uint16_t* o, int batch,
                                      int n_q_heads, int n_kv_heads, int head_dim, int page_size, int pages_per_seq,
                                      int num_pages, int shared_pages, float scale, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  LARA_NVTX("lara_gqa_decode_shared");
  Args a{};
  if (const int rc = decode_args(a, q, k_pages, v_pages, block_table, seq_lens, o, batch, n_q_heads, n_kv_heads,
                                 head_dim, page_size, pages_per_seq, num_pages, scale, workspace))
    return rc;
  if (shared_pages < 0 || shared_pages > pages_per_seq)
    return set_last_error(LARA_ERR_BAD_CFG, "shared_pages must be in [0, pages_per_seq]");
  if (batch == 0) return LARA_OK;
  const long long tokens = (long long)shared_pages * page_size;
  const PrefixPlan plan = prefix_plan(batch, n_kv_heads, a.group, (int)tokens);
  const Layout w = layout(batch, n_kv_heads, a.group, head_dim, 0,
                          tokens ? (size_t)batch * n_q_heads * plan.splits : 0);
  if (workspace_bytes < w.total) return set_last_error(LARA_ERR_RESULT_LEN, "shared decode workspace too small");
  place(a, w, workspace);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if (tokens) {
    char* base = static_cast<char*>(workspace);
    float2* const ml = reinterpret_cast<float2*>(base + w.prefix_ml_off);
    float* const acc = reinterpret_cast<float*>(base + w.prefix_acc_off);
    a.shared_tokens = (int)tokens;
    a.splits = plan.splits;
    a.prefix_ml = ml;
    a.prefix_acc = acc;
    e = prefix_launch(plan, q, k_pages, v_pages, a.index, (int)tokens, batch, n_q_heads, head_dim, a.scale_log2, ml,
                      acc, a.status, st);
  }
  if (e == cudaSuccess) e = launch_any<false>(a, head_dim, st);
  if (e != cudaSuccess)
    return set_last_error(LARA_ERR_CUDA, std::string("shared decode launch: ") + cudaGetErrorString(e));
  return LARA_OK;
}
