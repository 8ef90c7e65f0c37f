// The pass over the tokens that sequences have for themselves, in decodes over
// the paged bf16 cache (sm_100a).
#pragma once

#include "paged.cuh"

namespace lara {
namespace paged {

constexpr int kTile = 16;            // tokens per warp and stage: never across pages
constexpr int kGroup = 32;           // tokens whose scores lie together, head by head (a line of 128 bytes)
constexpr int kUnitCost = 8;         // what a unit costs beside its tiles, in tiles
constexpr int kMostPerSm = 12;       // CTAs or, of short units, warps to an SM that take parts of units
// Tiles go to warps, not CTAs, while that leaves at most this many parts of a unit: 64 sequences of up
// to 512 own tokens behind 8192 42 us, 70 by CTAs; 4 of up to 48 12.2 against 13.7; 37 of up to 333 (16
// parts) 22.4 by warps, 19.7 by CTAs.  Scored, always CTAs: 64 x 4096 tokens 193 us by warps, 181.
constexpr int kSoloParts = 4;
constexpr int kLensCached = 1024;    // lengths kept in shared memory
// R moves only when a score passes it by this much (log2): weights stay below 2^8.
constexpr float kSlack = 8.f;

// A pass by CTAs of W warps, each with a ring of S stages.
template <int D, int NG, int W, int S>
struct OwnPass {
  static constexpr int kWarps = W, kThreads = W * 32, kStages = S;
  static constexpr int kMinTiles = W;  // tiles per CTA below which fewer CTAs run
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kRowsBytes = kTile * kRowBytes;  // K (or V) of a stage
  static constexpr int kStageBytes = 2 * kRowsBytes;
  static constexpr int kWarpBytes = kStages * kStageBytes;
  static constexpr int kSmemBytes = kWarps * kWarpBytes + 128;
  static constexpr int kPitch = D + 4;  // floats per head in the join (lanes of a store hit distinct banks)
  static_assert(8 * kPitch * 4 <= kStageBytes, "a stage holds the sums of eight heads");
};

struct DecodeArgs {
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
  // behind a shared prefix: its tokens, and what the pass over it leaves (PrefixPlan)
  int shared_tokens;
  PrefixPlan prefix;
  UnitParts* prefix_units;  // [kv heads * prefix.units]
  float2* prefix_ml;        // [prefix units + CTAs][prefix.rows] (reference, sum)
  float* prefix_acc;        // [prefix units + CTAs][prefix.rows][D]
  // scoring
  float* scores;           // [groups][group][kGroup], in the order of the units
  long long score_groups;  // that there is room for
  const float* w_in;      // [pages][kv heads][page]
  float* w_out;
};

// The first launch of a decode behind a shared prefix (paged_shared.cu).
cudaError_t shared_launch(const DecodeArgs& a, int head_dim, cudaStream_t stream);

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
__device__ __forceinline__ Own own_tokens(const DecodeArgs& a, int len) {
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
//
// First all threads of the block count the tokens (`totals`), then the pass's warps run `run`.
template <int D, int NG, int W, int S, bool kScored>
struct OwnTokens {
  using C = OwnPass<D, NG, W, S>;
  static constexpr long long kLow = (1ll << 40) - 1;
  struct Shared {
    long long sum[2][W];
    long long ahead[W * 32];                       // of each thread's sequences, packed as `mine`
    long long groups_ahead[kScored ? W * 32 : 1];
    float2 ml[W][NG * 8];
    int idle[W];
    int lens[kLensCached];
  };
  const DecodeArgs& a;
  Shared& sh_;
  long long total = 0, units = 0;  // tiles, and units with tokens
  int covering = 0x7fffffff;  // the first of the thread's sequences that covers the shared prefix

  __device__ __forceinline__ OwnTokens(const DecodeArgs& args, Shared& shared) : a(args), sh_(shared) {}

  __device__ __forceinline__ int load_len(int b) const {
    return (int)min((long long)max(__ldcg(a.lens + b), 0), a.index.capacity());
  }
  __device__ __forceinline__ int len_of(int b) const { return b < kLensCached ? sh_.lens[b] : load_len(b); }
  __device__ __forceinline__ void sync() const { asm volatile("bar.sync 9, %0;" ::"n"(C::kThreads) : "memory"); }

  // exclusive prefix over the pass's threads, and the sum of all; by the whole block
  __device__ __forceinline__ long long prefix(long long x, long long* sum, long long& all) const {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    long long ahead = x;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, ahead, off);
      if (lane >= off) ahead += y;
    }
    if (lane == 31 && warp < W) sum[warp] = ahead;
    __syncthreads();
    ahead -= x;
    all = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w < warp) ahead += sum[w];
      all += sum[w];
    }
    return ahead;
  }

  __device__ __forceinline__ void totals() {
    const int per_thread = (a.batch + C::kThreads - 1) / C::kThreads;
    const int b_lo = min(a.batch, (int)threadIdx.x * per_thread), b_hi = min(a.batch, b_lo + per_thread);
    long long mine = 0;    // tiles in the low 40 bits, sequences that have some above
    long long groups = 0;  // scoring: of scores
    for (int b = b_lo; b < b_hi; ++b) {
      const int raw = __ldcg(a.lens + b);
      const int len = (int)min((long long)max(raw, 0), a.index.capacity());
      if (raw != len) atomicOr(a.status, kDevBadLength);
      if (b < kLensCached) sh_.lens[b] = len;
      const Own own = own_tokens(a, len);
      mine += tiles_of(own.len) + (own.len > 0 ? 1ll << 40 : 0);
      groups += groups_of(tiles_of(own.len));
      if (own.start > 0) covering = min(covering, b);
    }
    long long all;
    const long long ahead = prefix(mine, sh_.sum[0], all);
    if (threadIdx.x < C::kThreads) sh_.ahead[threadIdx.x] = ahead;
    if constexpr (kScored) {
      long long all_groups;
      const long long groups_ahead = prefix(groups, sh_.sum[1], all_groups);
      sh_.groups_ahead[threadIdx.x] = groups_ahead;
      if (blockIdx.x == 0) {
        long long at = groups_ahead;
        for (int b = b_lo; b < b_hi; ++b) {
          a.seq_groups[b] = at;
          at += groups_of(tiles_of(len_of(b)));
        }
        if (threadIdx.x == 0) a.seq_groups[a.batch] = all_groups;
      }
    }
    total = (all & kLow) * a.index.n_kv_heads;
    units = (all >> 40) * a.index.n_kv_heads;
    __syncthreads();
  }

  __device__ __forceinline__ bool solo_units(int ctas) const {
    return !kScored && min((long long)ctas * W, total) <= units * kSoloParts;
  }

  // The pass's part `part` of `ctas`, by its warps.
  __device__ __forceinline__ void run(int part, int ctas, uint8_t* smem) {
    constexpr int KS = D / 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int G = a.group, hkv = a.index.n_kv_heads;
    if (total == 0) return;

    // ---- this CTA's share of all tiles, and the unit in which it starts ----
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
    const long long span = total + units * kUnitCost;
    // Short units go to warps, which leave a part each; longer ones to CTAs, whose warps take their
    // tiles in turn and join at the end.
    const bool solo = solo_units(ctas);
    const int step = solo ? 1 : W, offset = solo ? 0 : warp;
    const int workers = solo ? (int)min((long long)ctas * W, total)
                             : (int)min((long long)ctas, max((total + C::kMinTiles - 1) / C::kMinTiles, units));
    const int me = solo ? part * W + warp : part;
    if (me >= workers) return;  // no warp of a CTA that joins, or this warp for itself
    const Shares sh{quotient(span, workers), span - quotient(span, workers) * workers};
    const int share = (int)(sh.start(me + 1) - sh.start(me));
    Unit u0;
    {
      // the unit in which the share starts: the last thread that counted from at or before there,
      // then by whole sequences
      const long long x = sh.start(me);
      auto place = [&](long long packed) { return ((packed & kLow) + (packed >> 40) * kUnitCost) * hkv; };
      int of = 0;
      for (int bit = 1 << (31 - __clz(C::kThreads)); bit; bit >>= 1)
        if (of + bit < C::kThreads && place(sh_.ahead[of + bit]) <= x) of += bit;
      const int per_thread = (a.batch + C::kThreads - 1) / C::kThreads;
      long long at = place(sh_.ahead[of]), group0 = kScored ? sh_.groups_ahead[of] * hkv : 0;
      Unit u{0, 0, 0, 0, 0, of * per_thread, 0};
      for (;; ++u.b) {
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
      u0 = u;
    }
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
    int pid = max(pu.base, 0) + offset;     // its number
    int pages = 0, page_at = 32;            // pages of the unit's next tiles, one to a lane, and the next one's
    bool more = in_share(pu);
    const int log2 = a.index.page_log2;
    auto fetch_pages = [&] {  // a tile ahead
      bool moved = page_at == 32;
      while (more && pid >= tiles_end(pu)) {
        next_unit(pu);
        pid = pu.base + offset;
        more = in_share(pu);
        moved = true;
      }
      if (!more || !moved) return;
      page_at = 0;
      const int t = (pid - pu.base + lane * step) * kTile;
      if (t < pu.len)
        pages = __ldcg(a.index.block_table + (long long)pu.b * a.index.pages_per_seq + ((pu.start + t) >> log2));
    };
    auto fetch_tile = [&](int stage) {
      if (more) {
        const uint32_t st = smem_addr(ring) + stage * C::kStageBytes + copy_at;
        const int pos = pu.start + (pid - pu.base) * kTile;
        int page = __shfl_sync(0xffffffffu, pages, page_at++);
        if ((unsigned)page >= (unsigned)a.index.num_pages) {
          if (lane == 0) atomicOr(a.status, kDevBadPage);
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
        pid += step;
        fetch_pages();
      }
      cp_async_commit();
    };
    fetch_pages();
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

      for (int id = max(u.base, 0) + offset; id < end; id += step) {
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
        for (int n = 0; n < NG; ++n) {
          // while all scores were -inf they weigh nothing: -inf - -inf would be NaN
          const float r0 = R[n][0] == -INFINITY ? 0.f : R[n][0], r1 = R[n][1] == -INFINITY ? 0.f : R[n][1];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float p0 = ex2_ftz(s[n][2 * i] - r0), p1 = ex2_ftz(s[n][2 * i + 1] - r1);
            l[n][0] += p0;
            l[n][1] += p1;
            const uint32_t hi = pack2_rn(p0, p1);
            pf[n][i] = transpose8x8(hi);
            pr[n][i] = transpose8x8(pack2_rn(p0 - bf16lo(hi), p1 - bf16hi(hi)));
          }
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

      // ---- the unit's end: sums go through the stage that held the warp's last tile ----
      const int idle = (stage == 0 ? C::kStages : stage) - 1;
      float* const sums = reinterpret_cast<float*>(ring + idle * C::kStageBytes);
      const long long at0 = sh.start(me) + u.base;
      const int index = u.b * hkv + u.kvh, slot = index + me;
      if ((solo ? lane : threadIdx.x) == 0 && u.base >= 0)  // the unit starts here
        a.units[index] = UnitParts{slot, sh.cta(at0 + u.tiles - 1) - me + 1};
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], off);
          if (g == 0) sh_.ml[warp][n * 8 + 2 * t4 + c] = make_float2(R[n][c], l[n][c]);
        }
      if (solo) {
        __syncwarp();
        if (lane < G) a.part_ml[(long long)slot * G + lane] = sh_.ml[warp][lane];
#pragma unroll
        for (int n = 0; n < NG; ++n) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < KS; ++i) {
              sums[(2 * t4 + c) * C::kPitch + 16 * i + g] = o[n][i][c];
              sums[(2 * t4 + c) * C::kPitch + 16 * i + g + 8] = o[n][i][2 + c];
            }
          __syncwarp();
          for (int item = lane; item < min(8, G - 8 * n) * (D / 4); item += 32) {
            const int hl = item / (D / 4), d = item % (D / 4) * 4;
            *reinterpret_cast<float4*>(a.part_acc + ((long long)slot * G + 8 * n + hl) * D + d) =
                *reinterpret_cast<const float4*>(sums + hl * C::kPitch + d);
          }
          __syncwarp();
        }
        continue;
      }
      // the warps join
      if (lane == 0) sh_.idle[warp] = warp * C::kWarpBytes + idle * C::kStageBytes;
      sync();
#pragma unroll
      for (int n = 0; n < NG; ++n) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float top = -INFINITY;
#pragma unroll
          for (int w = 0; w < W; ++w) top = fmaxf(top, sh_.ml[w][n * 8 + 2 * t4 + c].x);
          const float f = R[n][c] == top ? 1.f : ex2_ftz(R[n][c] - top);
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            sums[(2 * t4 + c) * C::kPitch + 16 * i + g] = o[n][i][c] * f;
            sums[(2 * t4 + c) * C::kPitch + 16 * i + g + 8] = o[n][i][2 + c] * f;
          }
        }
        sync();
        const int heads = min(8, G - 8 * n);
        for (int item = threadIdx.x; item < heads * (D / 4); item += C::kThreads) {
          const int hl = item / (D / 4), d = item % (D / 4) * 4, h = 8 * n + hl;
          float top = -INFINITY, L = 0.f;
#pragma unroll
          for (int w = 0; w < W; ++w) top = fmaxf(top, sh_.ml[w][h].x);
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < W; ++w) {
            const float2 ml = sh_.ml[w][h];
            L = fmaf(ml.y, ml.x == top ? 1.f : ex2_ftz(ml.x - top), L);
            const float4 y = *reinterpret_cast<const float4*>(
                reinterpret_cast<const float*>(smem + sh_.idle[w]) + hl * C::kPitch + d);
            x.x += y.x;
            x.y += y.y;
            x.z += y.z;
            x.w += y.w;
          }
          *reinterpret_cast<float4*>(a.part_acc + ((long long)slot * G + h) * D + d) = x;
          if (d == 0) a.part_ml[(long long)slot * G + h] = make_float2(top, L);
        }
        sync();  // the idle stages may be filled again
      }
    }
    cp_async_wait<0>();
  }
};

}  // namespace paged
}  // namespace lara
