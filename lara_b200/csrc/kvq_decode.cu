// GQA decode over the paged 8-bit KV pool (declared in include/lara_b200.h).
//
//   o[b,h,:] = sum_t p_t v_t / sum_t p_t,  p_t = 2^(s_t - R),  s_t = scale log2(e) q.k_t
//   k_t = ks_t ck_t, v_t = vs_t cv_t       (codes c, one fp32 scale per row)
//
// Bound by HBM: every cached row is read once, 2 (D + 4) bytes per token and kv
// head, for 4 D G multiply-adds.  What a byte costs on the SM is kept far
// below the time it takes to arrive:
//
//  * Products run on the tensor cores as mma.m16n8k16 (fp16 in, fp32 out) with
//    the cache as the 16-row operand and the group's query heads as the 8
//    columns: S^T[token][head] = K q^T, then O^T[dim][head] = V^T P^T.  The
//    columns of S^T and O^T lie in the same lanes, so rescaling needs no
//    exchange, and movmatrix turns a tile of P into the second operand.  At
//    one byte per element the cache itself is the bound, and eight heads share
//    each product, so the 5th-generation path (128-row tiles, TMEM, operands
//    described per tile) has nothing to win here.
//  * Codes become fp16 in registers, exactly: int8 by setting the exponent
//    byte (0x6400 | code + 128 is 1152 + code) and one subtraction, e4m3 by
//    moving its bits into place (the value times 2^-8; any byte is finite, so
//    garbage past a sequence's end cannot reach a sum).  The order in which a
//    lane's bytes meet q, and the output dims a lane ends up with, are chosen
//    so that no byte has to be moved between lanes.
//  * ks multiplies the fp32 scores, vs the fp32 weights.  Weights are rounded
//    to fp16 (2^-11 each, below bf16's 2^-8 of the output); R follows the
//    largest s_t + log2 vs_t, so the weights that carry the sum stay in fp16's
//    normal range whatever the scales are.  R is moved only when a weight
//    would pass 2^8, and by whole powers of two, so most tiles rescale nothing.
//  * q is brought to fp16 by a power of two per head (exact within 2^-29 of
//    the head's largest value).
//
// Work is split evenly, by the kernel itself: all (sequence, kv head) units
// are laid end to end in tiles of 32 tokens, CTA c takes an equal share, and
// its warps take tiles in turn, each through its own ring of cp.async stages
// (no barrier per tile, no plan from the host, lengths stay on the device).
// Warps join at the end of a unit; a unit that several CTAs share is joined by
// the last of them to finish, in CTA order, so results do not depend on timing.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "kvq.cuh"

namespace lara {

using namespace kvq;

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 32;          // tokens per warp and stage
constexpr int kMinTiles = kWarps;  // tiles per CTA below which fewer CTAs run
constexpr size_t kStatusBytes = 256;

template <int D, int NG>
struct Cfg {
  static constexpr int kStages = D == 128 ? 3 : 4;
  static constexpr int kCtasPerSm = D == 128 ? 2 : 3;
  static constexpr int kRowsBytes = kTile * D;                     // K (or V) codes of a stage
  static constexpr int kStageBytes = 2 * kRowsBytes + 2 * kTile * 4;
  static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
  static constexpr int kMergeBytes = (kWarps - 1) * 8 * D * 4;     // one group of 8 heads at a time
  static constexpr int kSmemBytes = kRingBytes + kMergeBytes;
  static constexpr int kJoinChunk = kMergeBytes / (NG * 8 * 8);    // partial (R, l) the join stages at a time
};

struct KvqDecodeArgs {
  lara_kvq_pool pool;
  PoolIndex index;
  const uint16_t* q;
  const int32_t* lens;
  uint16_t* o;
  int batch, n_q_heads, group;
  float scale_log2;
  int* status;
  int* counters;    // [batch * Hkv], zero between launches
  float2* part_ml;  // [2 * grid][group] (R, l)
  float* part_acc;  // [2 * grid][group][D]
};

// 16 bytes from src + kSrc to dst + kDst (immediate offsets: one address pair
// serves a tile's copies).
template <int kDst, int kSrc>
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0+%2], [%1+%3], 16;" ::"r"(dst), "l"(src), "n"(kDst), "n"(kSrc)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma_f16(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float lg2_ftz(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bytes 0 and 2 (even) and bytes 1 and 3 (odd) of four codes as fp16 pairs.
template <int FMT>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& even, uint32_t& odd) {
  if constexpr (FMT == LARA_KVQ_INT8) {
    const uint32_t x = w ^ 0x80808080u;
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
    uint32_t e = __byte_perm(x, 0x64646464u, 0x4240), o = __byte_perm(x, 0x64646464u, 0x4341);
    const __half2 he = __hsub2(reinterpret_cast<__half2&>(e), bias);
    const __half2 ho = __hsub2(reinterpret_cast<__half2&>(o), bias);
    even = reinterpret_cast<const uint32_t&>(he);
    odd = reinterpret_cast<const uint32_t&>(ho);
  } else {
    // s eeee mmm -> s 0 eeee mmm 0000000: fp16 with the exponent 8 too small
    even = ((w << 7) & 0x3f803f80u) | ((w << 8) & 0x80008000u);
    odd = ((w >> 1) & 0x3f803f80u) | (w & 0x80008000u);
  }
}

// Where the 16-byte chunk c of a row lies in a stage, so that the eight lanes
// of a shared-memory phase (rows 2t of V, or two rows of K) hit distinct banks.
// Rows eight apart are laid out alike.
template <int D>
__device__ __forceinline__ uint32_t chunk_offset(int row, int c) {
  if constexpr (D == 128) return row * 128 + ((c ^ (row & 7)) << 4);
  return row * 64 + ((c ^ ((row >> 1) & 3)) << 4);
}

__device__ __forceinline__ int seq_tiles(const KvqDecodeArgs& a, int b, int* len_out = nullptr) {
  int len = __ldcg(a.lens + b);
  const long long cap = a.index.capacity();
  if (len < 0 || len > cap) {
    atomicOr(a.status, kDevBadLength);
    len = len < 0 ? 0 : (int)cap;
  }
  if (len_out) *len_out = len;
  return (len + kTile - 1) / kTile;
}

// A unit (b, kvh) in the end-to-end order of tiles; `base` is its first tile,
// counted from the CTA's own first.
struct Unit {
  int base, tiles, len, b, kvh;
  __device__ __forceinline__ void next(const KvqDecodeArgs& a) {
    base += tiles;
    if (++kvh == a.pool.n_kv_heads) {
      kvh = 0;
      do {
        ++b;
        tiles = b < a.batch ? seq_tiles(a, b, &len) : 0x3fffffff;
      } while (tiles == 0);
    }
  }
};

template <int D, int FMT, int NG>
__global__ void __launch_bounds__(kThreads, Cfg<D, NG>::kCtasPerSm)
    kvq_decode_kernel(const __grid_constant__ KvqDecodeArgs a) {
  using C = Cfg<D, NG>;
  constexpr int KS = D / 16;   // k steps of the scores = dim blocks of the output
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long s_sum[kWarps];
  __shared__ Unit s_first;
  __shared__ float2 s_ml[kWarps][NG * 8];
  __shared__ int s_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int G = a.group, hkv = a.pool.n_kv_heads;

  allow_dependent_launch();
  grid_dependency_wait();

  // ---- this CTA's share [w0, w1) of all tiles, and the unit w0 lies in ----
  const int per_thread = (a.batch + kThreads - 1) / kThreads;
  const int b_lo = min(a.batch, (int)threadIdx.x * per_thread), b_hi = min(a.batch, b_lo + per_thread);
  long long mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += seq_tiles(a, b);
  long long incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += x;
  }
  if (lane == 31) s_sum[warp] = incl;
  __syncthreads();
  long long before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
  }
  before *= hkv;
  total *= hkv;
  // sequences without tokens give zeros
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x)
    if (__ldcg(a.lens + b) <= 0)
      for (int i = threadIdx.x; i < a.n_q_heads * D / 8; i += kThreads)
        reinterpret_cast<uint4*>(a.o + (long long)b * a.n_q_heads * D)[i] = make_uint4(0, 0, 0, 0);
  const int n_ctas = (int)min((long long)gridDim.x, (total + kMinTiles - 1) / kMinTiles);
  if ((int)blockIdx.x >= n_ctas) return;
  const long long per = total / n_ctas, rem = total % n_ctas;
  auto cta_start = [&](long long c) { return c * per + min(c, rem); };
  auto cta_of = [&](long long id) {
    return (int)(id < rem * (per + 1) ? id / (per + 1) : rem + (id - rem * (per + 1)) / per);
  };
  const long long w0 = cta_start(blockIdx.x), w1 = cta_start(blockIdx.x + 1);
  if (w0 >= before && w0 < before + mine * hkv) {
    Unit u{0, 0, 0, b_lo, 0};
    u.tiles = seq_tiles(a, u.b, &u.len);
    while (w0 >= before + (long long)u.tiles * hkv) {  // by whole sequences (tiles may be 0)
      before += (long long)u.tiles * hkv;
      ++u.b;
      u.tiles = seq_tiles(a, u.b, &u.len);
    }
    u.kvh = (int)((w0 - before) / u.tiles);
    u.base = (int)(before + (long long)u.kvh * u.tiles - w0);  // at most 0
    s_first = u;
  }
  __syncthreads();
  const int share = (int)(w1 - w0);

  // ---- the warp's ring ----
  uint8_t* const ring = smem + warp * (C::kStages * C::kStageBytes);
  constexpr int kChunks = D / 16, kRowsPer = 32 / kChunks;  // a warp copies kRowsPer rows (512 bytes) at a time
  const uint32_t copy_even = chunk_offset<D>(lane / kChunks, lane % kChunks);
  const uint32_t copy_odd = chunk_offset<D>(lane / kChunks + kRowsPer, lane % kChunks) - 512;
  const uint32_t copy_scale = 2 * C::kRowsBytes + (lane & 3) * 16 + (lane < 4 ? 0 : kTile * 4);
  Unit pu = s_first;     // where the next tile to fetch lies
  int pid = warp;        // its number
  int page[2];           // its pages (one per 16 tokens), fetched a tile ahead
  const bool big_pages = a.index.page_log2 >= 5;
  auto fetch_pages = [&] {
    if (pid >= share) return;
    while (pid >= pu.base + pu.tiles) pu.next(a);
    const int pos = (pid - pu.base) * kTile;
    const int32_t* entry = a.index.block_table + (long long)pu.b * a.index.pages_per_seq + (pos >> a.index.page_log2);
    page[0] = __ldcg(entry);
    page[1] = big_pages || pos + 16 >= pu.len ? 0 : __ldcg(entry + 1);
  };
  auto fetch_half = [&](uint32_t st, int half, int pg, int pos) {
    if ((unsigned)pg >= (unsigned)a.index.num_pages) {
      atomicOr(a.status, kDevBadPage);
      pg = 0;
    }
    const long long row =
        (((long long)pg * hkv + pu.kvh) << a.index.page_log2) + (pos & ((1 << a.index.page_log2) - 1));
    const uint8_t* ks = a.pool.k_codes + row * D + lane * 16;
    const uint8_t* vs = a.pool.v_codes + row * D + lane * 16;
    const uint32_t even = st + half * (16 * D) + copy_even, odd = st + half * (16 * D) + copy_odd;
    if constexpr (D == 128) {
      cp_async16<0, 0>(even, ks);
      cp_async16<512, 512>(odd, ks);
      cp_async16<1024, 1024>(even, ks);
      cp_async16<1536, 1536>(odd, ks);
      cp_async16<C::kRowsBytes, 0>(even, vs);
      cp_async16<C::kRowsBytes + 512, 512>(odd, vs);
      cp_async16<C::kRowsBytes + 1024, 1024>(even, vs);
      cp_async16<C::kRowsBytes + 1536, 1536>(odd, vs);
    } else {
      cp_async16<0, 0>(even, ks);
      cp_async16<512, 512>(odd, ks);
      cp_async16<C::kRowsBytes, 0>(even, vs);
      cp_async16<C::kRowsBytes + 512, 512>(odd, vs);
    }
    if (lane < 8)  // 16 scales of K (lanes 0-3) and of V (lanes 4-7)
      cp_async16<0, 0>(st + half * 64 + copy_scale,
                       (lane < 4 ? a.pool.k_scales : a.pool.v_scales) + row + 4 * (lane & 3));
  };
  auto fetch_tile = [&](int stage) {
    if (pid < share) {
      const uint32_t st = smem_addr(ring) + stage * C::kStageBytes;
      const int pos = (pid - pu.base) * kTile;
      fetch_half(st, 0, page[0], pos);
      if (pos + 16 < pu.len) fetch_half(st, 1, big_pages ? page[0] : page[1], pos + 16);
      pid += kWarps;
      fetch_pages();
    }
    cp_async_commit();
  };
  fetch_pages();
#pragma unroll
  for (int s = 0; s < C::kStages - 1; ++s) fetch_tile(s);

  // lane-constant places in a stage: the K chunks of rows g (+ 8, 16, 24), the
  // V chunks of rows 2 t4 and 2 t4 + 1 (+ 8, 16, 24)
  uint32_t k_at[D / 64], v_at[2];
#pragma unroll
  for (int c = 0; c < D / 64; ++c) k_at[c] = chunk_offset<D>(g, t4 * (D / 64) + c);
#pragma unroll
  for (int r = 0; r < 2; ++r)
    v_at[r] = C::kRowsBytes + (D == 128 ? chunk_offset<D>(2 * t4 + r, g)
                                        : chunk_offset<D>(2 * t4 + r, g >> 1) + 8 * (g & 1));

  // ---- units of this CTA ----
  int stage = 0;
  int id = warp;         // next tile to work on
  Unit u = s_first;
  for (; u.base < share; u.next(a)) {
    const int end = min(share, u.base + u.tiles);
    // q of the group's heads as the 8-column operand: column g, rows in the
    // order in which codes_to_f16 hands out a lane's K bytes
    uint32_t qf[NG][KS][2];
    float2 qs[NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const int h = n * 8 + g;
      uint32_t w[D / 8];
      if (h < G) {
        const uint4* src = reinterpret_cast<const uint4*>(
            a.q + ((long long)u.b * a.n_q_heads + u.kvh * G + h) * D + t4 * (D / 4));
#pragma unroll
        for (int i = 0; i < D / 32; ++i) *reinterpret_cast<uint4*>(w + 4 * i) = __ldcg(src + i);
      } else {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) w[i] = 0;
      }
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
      m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 2));
      m = max(m & 0xffffu, m >> 16);
      // largest value to [2^14, 2^15); a NaN or infinity goes through as it is
      const int e = m >= 0x7f80u ? 0 : max((int)(m >> 7) - 127, -100) - 14;
      const float down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const __half2 lo = __floats2half2_rn(bf16lo(w[2 * j]) * down, bf16lo(w[2 * j + 1]) * down);
        const __half2 hi = __floats2half2_rn(bf16hi(w[2 * j]) * down, bf16hi(w[2 * j + 1]) * down);
        qf[n][j][0] = reinterpret_cast<const uint32_t&>(lo);
        qf[n][j][1] = reinterpret_cast<const uint32_t&>(hi);
      }
      // the score factor of heads 2 t4 and 2 t4 + 1, from the lanes that hold them
      const float f = __uint_as_float((uint32_t)(127 + e) << 23) * a.scale_log2 *
                      (FMT == LARA_KVQ_FP8_E4M3 ? 256.f : 1.f);
      qs[n].x = __shfl_sync(0xffffffffu, f, 8 * t4);
      qs[n].y = __shfl_sync(0xffffffffu, f, 8 * t4 + 4);
    }
    float R[NG][2], o[NG][KS][4];
    float2 l2[NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      R[n][0] = R[n][1] = -INFINITY;
      l2[n] = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < KS; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }

    for (; id < end; id += kWarps) {
      cp_async_wait<C::kStages - 2>();
      __syncwarp();
      fetch_tile(stage == 0 ? C::kStages - 1 : stage - 1);
      const uint8_t* st = ring + stage * C::kStageBytes;
      stage = stage + 1 == C::kStages ? 0 : stage + 1;

      // ---- scores: s2[i][n], token 8 i + g of the tile, heads 2 t4 and 2 t4 + 1 ----
      float s[2][NG][4];
      uint32_t k[4][D / 16];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          *reinterpret_cast<uint4*>(k[i] + 4 * c) = *reinterpret_cast<const uint4*>(st + k_at[c] + i * 8 * D);
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int n = 0; n < NG; ++n) s[mb][n][0] = s[mb][n][1] = s[mb][n][2] = s[mb][n][3] = 0.f;
#pragma unroll
      for (int j = 0; j < KS; ++j)
#pragma unroll
        for (int mb = 0; mb < 2; ++mb) {
          uint32_t a0, a1, a2, a3;
          codes_to_f16<FMT>(k[2 * mb][j], a0, a2);
          codes_to_f16<FMT>(k[2 * mb + 1][j], a1, a3);
#pragma unroll
          for (int n = 0; n < NG; ++n) mma_f16(s[mb][n], a0, a1, a2, a3, qf[n][j][0], qf[n][j][1]);
        }
      float2 s2[4][NG];
      float vsc[4], lw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float ks = *reinterpret_cast<const float*>(st + 2 * C::kRowsBytes + (8 * i + g) * 4);
        vsc[i] = *reinterpret_cast<const float*>(st + 2 * C::kRowsBytes + (kTile + 8 * i + g) * 4);
        lw[i] = fmaxf(lg2_ftz(vsc[i]), -100.f);
#pragma unroll
        for (int n = 0; n < NG; ++n)
          s2[i][n] = mul2(mul2(make_float2(s[i / 2][n][2 * (i & 1)], s[i / 2][n][2 * (i & 1) + 1]), qs[n]),
                          make_float2(ks, ks));
      }
      const int valid = u.len - (id - u.base) * kTile;
      if (valid < kTile) {  // the sequence's last tile: nothing past its end counts, whatever lies there
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (8 * i + g >= valid) {
            vsc[i] = 0.f;
            lw[i] = -100.f;
#pragma unroll
            for (int n = 0; n < NG; ++n) s2[i][n] = make_float2(-INFINITY, -INFINITY);
          }
      }

      // ---- move R where a weight would pass 2^8 ----
      bool over = false;
      float2 top[NG];
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float2 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = add2(s2[i][n], make_float2(lw[i], lw[i]));
        top[n].x = fmaxf(fmaxf(x[0].x, x[1].x), fmaxf(x[2].x, x[3].x));
        top[n].y = fmaxf(fmaxf(x[0].y, x[1].y), fmaxf(x[2].y, x[3].y));
        over |= top[n].x > R[n][0] + 8.f || top[n].y > R[n][1] + 8.f;
      }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float m = c ? top[n].y : top[n].x;
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
            if (m > R[n][c] + 8.f) {
              const float to = ceilf(m), f = ex2_ftz(R[n][c] - to);
              R[n][c] = to;
              (c ? l2[n].y : l2[n].x) *= f;
#pragma unroll
              for (int i = 0; i < KS; ++i) {
                o[n][i][c] *= f;
                o[n][i][2 + c] *= f;
              }
            }
          }
      }

      // ---- weights, as the second operand: tokens 2 t4, +1 and + 8 of column g ----
      uint32_t pf[4][NG];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          float2 p = add2(s2[i][n], make_float2(-R[n][0], -R[n][1]));
          p.x = ex2_ftz(p.x);
          p.y = ex2_ftz(p.y);
          l2[n] = add2(l2[n], p);
          const float2 wv = mul2(p, make_float2(vsc[i], vsc[i]));
          const __half2 w = __floats2half2_rn(wv.x, wv.y);
          pf[i][n] = transpose8x8(reinterpret_cast<const uint32_t&>(w));
        }

      // ---- O^T += V^T P^T: this lane's dims are D / 8 g .. of four tokens ----
#pragma unroll
      for (int mb = 0; mb < 2; ++mb) {
        uint32_t v[4][D / 32];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint8_t* at = st + v_at[r & 1] + (16 * mb + 8 * (r >> 1)) * D;
          if constexpr (D == 128) *reinterpret_cast<uint4*>(v[r]) = *reinterpret_cast<const uint4*>(at);
          else *reinterpret_cast<uint2*>(v[r]) = *reinterpret_cast<const uint2*>(at);
        }
#pragma unroll
        for (int w = 0; w < D / 32; ++w)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const uint32_t sel = hf ? 0x7632 : 0x5410;
            uint32_t a0, a1, a2, a3;
            codes_to_f16<FMT>(__byte_perm(v[0][w], v[1][w], sel), a0, a1);
            codes_to_f16<FMT>(__byte_perm(v[2][w], v[3][w], sel), a2, a3);
#pragma unroll
            for (int n = 0; n < NG; ++n) mma_f16(o[n][2 * w + hf], a0, a1, a2, a3, pf[2 * mb][n], pf[2 * mb + 1][n]);
          }
      }
    }
    float l[NG][2];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      l[n][0] = l2[n].x;
      l[n][1] = l2[n].y;
    }

    // ---- join the warps: R and l first, then the scaled sums ----
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], off);
        if (g == 0) s_ml[warp][n * 8 + 2 * t4 + c] = make_float2(R[n][c], l[n][c]);
      }
    __syncthreads();
    float4* merge = reinterpret_cast<float4*>(smem + C::kRingBytes);
    const bool whole = u.base >= 0 && u.base + u.tiles <= share;
    const int slot = 2 * (int)blockIdx.x + (u.base > 0 ? 1 : 0);
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      float L[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_ml[w][n * 8 + 2 * t4 + c].x);
        L[c] = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float2 ml = s_ml[w][n * 8 + 2 * t4 + c];
          L[c] = fmaf(ml.y, ml.x == top ? 1.f : ex2_ftz(ml.x - top), L[c]);
        }
        const float f = R[n][c] == top ? 1.f : ex2_ftz(R[n][c] - top);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          o[n][i][c] *= f;
          o[n][i][2 + c] *= f;
        }
        R[n][c] = top;
      }
      if (n > 0) __syncthreads();  // warp 0 has read the first eight heads
      if (warp > 0)
#pragma unroll
        for (int i = 0; i < KS; ++i)
          merge[((warp - 1) * KS + i) * 32 + lane] = make_float4(o[n][i][0], o[n][i][1], o[n][i][2], o[n][i][3]);
      __syncthreads();
      if (warp == 0) {
#pragma unroll
        for (int w = 0; w < kWarps - 1; ++w)
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            const float4 x = merge[(w * KS + i) * 32 + lane];
            o[n][i][0] += x.x;
            o[n][i][1] += x.y;
            o[n][i][2] += x.z;
            o[n][i][3] += x.w;
          }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int h = n * 8 + 2 * t4 + c;
          if (h >= G) continue;
          if (whole) {
            const float inv = (FMT == LARA_KVQ_FP8_E4M3 ? 256.f : 1.f) / L[c];
            uint16_t* dst = a.o + ((long long)u.b * a.n_q_heads + u.kvh * G + h) * D + g * (D / 8);
#pragma unroll
            for (int i = 0; i < KS; i += 4)
              *reinterpret_cast<uint4*>(dst + 2 * i) =
                  make_uint4(pack2_rn(o[n][i][c] * inv, o[n][i][2 + c] * inv),
                             pack2_rn(o[n][i + 1][c] * inv, o[n][i + 1][2 + c] * inv),
                             pack2_rn(o[n][i + 2][c] * inv, o[n][i + 2][2 + c] * inv),
                             pack2_rn(o[n][i + 3][c] * inv, o[n][i + 3][2 + c] * inv));
          } else {
            float* dst = a.part_acc + ((long long)slot * G + h) * D + g * (D / 8);
#pragma unroll
            for (int i = 0; i < KS; i += 2)
              *reinterpret_cast<float4*>(dst + 2 * i) =
                  make_float4(o[n][i][c], o[n][i][2 + c], o[n][i + 1][c], o[n][i + 1][2 + c]);
            if (g == 0) a.part_ml[(long long)slot * G + h] = make_float2(R[n][c], L[c]);
          }
        }
      }
    }
    if (whole) continue;

    // ---- a unit of several CTAs: the last one joins the partial results ----
    const long long first_tile = w0 + u.base;
    const int c_first = cta_of(first_tile), c_last = cta_of(first_tile + u.tiles - 1), parts = c_last - c_first + 1;
    if (warp == 0) {
      __threadfence();
      __syncwarp();
      if (lane == 0) {
        int* ctr = a.counters + (long long)u.b * hkv + u.kvh;
        const int last = atomicAdd(ctr, 1) == parts - 1;
        if (last) *ctr = 0;
        s_flag = last;
      }
    }
    __syncthreads();
    if (s_flag) {
      __threadfence();
      // thread -> four dims of a head, items G * D / 4; every (R, l) of a
      // chunk of parts goes through shared memory
      float2* ml = reinterpret_cast<float2*>(merge);
      constexpr int kItemsMax = NG * 8 * D / 4;
      constexpr int kPer = (kItemsMax + kThreads - 1) / kThreads;
      float4 acc[kPer];
      float top[kPer], L[kPer];
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        top[k] = -INFINITY;
        L[k] = 0.f;
      }
      auto slot_of = [&](int c) { return 2 * c + (first_tile > cta_start(c) ? 1 : 0); };
      for (int p0 = 0; p0 < parts; p0 += C::kJoinChunk) {
        const int np = min(C::kJoinChunk, parts - p0);
        __syncthreads();
        for (int i = threadIdx.x; i < np * G; i += kThreads)
          ml[i] = __ldcg(a.part_ml + (long long)slot_of(c_first + p0 + i / G) * G + i % G);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
          const int item = threadIdx.x + k * kThreads;
          if (item >= G * D / 4) continue;
          const int h = item / (D / 4), d = item % (D / 4);
          float m = top[k];
          for (int i = 0; i < np; ++i) m = fmaxf(m, ml[i * G + h].x);
          const float f = top[k] == m ? 1.f : ex2_ftz(top[k] - m);
          top[k] = m;
          L[k] *= f;
          acc[k].x *= f;
          acc[k].y *= f;
          acc[k].z *= f;
          acc[k].w *= f;
#pragma unroll 8
          for (int i = 0; i < np; ++i) {
            const float4 x = __ldcg(reinterpret_cast<const float4*>(
                                        a.part_acc + ((long long)slot_of(c_first + p0 + i) * G + h) * D) + d);
            const float2 r = ml[i * G + h];
            const float w = r.x == m ? 1.f : ex2_ftz(r.x - m);
            L[k] = fmaf(r.y, w, L[k]);
            acc[k].x = fmaf(x.x, w, acc[k].x);
            acc[k].y = fmaf(x.y, w, acc[k].y);
            acc[k].z = fmaf(x.z, w, acc[k].z);
            acc[k].w = fmaf(x.w, w, acc[k].w);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const int item = threadIdx.x + k * kThreads;
        if (item >= G * D / 4) continue;
        const int h = item / (D / 4), d = item % (D / 4);
        const float inv = (FMT == LARA_KVQ_FP8_E4M3 ? 256.f : 1.f) / L[k];
        *reinterpret_cast<uint2*>(a.o + ((long long)u.b * a.n_q_heads + u.kvh * G + h) * D + 4 * d) =
            make_uint2(pack2_rn(acc[k].x * inv, acc[k].y * inv), pack2_rn(acc[k].z * inv, acc[k].w * inv));
      }
    }
    __syncthreads();  // s_flag and the merge area are free again
  }
  cp_async_wait<0>();
}

// Workspace: status word | partial results (two slots per CTA) | counters.
struct Layout {
  size_t ml_off, acc_off, counters_off, total;
};

template <int D, int NG>
int max_ctas() {
  return device_sm_count() * Cfg<D, NG>::kCtasPerSm;
}

int max_ctas(int head_dim) { return head_dim == 128 ? max_ctas<128, 1>() : max_ctas<64, 1>(); }

Layout layout(int batch, int group, int n_kv_heads, int head_dim) {
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  const size_t slots = 2 * (size_t)max_ctas(head_dim);
  Layout w;
  w.ml_off = kStatusBytes;
  w.acc_off = w.ml_off + up(slots * group * sizeof(float2));
  w.counters_off = w.acc_off + up(slots * group * head_dim * sizeof(float));
  w.total = w.counters_off + up((size_t)batch * n_kv_heads * sizeof(int));
  return w;
}

template <int D, int FMT, int NG>
cudaError_t launch(const KvqDecodeArgs& a, cudaStream_t stream) {
  using C = Cfg<D, NG>;
  const void* fn = reinterpret_cast<const void*>(&kvq_decode_kernel<D, FMT, NG>);
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
  // no more CTAs than tiles of a full cache could feed
  const long long tiles = (long long)a.batch * a.pool.n_kv_heads * ((a.index.capacity() + kTile - 1) / kTile);
  const long long ctas = std::min<long long>(max_ctas<D, NG>(), (tiles + kMinTiles - 1) / kMinTiles);
  KvqDecodeArgs args = a;
  void* p[] = {&args};
  return launch_with_pdl(fn, dim3((unsigned)ctas), dim3(kThreads), p, C::kSmemBytes, stream);
}

}  // namespace

}  // namespace lara

using namespace lara;

extern "C" size_t lara_kvq_decode_workspace_bytes(int batch, int n_q_heads, int n_kv_heads, int head_dim) {
  if (batch < 1 || n_q_heads < 1 || n_kv_heads < 1 || head_dim < 1) return 0;
  return layout(batch, (n_q_heads + n_kv_heads - 1) / n_kv_heads, n_kv_heads, head_dim).total;
}

extern "C" int lara_gqa_decode_kvq(const uint16_t* q, const lara_kvq_pool* pool, const int32_t* block_table,
                                   int pages_per_seq, const int32_t* seq_lens, uint16_t* o, int batch, int n_q_heads,
                                   float scale, void* workspace, size_t workspace_bytes, void* stream) {
  LARA_NVTX("lara_gqa_decode_kvq");
  KvqDecodeArgs a{};
  if (const int rc = check_pool(pool, block_table, pages_per_seq, batch, &a.index)) return rc;
  if (batch < 0 || batch > 65535 || n_q_heads < 1 || n_q_heads % pool->n_kv_heads)
    return set_last_error(LARA_ERR_BAD_CFG, "batch must be at most 65535, n_q_heads a multiple of n_kv_heads");
  if (n_q_heads / pool->n_kv_heads > 16)
    return set_last_error(LARA_ERR_UNSUPPORTED, "groups of at most 16 query heads per kv head");
  if (!(scale > 0.f) || !std::isfinite(scale))
    return set_last_error(LARA_ERR_BAD_CFG, "scale must be positive and finite");
  if (batch == 0) return LARA_OK;
  if (!q || !seq_lens || !o || !workspace) return set_last_error(LARA_ERR_STREAM_DEST, "null pointer");
  if (!aligned(q, 16) || !aligned(o, 16) || !aligned(seq_lens, 4) || !aligned(workspace, 256))
    return set_last_error(LARA_ERR_STREAM_DEST, "q and o must be 16-byte aligned, the workspace 256-byte");
  a.group = n_q_heads / pool->n_kv_heads;
  const Layout w = layout(batch, a.group, pool->n_kv_heads, pool->head_dim);
  if (workspace_bytes < w.total) return set_last_error(LARA_ERR_RESULT_LEN, "decode workspace too small");
  a.pool = *pool;
  a.q = q;
  a.lens = seq_lens;
  a.o = o;
  a.batch = batch;
  a.n_q_heads = n_q_heads;
  a.scale_log2 = scale * 1.4426950408889634f;
  char* base = static_cast<char*>(workspace);
  a.status = reinterpret_cast<int*>(base);
  a.part_ml = reinterpret_cast<float2*>(base + w.ml_off);
  a.part_acc = reinterpret_cast<float*>(base + w.acc_off);
  a.counters = reinterpret_cast<int*>(base + w.counters_off);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaErrorInvalidValue;
#define LARA_CASE(d, f)                                  \
  if (pool->head_dim == d && pool->format == f)          \
    e = a.group <= 8 ? launch<d, f, 1>(a, st) : launch<d, f, 2>(a, st);
  LARA_CASE(128, LARA_KVQ_INT8) LARA_CASE(128, LARA_KVQ_FP8_E4M3)
  LARA_CASE(64, LARA_KVQ_INT8) LARA_CASE(64, LARA_KVQ_FP8_E4M3)
#undef LARA_CASE
  if (e != cudaSuccess)
    return set_last_error(LARA_ERR_CUDA, std::string("kvq decode launch: ") + cudaGetErrorString(e));
  return LARA_OK;
}
