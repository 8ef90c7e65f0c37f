// GQA decode over the paged 8-bit KV pool (declared in include/lara_b200.h).
//
//   o[b,h,:] = sum_t p_t v_t / sum_t p_t,  p_t = 2^(s_t - R),  s_t = scale log2(e) q.k_t
//   k_t = ks_t ck_t, v_t = vs_t cv_t       (codes c, one fp32 scale per row)
//
// Bound by HBM: every cached row is read once, 2 (D + 4) bytes per token and kv
// head, for 4 D G multiply-adds.  What a byte costs on the SM is kept below the
// time it takes to arrive:
//
//  * Products run on the tensor cores as warp-wide mma with the cache as the
//    16-row operand and the group's query heads as the 8 columns:
//    S^T[token][head] = K q^T, then O^T[dim][head] = V^T P^T.  The columns of
//    both lie in the same lanes, so rescaling needs no exchange, and movmatrix
//    turns a tile of P into the second operand.  At one byte per element the
//    cache itself is the bound, and eight heads share each product, so the
//    5th-generation path (128-row tiles, TMEM) has nothing to win here.
//  * K codes become fp16 in registers, exactly (int8 by setting the exponent
//    byte, 0x6400 | code + 128 is 1152 + code, and one subtraction), and so does
//    q 2^k (exactly within 2^-29 of the head's largest).  8-bit products instead
//    were slower (measured with weights of one fp16 number): of int8 codes with q
//    in three base-256 digits, 128 query heads 109 against 101 us, one sequence of
//    300 tokens 6.7 against 6.4; of e4m3 codes with q in e4m3 digits 99 against 87.
//  * V codes become fp16 the same way, after ldmatrix has transposed the bytes.
//  * ks multiplies the fp32 scores, vs the fp32 weights.  A weight is the sum of
//    two fp16 numbers, the second what the first leaves, and what both leave is
//    2^-22 of it: one alone leaves 2^-11, which shows wherever values nearly cancel
//    in an output.  The second product costs up to eight heads 1 % (64 x 4096 tokens
//    87.9 -> 88.6 us), 16 heads, bound by the products, 12 % (100.3 -> 112.6; e4m3
//    97.0 -> 103.8).  R follows the largest s_t + log2 vs_t, so that weights keep 32
//    binary orders below the largest one whatever the scales are.  R moves only when
//    a weight would pass 2^15, and by whole powers of two, so most tiles rescale
//    nothing.
//
// Work is split by the kernel itself, so that no plan from the host depends on
// the lengths: all (sequence, kv head) units are laid end to end in tiles of 32
// tokens, CTA c takes an equal share, and its warps take tiles in turn, each
// through its own ring of cp.async stages (no barrier per tile).  Warps join at
// the end of a unit; a unit that several CTAs share is joined by the last of
// them to finish, in CTA order, so results do not depend on timing.  Short or
// few units are shared out otherwise, see below.
//
// Measured (head_dim 128, 8 kv heads, int8 where not said): 64 sequences of
// 4096 tokens 88 us, 0.97 of the copy rate of 6534 GB/s (e4m3 87 us; 64 query
// heads 91 us; 128 query heads 114 us, e4m3 104 us, bound by the products' issue
// and latency with eight warps per SM), of 8192 tokens 167 us (1.02; head_dim 64
// 93 us, 0.94, of 4096 tokens 53 us, 0.82); one of 1,048,576 tokens 317 us (1.07: it
// only reads); one of 300 tokens 6.5 us.
// About 10 us of a large call do not stream: 2 us until a CTA knows its share,
// 3 us until its first rows arrive, and at the end CTAs finish over 10 us.
// Three stages with two CTAs per SM, separate K and V slots (K fetched two
// tiles ahead) and L2 prefetch hints were no faster.
#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>

#include "kvq.cuh"

namespace lara {

using namespace kvq;

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 32;          // tokens per warp and stage
constexpr int kMinTiles = kWarps;  // tiles per CTA below which fewer CTAs run
// Units up to this long are not split while each has a CTA.  8 units of 20 tiles
// take 8.5 us, 9.6 split; of 25 tiles 10.3 against 9.6, of 32 tiles 11.2 against
// 10.7, 48 units of 32 tiles 16.1 against 12.4; with 16 heads to a unit 11.6
// against 12.3, 13.7 against 14.4, 14.9 against 14.3, 19.3 against 16.1.
constexpr int kWholeTiles = 24;
// Units up to this long, and up to four times as long as there are units per
// CTA, go to a warp each: 2400 units of 1-4 tiles 18 us, 27 by CTA, of 1-10 tiles
// 30 against 37; 512 units of 7 tiles would take 18 us against 14.
constexpr int kSoloTiles = 16;
// Units up to this long, more than CTAs, go to CTAs whole: shares end between
// units (8 query heads and 16, by head blocks).  512 units of 7 tiles 13.6 us,
// 15.2 cut, of 16 tiles 20.2 against 19.7 (800 of them 23.9 against 27.6), of 17
// 21.7 against 20.2, of 24 28.2 against 25.0; with 16 heads, of 16, 24, 25, 47 tiles
// 24.8, 33.4, 35.3, 53 against 30.5, 38.2, 39.9, 56, but 904 of 47 tiles 96 against 89.
constexpr int kUncutTiles[2] = {16, 24};
// What a unit costs beside its tiles, in tiles, where shares are measured out, for
// each block of eight heads: 2400 units of 1-47 tiles 88 us, 98 with 4, 129 with
// none; with 16 heads 142 us (8 per block), 158, 236.  Where units go to a warp:
// 2400 of 1-10 tiles 30 us, 32 with none, 31 with 4; with 16 heads 45, 59, 45.
constexpr int kUnitCost = 8, kUnitCostSolo = 2;
// Units have CTAs of their own where each can have this many on average.  48 units of
// 8000 tokens 23.2 us, 23.3 in equal shares (64 query heads 24.6 against 26.2), of 2000
// tokens 13.3 against 12.6; 56 units of 8000 tokens 27.4 either way (29.0 against 30.2),
// of 2000 tokens 14.1 against 13.2.
constexpr int kFewCtas = 8;
// Where a unit has CTAs of its own: in microseconds, a tile takes a CTA kTileUs,
// a part its join kPartUs per head and dim, and a join in two steps (of groups of
// parts, then of the groups; more than kOneJoin parts) kTwoStepsUs on top.  One
// kv head, 4 query heads, of 16384, 65536, 262144 tokens: 14, 26, 64 us with the
// parts that pay in one step, 18, 42, 51 with one for every CTA, 15, 19, 26 so in
// two steps; 16 query heads 24, 45, 82; 44, 105, 114; 25, 34, 44.
constexpr float kTileUs = 0.21f, kPartUs = 0.025f / 128.f, kTwoStepsUs = 6.f;
constexpr int kOneJoin = 64;
constexpr int kFewParts = 4;       // parts of a unit that its last CTA joins without publishing its own
constexpr int kLensCached = 1024;  // lengths kept in shared memory
constexpr size_t kStatusBytes = 256;

// Weights lie in fp16 between 2^kStart (the largest, when R is set) and 2^kHigh.
constexpr float kStart = 7.f, kHigh = 15.f;
// No scale of V counts as less than 2^kFloor when R is set, so that a term of the
// plain sum of 2^(s - R), which has no scale, is at most 2^(kHigh - kFloor): the
// sum is finite up to 2^28 tokens of zeros.  The smallest scale, 2^-107, still has
// its weights at 2^-15, 2^-10 of which fp16's last place is.  At the other end, a
// term is 0 below 2^-126: with scales of V up to 2^100 (values up to 1e32) that is
// a token 33 octaves less likely than the one that set R.
constexpr float kFloor = -85.f;

template <int D, int NG>
struct Cfg {
  static constexpr int kStages = 2;
  static constexpr int kCtasPerSm = D == 128 ? (NG == 1 ? 3 : 2) : (NG == 1 ? 4 : 3);
  static constexpr int kRowsBytes = kTile * D;                     // K (or V) codes of a stage
  static constexpr int kStageBytes = 2 * kRowsBytes + 2 * kTile * 4;
  static constexpr int kWarpBytes = kStages * kStageBytes;
  static constexpr int kSmemBytes = kWarps * kWarpBytes + 128;
  static constexpr int kPitch = D + 4;  // floats per head in the join (lanes of a store hit distinct banks)
  static_assert(kStageBytes % 128 == 0, "rows start on 128-byte boundaries");
  static_assert(8 * kPitch * 4 <= kStageBytes, "a stage holds the sums of eight heads");
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
  int* counters;        // [2 * grid], of a unit by its first slot, and
  int* group_counters;  // [2 * grid], of a group of parts; zero between launches
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

// Two 16 x 16 blocks of bytes, transposed: lanes 0-15 and 16-31 name the rows
// (tokens) of one block each; the lane gets tokens 4 t4 .. + 3 of dims g (v[0],
// v[2]) and g + 8 (v[1], v[3]).
__device__ __forceinline__ void load_transposed(uint32_t v[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ float lg2_ftz(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Sums of tokens of zeros have terms up to 2^100, at an R so low that beside rows
// of large values 2^(R - top) alone is below fp32.  l 2^d, f = 2^d, for a whole d <= 0:
__device__ __forceinline__ float scale_down(float l, float f, float d) {
  return f > 0.f ? l * f : l * 0x1p-126f * ex2_ftz(d + 126.f);
}
// and (R, l) as joins take it: what l has past 2^32 goes to R.
__device__ __forceinline__ float2 to_join(float R, float l) {
  const int e = max((int)(__float_as_uint(l) >> 23) - (127 + 32), 0);
  return make_float2(R + (float)e, l * __uint_as_float((uint32_t)(127 - e) << 23));
}

// Bytes 0, 1 (lo) and 2, 3 (hi) of four codes as fp16 pairs.
template <int FMT>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FMT == LARA_KVQ_INT8) {
    const uint32_t x = w ^ 0x80808080u;
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
    uint32_t l = __byte_perm(x, 0x64646464u, 0x4140), h = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 hl = __hsub2(reinterpret_cast<__half2&>(l), bias);
    const __half2 hh = __hsub2(reinterpret_cast<__half2&>(h), bias);
    lo = reinterpret_cast<const uint32_t&>(hl);
    hi = reinterpret_cast<const uint32_t&>(hh);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\t"
        "mov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}

// q 2^-e, below 2^15, in fp16 as the second operand, two registers per four
// dims.  m: the head's largest |q| as bf16 magnitude bits; factor() brings a
// score back.
template <int FMT, int NG>
struct Query {
  static __device__ __forceinline__ int exponent(uint32_t m) { return max((int)(m >> 7) - 127, -100) - 14; }
  static __device__ __forceinline__ float factor(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
  static __device__ __forceinline__ void split(const float x[4], uint32_t out[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      out[i] = reinterpret_cast<const uint32_t&>(h);
    }
  }
  template <int D>
  static __device__ __forceinline__ void scores(float (*s)[4], const uint32_t* a, const uint32_t* b,
                                                const uint32_t (*q)[D / 16][2]) {
#pragma unroll
    for (int n = 0; n < NG; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      uint32_t a0, a1, a2, a3;
      codes_to_f16<FMT>(a[j], a0, a2);
      codes_to_f16<FMT>(b[j], a1, a3);
#pragma unroll
      for (int n = 0; n < NG; ++n) mma_f16(s[n], a0, a1, a2, a3, q[n][j][0], q[n][j][1]);
    }
  }
};

// Where the 16-byte chunk c of a row lies in a stage, so that the rows which a
// shared-memory phase reads (two rows of K, eight of V) hit distinct banks.
// Rows eight apart are laid out alike.
template <int D>
__device__ __forceinline__ uint32_t chunk_offset(int row, int c) {
  if constexpr (D == 128) return row * 128 + ((c ^ (row & 7)) << 4);
  return row * 64 + ((c ^ ((row >> 1) & 3)) << 4);
}

__device__ __forceinline__ int tiles_of(int len) { return (len + kTile - 1) / kTile; }

// a / b, by 32-bit arithmetic where both fit.
__device__ __forceinline__ long long quotient(long long a, long long b) {
  if (((a | b) >> 31) == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}

// A unit (b, kvh); `base` is its first tile, counted from the start of the
// share that this CTA (or warp) works on.
struct Unit {
  int base, tiles, len, b, kvh;
};

// Parts of a unit are joined as o = sum_i 2^(R_i - R) o_i / sum_i 2^(R_i - R) l_i
// with R the largest R_i, i in CTA order: the same words whichever CTA does it.
__device__ __forceinline__ void join_start(float& top, float& L, float4& x) {
  top = -INFINITY;
  L = 0.f;
  x = make_float4(0.f, 0.f, 0.f, 0.f);
}
__device__ __forceinline__ void join_add(float top, float& L, float4& x, const float2& ml, const float4& y) {
  const float w = ml.x == top ? 1.f : ex2_ftz(ml.x - top);
  L = __fmaf_rn(ml.y, w, L);
  x.x = __fmaf_rn(y.x, w, x.x);
  x.y = __fmaf_rn(y.y, w, x.y);
  x.z = __fmaf_rn(y.z, w, x.z);
  x.w = __fmaf_rn(y.w, w, x.w);
}

// The published parts of one unit: slots `first` (an odd one where its CTA
// started in another unit), then one per CTA; `own` is this CTA's.
struct Join {
  int first, parts, own;
  __device__ __forceinline__ int slot(int i) const { return i == 0 ? first : (first & ~1) + 2 * i; }
};

// Joins published parts first, first + step, .. (`parts` of them) of a unit, all
// threads together, into slot `dest` or, where that is negative, the output.
// `room` bytes at `mine`, the warp's own, take as many parts at a time as they
// hold: each lane copies the 16 bytes of every sum that it adds up, so that the
// loads of a whole round are in flight at once without registers of their own
// (9 sequences of 7007 tokens, one kv head of 8 query heads: 17.5 us; with weights of
// one fp16 number 17.0, and 20.4 with eight loads at a time in registers; of 28000
// tokens, 8 kv heads of 16: 104; 101 and 107).
template <int D, int kItems>
__device__ __forceinline__ void join_published(const KvqDecodeArgs& a, const Join& j, int first, int step, int parts,
                                               int dest, long long out_row, uint8_t* mine, int room) {
  constexpr int kHeads = 128 / D;  // heads of a warp's 32 items
  const int G = a.group, lane = threadIdx.x & 31;
  const int items = (G * (D / 4) + kThreads - 1) / kThreads;  // of a thread, at most
  const int most = room / (items * (512 + 8 * kHeads));
  float2* const ml = reinterpret_cast<float2*>(mine + most * items * 512);
  const uint32_t to = smem_addr(mine) + lane * 16;
  const int h0 = threadIdx.x / (D / 4), hw = (threadIdx.x & ~31) / (D / 4), d = threadIdx.x % (D / 4) * 4;
  constexpr int kHeadStep = kThreads / (D / 4);  // from a thread's item to its next
  float4 x[kItems];
  float top[kItems], L[kItems];
#pragma unroll
  for (int k = 0; k < kItems; ++k) join_start(top[k], L[k], x[k]);
  for (int p0 = 0; p0 < parts; p0 += most) {
    const int np = min(most, parts - p0);
    for (int i = 0; i < np; ++i) {
      const long long row = (long long)j.slot(first + (p0 + i) * step) * G;
#pragma unroll
      for (int k = 0; k < kItems; ++k)
        if (h0 + k * kHeadStep < G)
          cp_async16<0, 0>(to + (i * items + k) * 512, a.part_acc + (row + h0 + k * kHeadStep) * D + d);
    }
    cp_async_commit();
    for (int i = lane; i < np * items * kHeads; i += 32) {
      const int p = i / (items * kHeads), r = i - p * (items * kHeads), h = hw + r / kHeads * kHeadStep + r % kHeads;
      if (h < G) ml[i] = __ldcg(a.part_ml + (long long)j.slot(first + (p0 + p) * step) * G + h);
    }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      if (h0 + k * kHeadStep >= G) continue;
      float m = top[k];
      for (int i = 0; i < np; ++i) m = fmaxf(m, ml[(i * items + k) * kHeads + h0 - hw].x);
      const float f = top[k] == m ? 1.f : ex2_ftz(top[k] - m);
      top[k] = m;
      L[k] *= f;
      x[k] = make_float4(x[k].x * f, x[k].y * f, x[k].z * f, x[k].w * f);
    }
    cp_async_wait<0>();
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      if (h0 + k * kHeadStep >= G) continue;
#pragma unroll 4
      for (int i = 0; i < np; ++i)
        join_add(top[k], L[k], x[k], ml[(i * items + k) * kHeads + h0 - hw],
                 *reinterpret_cast<const float4*>(mine + (i * items + k) * 512 + lane * 16));
    }
    __syncwarp();
  }
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int h = h0 + k * kHeadStep;
    if (h >= G) continue;
    if (dest < 0) {
      const float inv = 1.f / L[k];
      *reinterpret_cast<uint2*>(a.o + (out_row + h) * D + d) =
          make_uint2(pack2_rn(x[k].x * inv, x[k].y * inv), pack2_rn(x[k].z * inv, x[k].w * inv));
    } else {
      *reinterpret_cast<float4*>(a.part_acc + ((long long)dest * G + h) * D + d) = x[k];
      if (d == 0) a.part_ml[(long long)dest * G + h] = make_float2(top[k], L[k]);
    }
  }
}

// Equal shares: the first `rem` take one more.
struct Shares {
  long long per, rem;
  __device__ __forceinline__ long long start(long long c) const { return c * per + min(c, rem); }
  __device__ __forceinline__ int cta(long long tile) const {
    return (int)(tile < rem * (per + 1) ? quotient(tile, per + 1) : rem + quotient(tile - rem * (per + 1), per));
  }
};

// Few units: the first CTA of this one's unit, how many it has, this one's tiles.
struct Part {
  int first, parts, tiles;
};

__device__ __forceinline__ int load_acquire(const int* p) {
  int v;
  asm volatile("ld.acquire.gpu.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

template <int D, int FMT, int NG>
__global__ void __launch_bounds__(kThreads, Cfg<D, NG>::kCtasPerSm)
    kvq_decode_kernel(const __grid_constant__ KvqDecodeArgs a) {
  using C = Cfg<D, NG>;
  using Q = Query<FMT, NG>;
  constexpr int KS = D / 16;   // dim blocks of the output
  extern __shared__ uint8_t smem_raw[];
  __shared__ long long s_sum[kWarps];
  __shared__ int s_max[kWarps], s_some[kWarps];
  __shared__ Unit s_first[kWarps];
  __shared__ Part s_part;
  __shared__ Shares s_shares;
  __shared__ float2 s_ml[kWarps][NG * 8];
  __shared__ int s_flag, s_idle[kWarps];
  __shared__ int s_lens[kLensCached];
  // chunk_offset's rows start on 128-byte boundaries
  uint8_t* const smem = smem_raw + (-smem_addr(smem_raw) & 127);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int G = a.group, hkv = a.pool.n_kv_heads;
  const long long cap = a.index.capacity();

  allow_dependent_launch();
  grid_dependency_wait();

  // ---- this CTA's share of all tiles, and the unit in which it starts ----
  auto load_len = [&](int b) {
    const int len = __ldcg(a.lens + b);
    return (int)min((long long)max(len, 0), cap);
  };
  auto len_of = [&](int b) { return b < kLensCached ? s_lens[b] : load_len(b); };
  int gap = 0;  // units lie this far apart in the order that is shared out
  auto next_unit = [&](Unit& u) {
    u.base += u.tiles + gap;
    if (++u.kvh == hkv) {
      u.kvh = 0;
      do {
        ++u.b;
        u.len = u.b < a.batch ? len_of(u.b) : 0;
        u.tiles = u.b < a.batch ? tiles_of(u.len) : 0x3fffffff;
      } while (u.tiles == 0);
    }
  };
  const int per_thread = (a.batch + kThreads - 1) / kThreads;
  const int b_lo = min(a.batch, (int)threadIdx.x * per_thread), b_hi = min(a.batch, b_lo + per_thread);
  long long mine = 0;
  int longest = 0, some = 0;
  for (int b = b_lo; b < b_hi; ++b) {
    const int raw = __ldcg(a.lens + b);
    const int len = (int)min((long long)max(raw, 0), cap);
    if (raw != len) atomicOr(a.status, kDevBadLength);
    if (b < kLensCached) s_lens[b] = len;
    mine += tiles_of(len);
    longest = max(longest, tiles_of(len));
    some += len > 0;
  }
  // exclusive prefix of one number per thread, and the sum of all; reads and
  // writes s_sum between two barriers
  auto prefix = [&](long long x, long long& sum) {
    long long incl = x;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += y;
    }
    if (lane == 31) s_sum[warp] = incl;
    __syncthreads();
    long long ahead = incl - x;
    sum = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) ahead += s_sum[w];
      sum += s_sum[w];
    }
    return ahead;
  };
  const int mine_some = some;
  longest = __reduce_max_sync(0xffffffffu, longest);
  some = __reduce_add_sync(0xffffffffu, some);
  if (lane == 31) {
    s_max[warp] = longest;
    s_some[warp] = some;
  }
  // tiles in the low 40 bits, sequences that have some above
  long long all;
  const long long ahead = prefix(mine + ((long long)mine_some << 40), all);
  constexpr long long kLow = (1ll << 40) - 1;
  longest = some = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    longest = max(longest, s_max[w]);
    some += s_some[w];
  }
  const long long total = (all & kLow) * hkv;
  // sequences without tokens give zeros
  if (some < a.batch)
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x)
      if (len_of(b) == 0)
        for (int i = threadIdx.x; i < a.n_q_heads * D / 8; i += kThreads)
          reinterpret_cast<uint4*>(a.o + (long long)b * a.n_q_heads * D)[i] = make_uint4(0, 0, 0, 0);
  if (total == 0) return;
  // How the tiles are shared.  Short units, each with a CTA: one each.  Few
  // units: as many CTAs for a unit as it has tiles for, none with parts of two.
  // Short units, more than CTAs: whole ones to each warp (solo) or CTA (uncut).
  // Else equal shares for each CTA, across units, with a cost of its own for each
  // unit.
  const long long units = (long long)some * hkv;
  const bool one_each = longest <= kWholeTiles && (long long)a.batch * hkv <= gridDim.x;
  const bool few = !one_each && units * kFewCtas <= gridDim.x;
  const bool solo = !one_each && !few && longest <= kSoloTiles && (long long)longest * gridDim.x <= 4 * units;
  const bool uncut = !one_each && !few && !solo && longest <= kUncutTiles[NG - 1];
  const bool entire = solo || uncut;  // a share has the units that start in it
  if (!one_each && !few) gap = solo ? kUnitCostSolo : NG * kUnitCost;
  int share;
  if (one_each) {
    const int b = blockIdx.x / hkv;
    if (b >= a.batch || len_of(b) == 0) return;
    share = tiles_of(len_of(b));
    if (threadIdx.x == 0) s_first[0] = Unit{0, share, len_of(b), b, (int)blockIdx.x - b * hkv};
  } else if (few) {
    const long long ctas = max(1ll, min(gridDim.x - units, quotient(total, kMinTiles)));
    const long long per = quotient(total + ctas - 1, ctas);
    auto parts_of = [&](int b) {
      const int tiles = tiles_of(len_of(b));
      const int most = (int)quotient(tiles + per - 1, per);
      const float t = kTileUs * tiles, c = kPartUs * (G * D);
      const int one = min(min(max((int)sqrtf(t / c), 1), kOneJoin), most);
      const bool two_steps =
          most > kOneJoin && t / most + 2.f * c * sqrtf((float)most) + kTwoStepsUs < t / one + c * one;
      return two_steps ? most : one;  // none without tiles
    };
    __syncthreads();  // s_sum is free again
    mine = 0;
    for (int b = b_lo; b < b_hi; ++b) mine += parts_of(b);
    long long before = prefix(mine, all) * hkv;
    const int x = blockIdx.x;
    if (x >= all * hkv) return;
    if (x >= before && x < before + mine * hkv) {
      int b = b_lo;
      while (x >= before + (long long)parts_of(b) * hkv) before += (long long)parts_of(b++) * hkv;
      const int n = parts_of(b), at = x - (int)before, kvh = at / n, part = at - kvh * n, tiles = tiles_of(len_of(b));
      const int t0 = (int)quotient((long long)part * tiles, n), t1 = (int)quotient((long long)(part + 1) * tiles, n);
      s_first[0] = Unit{-t0, tiles, len_of(b), b, kvh};
      s_part = Part{x - part, n, t1 - t0};
    }
    __syncthreads();
    share = s_part.tiles;
  } else {
    const long long span = total + units * gap;
    const int workers = solo ? (int)gridDim.x * kWarps
                             : (int)min((long long)gridDim.x, max((total + kMinTiles - 1) / kMinTiles, units));
    const Shares sh{quotient(span, workers), span - quotient(span, workers) * workers};
    const int me = solo ? (int)blockIdx.x * kWarps + warp : (int)blockIdx.x;
    if (!solo && me >= workers) return;
    share = (int)(sh.start(me + 1) - sh.start(me));
    if (threadIdx.x == 0) s_shares = sh;
    // the unit in which each share starts: found by the thread that counted its sequence
    const long long begin = ((ahead & kLow) + (ahead >> 40) * gap) * hkv;
    const long long stop = begin + (mine + (long long)mine_some * gap) * hkv;
    for (int w = 0; w < (solo ? kWarps : 1); ++w) {
      const long long x = sh.start(solo ? (long long)blockIdx.x * kWarps + w : blockIdx.x);
      if (x < begin || x >= stop) continue;
      long long at = begin;
      Unit u{0, 0, 0, b_lo, 0};
      for (;; ++u.b) {  // by whole sequences
        u.len = len_of(u.b);
        u.tiles = tiles_of(u.len);
        const long long span_b = u.tiles ? (long long)(u.tiles + gap) * hkv : 0;
        if (x < at + span_b) break;
        at += span_b;
      }
      u.kvh = (int)quotient(x - at, u.tiles + gap);
      u.base = (int)(at + (long long)u.kvh * (u.tiles + gap) + gap - x);  // at most gap
      if (entire && u.base < gap) next_unit(u);  // it belongs to the share that it starts in
      s_first[w] = u;
    }
  }
  __syncthreads();
  const Unit u0 = s_first[solo ? warp : 0];
  const int step = solo ? 1 : kWarps, offset = solo ? 0 : warp;
  // a unit starts in this share / its tiles of this share are [max(base, 0), tiles_end)
  auto in_share = [&](const Unit& u) { return share > 0 && (entire ? u.base - gap : u.base) < share; };
  auto tiles_end = [&](const Unit& u) { return entire ? u.base + u.tiles : min(share, u.base + u.tiles); };

  // ---- the warp's ring ----
  uint8_t* const ring = smem + warp * C::kWarpBytes;
  constexpr int kChunks = D / 16, kRowsPer = 32 / kChunks;  // a warp copies kRowsPer rows (512 bytes) at a time
  const uint32_t copy_even = chunk_offset<D>(lane / kChunks, lane % kChunks);
  const uint32_t copy_odd = chunk_offset<D>(lane / kChunks + kRowsPer, lane % kChunks) - 512;
  Unit pu = u0;                           // where the next tile to fetch lies
  int pid = max(pu.base, 0) + offset;     // its number
  int page[2];                            // its pages (one per 16 tokens), fetched a tile ahead
  bool more = in_share(pu);
  const int log2 = a.index.page_log2;
  const bool big_pages = log2 >= 5;  // a tile lies in one page
  auto fetch_pages = [&] {
    while (more && pid >= tiles_end(pu)) {
      next_unit(pu);
      pid = pu.base + offset;
      more = in_share(pu);
    }
    if (!more) return;
    const int pos = (pid - pu.base) * kTile;
    const int32_t* entry = a.index.block_table + (long long)pu.b * a.index.pages_per_seq + (pos >> log2);
    page[0] = __ldcg(entry);
    page[1] = big_pages || pos + 16 >= pu.len ? 0 : __ldcg(entry + 1);
  };
  auto first_row = [&](int pg, int pos) {  // the pool's row of the unit's token `pos`
    if ((unsigned)pg >= (unsigned)a.index.num_pages) {
      atomicOr(a.status, kDevBadPage);
      pg = 0;
    }
    return (((long long)pg * hkv + pu.kvh) << log2) + (pos & ((1 << log2) - 1));
  };
  auto fetch_half = [&](uint32_t st, const uint8_t* ks, const uint8_t* vs) {
    const uint32_t even = st + copy_even, odd = st + copy_odd;
    cp_async16<0, 0>(even, ks);
    cp_async16<512, 512>(odd, ks);
    cp_async16<C::kRowsBytes, 0>(even, vs);
    cp_async16<C::kRowsBytes + 512, 512>(odd, vs);
    if constexpr (D == 128) {
      cp_async16<1024, 1024>(even, ks);
      cp_async16<1536, 1536>(odd, ks);
      cp_async16<C::kRowsBytes + 1024, 1024>(even, vs);
      cp_async16<C::kRowsBytes + 1536, 1536>(odd, vs);
    }
  };
  auto fetch_tile = [&](int stage) {
    if (more) {
      const uint32_t st = smem_addr(ring) + stage * C::kStageBytes;
      const int pos = (pid - pu.base) * kTile;
      const bool two = pos + 16 < pu.len;
      const long long row0 = first_row(page[0], pos);
      const uint8_t* ks = a.pool.k_codes + row0 * D + lane * 16;
      const uint8_t* vs = a.pool.v_codes + row0 * D + lane * 16;
      fetch_half(st, ks, vs);
      // scales: 16 bytes per lane, K by lanes 0-7 and V by lanes 8-15
      const float* sc = (lane < 8 ? a.pool.k_scales : a.pool.v_scales) + row0 + 4 * (lane & 7);
      if (two) {
        if (!big_pages) {
          const long long row1 = first_row(page[1], pos + 16);
          ks = a.pool.k_codes + row1 * D + lane * 16 - 16 * D;
          vs = a.pool.v_codes + row1 * D + lane * 16 - 16 * D;
          if (lane & 4) sc += row1 - row0 - 16;
        }
        fetch_half(st + 16 * D, ks + 16 * D, vs + 16 * D);
      }
      if (lane < 16 && (two || !(lane & 4))) cp_async16<2 * C::kRowsBytes, 0>(st + lane * 16, sc);
      pid += step;
      fetch_pages();
    }
    cp_async_commit();
  };
  fetch_pages();
#pragma unroll
  for (int s = 0; s < C::kStages - 1; ++s) fetch_tile(s);

  // Row g of a block of 16 scores is token 4 (g / 2) + g % 2 (row g + 8: two
  // on), so that the weights of a lane's column end up in ldmatrix's order.
  const int tok_at = 4 * (g >> 1) + (g & 1);
  uint32_t k_at[2][D / 64];  // the lane's chunks of those two rows
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int c = 0; c < D / 64; ++c) k_at[r][c] = chunk_offset<D>(tok_at + 2 * r, t4 * (D / 64) + c);
  const uint32_t v_at = C::kRowsBytes + chunk_offset<D>(lane & 15, lane >> 4);

  // ---- units of this CTA ----
  int stage = 0;
  Unit u = u0;
  for (; in_share(u); next_unit(u)) {
    const int end = tiles_end(u);
    // q of the group's heads as the 8-column operand: column g, this lane's
    // dims D / 4 t4 .., which are those of its K chunks
    uint32_t qf[NG][D / 16][2];
    float2 qs[NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const int h = n * 8 + g;
      uint32_t w[D / 8];
#pragma unroll
      for (int i = 0; i < D / 8; ++i) w[i] = 0;
      if (h < G) {
        const uint4* src = reinterpret_cast<const uint4*>(
            a.q + ((long long)u.b * a.n_q_heads + u.kvh * G + h) * D + t4 * (D / 4));
#pragma unroll
        for (int i = 0; i < D / 32; ++i) *reinterpret_cast<uint4*>(w + 4 * i) = __ldcg(src + i);
      }
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
      m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 2));
      m = max(m & 0xffffu, m >> 16);
      const bool finite = m < 0x7f80u;
      const int e = Q::exponent(finite ? m : 0);
      const float down = finite ? __uint_as_float((uint32_t)(127 - e) << 23) : 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        const float x[4] = {bf16lo(w[2 * j]) * down, bf16hi(w[2 * j]) * down, bf16lo(w[2 * j + 1]) * down,
                            bf16hi(w[2 * j + 1]) * down};
        Q::split(x, qf[n][j]);
      }
      // the score factor of heads 2 t4 and 2 t4 + 1, from the lanes that hold
      // them; a NaN or an infinity in q makes its head NaN
      const float f = finite ? Q::factor(e) * a.scale_log2 : __uint_as_float(0x7fffffffu);
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

    for (int id = max(u.base, 0) + offset; id < end; id += step) {
      cp_async_wait<C::kStages - 2>();
      __syncwarp();
      fetch_tile(stage == 0 ? C::kStages - 1 : stage - 1);
      const int at = stage;
      const uint8_t* st = ring + at * C::kStageBytes;
      stage = stage + 1 == C::kStages ? 0 : stage + 1;

      // ---- scores: s2[2 mb + r][n] of token 16 mb + 2 r + tok_at, heads 2 t4 and 2 t4 + 1 ----
      float2 s2[4][NG];
#pragma unroll
      for (int mb = 0; mb < 2; ++mb) {
        uint32_t k[2][D / 16];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            *reinterpret_cast<uint4*>(k[r] + 4 * c) =
                *reinterpret_cast<const uint4*>(st + k_at[r][c] + mb * 16 * D);
        float s[NG][4];
        Q::template scores<D>(s, k[0], k[1], qf);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          s2[2 * mb][n] = make_float2(s[n][0], s[n][1]);
          s2[2 * mb + 1][n] = make_float2(s[n][2], s[n][3]);
        }
      }
      float vsc[4], lw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float* sc = reinterpret_cast<const float*>(st + 2 * C::kRowsBytes) + tok_at + 16 * (i / 2) + 2 * (i & 1);
        vsc[i] = sc[kTile];
        lw[i] = fmaxf(lg2_ftz(vsc[i]), kFloor);
#pragma unroll
        for (int n = 0; n < NG; ++n) s2[i][n] = mul2(mul2(s2[i][n], qs[n]), make_float2(sc[0], sc[0]));
      }
      const int valid = u.len - (id - u.base) * kTile;
      if (valid < kTile) {  // the sequence's last tile: nothing past its end counts, whatever lies there
        if (FMT == LARA_KVQ_FP8_E4M3) {  // e4m3 garbage may be NaN, and 0 NaN is NaN
          for (int i = valid * (D / 16) + lane; i < C::kRowsBytes / 16; i += 32)
            reinterpret_cast<uint4*>(ring + at * C::kStageBytes + C::kRowsBytes)[i] = make_uint4(0, 0, 0, 0);
          __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (tok_at + 16 * (i / 2) + 2 * (i & 1) >= valid) {
            vsc[i] = 0.f;
            lw[i] = kFloor;
#pragma unroll
            for (int n = 0; n < NG; ++n) s2[i][n] = make_float2(-INFINITY, -INFINITY);
          }
      }

      // ---- move R where a weight would pass 2^15 ----
      bool over = false;
      float2 top[NG];
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float2 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = add2(s2[i][n], make_float2(lw[i], lw[i]));
        top[n].x = fmaxf(fmaxf(x[0].x, x[1].x), fmaxf(x[2].x, x[3].x));
        top[n].y = fmaxf(fmaxf(x[0].y, x[1].y), fmaxf(x[2].y, x[3].y));
        over |= top[n].x > R[n][0] + kHigh || top[n].y > R[n][1] + kHigh;
      }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float m = c ? top[n].y : top[n].x;
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
            if (m > R[n][c] + kHigh) {
              const float to = ceilf(m) - kStart, f = ex2_ftz(R[n][c] - to);
              (c ? l2[n].y : l2[n].x) = scale_down(c ? l2[n].y : l2[n].x, f, R[n][c] - to);
              R[n][c] = to;
#pragma unroll
              for (int i = 0; i < KS; ++i) {
                o[n][i][c] *= f;
                o[n][i][2 + c] *= f;
              }
            }
          }
      }

      // ---- weights, as the second operand: tokens 4 t4 .. + 3 of column g.  What fp16
      // leaves of a weight is a second one ----
      uint32_t pf[4][NG], pr[4][NG];
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
          const float2 back = __half22float2(w);
          const __half2 rest = __floats2half2_rn(wv.x - back.x, wv.y - back.y);
          pf[i][n] = transpose8x8(reinterpret_cast<const uint32_t&>(w));
          pr[i][n] = transpose8x8(reinterpret_cast<const uint32_t&>(rest));
        }

      // ---- O^T += V^T P^T: block c holds dims 16 c + g and 16 c + g + 8 ----
      const uint32_t v_base = smem_addr(st) + v_at;
#pragma unroll
      for (int mb = 0; mb < 2; ++mb) {
#pragma unroll
        for (int c = 0; c < KS; c += 2) {
          uint32_t v[4];
          load_transposed(v, (v_base ^ (c << 4)) + mb * 16 * D);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t a0, a1, a2, a3;
            codes_to_f16<FMT>(v[2 * i], a0, a2);
            codes_to_f16<FMT>(v[2 * i + 1], a1, a3);
#pragma unroll
            for (int n = 0; n < NG; ++n) {
              mma_f16(o[n][c + i], a0, a1, a2, a3, pf[2 * mb][n], pf[2 * mb + 1][n]);
              mma_f16(o[n][c + i], a0, a1, a2, a3, pr[2 * mb][n], pr[2 * mb + 1][n]);
            }
          }
        }
      }
    }
    float l[NG][2];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      l[n][0] = l2[n].x;
      l[n][1] = l2[n].y;
    }

    // ---- the unit's end.  Sums go through the stage that held the warp's last
    // tile (its next fetch will fill it) ----
    const int idle = (stage == 0 ? C::kStages : stage) - 1;
    float* const sums = reinterpret_cast<float*>(ring + idle * C::kStageBytes);
    const long long out_row = (long long)u.b * a.n_q_heads + u.kvh * G;
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], off);
    if (solo) {  // this warp has all of it
      __syncwarp();
#pragma unroll
      for (int n = 0; n < NG; ++n) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float inv = 1.f / l[n][c];
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            sums[(2 * t4 + c) * C::kPitch + 16 * i + g] = o[n][i][c] * inv;
            sums[(2 * t4 + c) * C::kPitch + 16 * i + g + 8] = o[n][i][2 + c] * inv;
          }
        }
        __syncwarp();
        for (int item = lane; item < min(8, G - 8 * n) * (D / 4); item += 32) {
          const int hl = item / (D / 4), d = item % (D / 4) * 4;
          const float4 x = *reinterpret_cast<const float4*>(sums + hl * C::kPitch + d);
          *reinterpret_cast<uint2*>(a.o + (out_row + 8 * n + hl) * D + d) =
              make_uint2(pack2_rn(x.x, x.y), pack2_rn(x.z, x.w));
        }
        __syncwarp();
      }
      continue;
    }
    // join the warps: R and l, then the scaled sums
    if (lane == 0) s_idle[warp] = warp * C::kWarpBytes + idle * C::kStageBytes;
    const bool whole = uncut || (u.base >= 0 && u.base + u.tiles <= share);
    // a unit of several CTAs: which ones, and whether all others are done
    Join j{0, 1, 0};
    if (!whole) {
      if (few) {
        j = Join{2 * s_part.first, s_part.parts, 2 * (int)blockIdx.x};
      } else {
        const long long tile0 = s_shares.start(blockIdx.x) + u.base;
        const int c0 = s_shares.cta(tile0);
        // a CTA shares at most two units: the one it starts in has slot 0, a later one slot 1
        j = Join{2 * c0 + (tile0 > s_shares.start(c0) ? 1 : 0), s_shares.cta(tile0 + u.tiles - 1) - c0 + 1,
                 2 * (int)blockIdx.x + (u.base > 0 ? 1 : 0)};
      }
    }
    int* const counter = a.counters + j.first;  // no other unit's
    if (threadIdx.x == 0) {
      const bool last = j.parts > 1 && j.parts <= kFewParts && load_acquire(counter) == j.parts - 1;
      if (last) *counter = 0;
      s_flag = last;
    }
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (g == 0) s_ml[warp][n * 8 + 2 * t4 + c] = to_join(R[n][c], l[n][c]);
      }
    __syncthreads();
    const bool last_here = s_flag;
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
        if (last_here) {  // the other parts lie ready: join them here, in CTA order
          float2 ml[kFewParts];
          float4 y[kFewParts];
#pragma unroll
          for (int i = 0; i < kFewParts; ++i) {
            ml[i] = make_float2(top, L);
            y[i] = x;
            if (i < j.parts && j.slot(i) != j.own) {
              const long long at = (long long)j.slot(i) * G + h;
              ml[i] = __ldcg(a.part_ml + at);
              y[i] = __ldcg(reinterpret_cast<const float4*>(a.part_acc + at * D + d));
            }
          }
          join_start(top, L, x);
#pragma unroll
          for (int i = 0; i < kFewParts; ++i)
            if (i < j.parts) top = fmaxf(top, ml[i].x);
#pragma unroll
          for (int i = 0; i < kFewParts; ++i)
            if (i < j.parts) join_add(top, L, x, ml[i], y[i]);
        }
        if (whole || last_here) {
          const float inv = 1.f / L;
          *reinterpret_cast<uint2*>(a.o + (out_row + h) * D + d) =
              make_uint2(pack2_rn(x.x * inv, x.y * inv), pack2_rn(x.z * inv, x.w * inv));
        } else {
          *reinterpret_cast<float4*>(a.part_acc + ((long long)j.own * G + h) * D + d) = x;
          if (d == 0) a.part_ml[(long long)j.own * G + h] = make_float2(top, L);
        }
      }
      if (n + 1 < NG || whole || last_here) __syncthreads();  // the idle stages may be filled again
    }
    if (whole || last_here) continue;

    // ---- this part is published; the last CTA to do so joins them all, or,
    // of many parts, those of its group, and the last group's the groups' ----
    auto last_of = [&](int* ctr, int n) {
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        const bool last = atomicAdd(ctr, 1) == n - 1;
        if (last) *ctr = 0;
        s_flag = last;
      }
      __syncthreads();
      const bool last = s_flag;
      if (last) __threadfence();
      return last;
    };
    constexpr int kItems = (NG * 8 * D / 4 + kThreads - 1) / kThreads;
    // no copy is under way where each CTA has one part
    uint8_t* const mine = few ? ring : ring + idle * C::kStageBytes;
    const int room = few ? C::kWarpBytes : C::kStageBytes;
    if (j.parts <= kOneJoin) {
      if (last_of(counter, j.parts))
        join_published<D, kItems>(a, j, 0, 1, j.parts, -1, out_row, mine, room);
    } else {
      const int size = (int)ceilf(sqrtf((float)j.parts)), lead = (j.own / 2 - j.first / 2) / size * size;
      const int groups = (j.parts + size - 1) / size, here = min(size, j.parts - lead), dest = j.slot(lead);
      if (last_of(a.group_counters + dest, here)) {
        join_published<D, kItems>(a, j, lead, 1, here, dest, out_row, mine, room);
        if (last_of(counter, groups))
          join_published<D, kItems>(a, j, 0, size, groups, -1, out_row, mine, room);
      }
    }
    __syncthreads();  // s_flag and the idle stages are free again
  }
  cp_async_wait<0>();
}

template <int D, int NG>
int max_ctas() {
  return device_sm_count() * Cfg<D, NG>::kCtasPerSm;
}

// Workspace: status word | counters | partial results (two slots per CTA).  The
// counters lie at the same place for every batch and geometry, and no call writes
// its partial results over them, so that a workspace serves any call that it is
// large enough for.
struct Layout {
  size_t counters_off, groups_off, ml_off, acc_off, total;
};

Layout layout(int group, int head_dim) {
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  const size_t slots = 2 * (size_t)std::max(max_ctas<64, 1>(), max_ctas<128, 1>());
  Layout w;
  w.counters_off = kStatusBytes;
  w.groups_off = w.counters_off + up(slots * sizeof(int));
  w.ml_off = w.groups_off + up(slots * sizeof(int));
  w.acc_off = w.ml_off + up(slots * group * sizeof(float2));
  w.total = w.acc_off + up(slots * group * head_dim * sizeof(float));
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
  // no more CTAs than a full cache could feed, one for each unit at least
  const long long units = (long long)a.batch * a.pool.n_kv_heads;
  const long long tiles = units * ((a.index.capacity() + kTile - 1) / kTile);
  const long long ctas = std::min<long long>(max_ctas<D, NG>(), std::max(units, (tiles + kMinTiles - 1) / kMinTiles));
  KvqDecodeArgs args = a;
  void* p[] = {&args};
  return launch_with_pdl(fn, dim3((unsigned)ctas), dim3(kThreads), p, C::kSmemBytes, stream);
}

}  // namespace

}  // namespace lara

using namespace lara;

extern "C" size_t lara_kvq_decode_workspace_bytes(int batch, int n_q_heads, int n_kv_heads, int head_dim) {
  if (batch < 1 || n_q_heads < 1 || n_kv_heads < 1 || head_dim < 1) return 0;
  return layout((n_q_heads + n_kv_heads - 1) / n_kv_heads, head_dim).total;
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
  const Layout w = layout(a.group, pool->head_dim);
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
  a.group_counters = reinterpret_cast<int*>(base + w.groups_off);
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
