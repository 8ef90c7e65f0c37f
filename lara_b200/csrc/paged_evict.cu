// Eviction from the paged bf16 cache by gathered attention weight (lara_kv_evict,
// declared in include/lara_b200.h).
//
// Of the n slots of a (sequence, kv head), its unit, `keep` stay: the first
// `first`, the last `last`, and the heaviest of the rest, ties to the lowest
// slot.  Kept slots from `keep` on ("movers") go, in order, into the slots
// before it that are given up ("holes"), in order: no slot is both read and
// written, so all rows move at once, in place, and a step that gives up one
// slot of each kv head moves one row.
//
// Two launches.  The first finds the border weight by three radix passes (11,
// 11 and 10 bits, the most significant first, weights as ordered integers) with
// a cluster of CTAs to a unit where a unit is long and units are few, then lists
// holes and movers in order by ballots and scans.  The second moves the rows,
// shared out equally over the GPU; where a unit has few, its CTA moves them in the
// first.  The bytes are 8 per slot and 8 D per row moved, in rows of 2 D bytes in
// random order.  Measured (8 kv heads, head_dim 128), one state replayed in a graph
// and, in brackets, inputs that change from pass to pass: 32 x 8192 slots cut to 2048
// 111 us (113), of which the moves take 87 (5.2 TB/s, 0.79 of the copy rate; 64 KB in
// flight per SM in place of 96 cost 5 us) and the selection 23; 524288 slots cut to
// 65536 176 us (180; 95 and 76); 16 x 2049 cut by one 9.9 us (9.9).  The selection is
// bound by latency: barriers, scans, and instructions that run once and are not in the
// cache.  The host, which does not know the lengths, chooses by the table's width, so a
// table that is wider than its sequences costs time: the last case takes 9.9 us from
// tables of 2112 slots, 19 of 4096 (two launches), 22 of 8192 to 32768, 42 of 131072
// (clusters).
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <mutex>
#include <set>
#include <utility>

#include "paged.cuh"

namespace cg = cooperative_groups;

namespace lara {

using namespace paged;

namespace {

constexpr int kBins = 2048;
constexpr int kRows = 2;             // rows of 128 slots that a warp has in flight
constexpr int kShortSlice = 8192;    // slots that a CTA selects from alone, all of them in shared memory
// Clusters grow while a CTA has more slots than kSlice and there are fewer CTAs than SMs (8 units of
// 8192 slots 23.2 us, 28.5 without; of 65536 31, 67; from 2048 slots on 16 x 2112 slots 24.0 for
// 10.8, from 8192 on 8 units of 8192 28.5), and while it has more than kLongSlice whatever the units
// (512 units of 32768 slots 239 us, 307 in clusters from 8192 on).
constexpr int kMaxCluster = 16, kSlice = 4096, kLongSlice = 32768;
constexpr int kMostEntries = 2048;   // of the block table in shared memory
// Dynamic shared memory: three small or two large CTAs to an SM; of slices of up to
// kMostSlots (2^24 slots to a sequence), whose bits alone are more, one.
constexpr int kShortSmem = 56 * 1024, kLongSmem = 92 * 1024, kMostSmem = 200 * 1024;
constexpr long long kMostSlots = 1ll << 24;
// Rows up to which a unit's CTA moves them itself, with an SM of its own and without.  128 units of
// 2304 slots cut by 256 12.7 us, 20.6 in two launches, by 512 20.0 against 24.4; 512 units cut by 128
// 31.0 against 33.8, by 256 54 against 50.
constexpr int kFewMoves = 512, kFewMovesShared = 128;
constexpr int kMoveThreads = 192;
constexpr int kMoveSmem = kMoveThreads / 32 * 2 * 32 * 512;

// A slot of a unit, and the pool's row that it is; kBadRow on a bad page.
struct __align__(8) Listed {
  int slot;
  uint32_t row;
};
constexpr uint32_t kBadRow = 0xffffffffu;

struct Args {
  uint16_t* k;
  uint16_t* v;
  const float* w_in;
  float* w_out;
  PoolIndex index;
  const int32_t* lens;
  int32_t* new_lens;  // or null
  int32_t* sources;   // [units][keep], or null
  int batch, head_dim, keep, first, last;
  int* status;
  int* counts;        // [units] rows to move
  Listed* holes;      // [units][keep]
  Listed* movers;     // [units][keep]
};

// Weights as integers of the same order: negative ones flipped, -0 as 0, NaN on top.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return x == x ? u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u) : 0xfffffffeu;
}

__device__ __forceinline__ int slots_of(const Args& a, int b, int* raw = nullptr) {
  const int n = __ldcg(a.lens + b);
  if (raw) *raw = n;
  return (int)min((long long)max(n, 0), a.index.capacity());
}

// Exclusive prefix of one number per thread over the block, and the sum of all.
template <int kWarpsHere, typename T>
__device__ __forceinline__ T block_prefix(T x, T* s_scan, T& all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  T incl = x;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += y;
  }
  __syncthreads();
  if (lane == 31) s_scan[warp] = incl;
  __syncthreads();
  T w = lane < kWarpsHere ? s_scan[lane] : T(0);
#pragma unroll
  for (int off = 1; off < kWarpsHere; off <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, w, off);
    if (lane >= off) w += y;
  }
  all = __shfl_sync(0xffffffffu, w, kWarpsHere - 1);
  return incl - x + (warp ? __shfl_sync(0xffffffffu, w, warp - 1) : T(0));
}

// What shared memory holds of a CTA's slice: which slots stay (a bit each), the
// keys of the first slots of each warp's run, the first entries of the table; each
// a multiple of four words.
struct SliceRoom {
  int words, run_keys, entries;
};

// kLong: clusters of CTAs, and slices that shared memory need not hold; without it, one CTA to a
// unit, and all of that left out, since code that runs once waits mostly for its own instructions.
// kMoves: no unit has more than kFewMoves rows to move, and its CTA moves them itself.
template <int kThreads, int kCtas, bool kLong, bool kMoves>
__global__ void __launch_bounds__(kThreads, kCtas) select_kernel(const __grid_constant__ Args a, const SliceRoom room) {
  constexpr int kWarps = kThreads / 32;
  constexpr uint32_t kFull = 0xffffffffu;
  extern __shared__ uint32_t s_kept[];
  uint32_t* const s_keys = s_kept + room.words;
  int* const s_entry = reinterpret_cast<int*>(s_keys + room.run_keys * kWarps);
  __shared__ uint32_t s_hist[2][kBins];  // of even and odd lanes: fewer of a warp meet in a bin
  __shared__ int s_scan[kWarps];
  __shared__ int s_totals[3];  // this CTA's, read by the cluster: ties, holes, movers
  __shared__ uint32_t s_pick[3];
  __shared__ __align__(16) float s_zero[4];
  __shared__ Listed s_listed[2][kMoves ? kFewMoves : 1];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = kLong ? cluster.block_rank() : 0, size = kLong ? cluster.num_blocks() : 1;
  const int unit = blockIdx.x / size, hkv = a.index.n_kv_heads, b = unit / hkv, h = unit % hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  allow_dependent_launch();
  for (int i = threadIdx.x; i < 2 * kBins; i += kThreads) s_hist[0][i] = 0;
  if (threadIdx.x < 4) s_zero[threadIdx.x] = 0.f;
  grid_dependency_wait();

  int raw;
  const int n = slots_of(a, b, &raw);
  int32_t* const src = a.sources ? a.sources + (long long)unit * a.keep : nullptr;
  if (rank == 0 && threadIdx.x == 0) {
    if (raw != n) atomicOr(a.status, kDevBadLength);
    if (h == 0 && a.new_lens) a.new_lens[b] = min(n, a.keep);
  }
  const bool copies = a.w_in != a.w_out;
  // this CTA's slots [lo, hi), and of them the warp's, 128 at a time
  const int per = ((n + size - 1) / size + 127) / 128 * 128;
  const int lo = min(n, rank * per), hi = min(n, lo + per);
  const int run = ((hi - lo + kWarps - 1) / kWarps + 127) / 128 * 128;
  const int r_lo = min(hi, lo + warp * run), r_hi = min(hi, r_lo + run);
  // where the rows of a page of this kv head start, in pages of one head; -1: a bad page
  const int32_t* const table = a.index.block_table + (long long)b * a.index.pages_per_seq;
  const int log2 = a.index.page_log2, entry0 = lo >> log2;
  auto look_up = [&](int entry) {
    const int page = __ldg(table + entry);
    return (unsigned)page < (unsigned)a.index.num_pages ? (long long)page * hkv + h : -1ll;
  };
  const int entries = hi > lo ? min(room.entries, ((hi - 1) >> log2) - entry0 + 1) : 0;
  for (int i = threadIdx.x; i < entries; i += kThreads) s_entry[i] = (int)look_up(entry0 + i);
  __syncthreads();
  auto row_of = [&](int t) {
    const int i = (t >> log2) - entry0;
    const long long e = !kLong || i < entries ? s_entry[i] : look_up(entry0 + i);
    return e < 0 ? -1 : (e << log2) + (t & ((1 << log2) - 1));
  };
  if (n <= a.keep) {
    if (!kMoves && rank == 0 && threadIdx.x == 0) a.counts[unit] = 0;
    for (int t = lo + threadIdx.x; t < hi; t += kThreads) {
      const long long r = row_of(t);
      if (r < 0)
        atomicOr(a.status, kDevBadPage);
      else if (copies)
        a.w_out[r] = a.w_in[r];
    }
    if (src)
      for (int t = rank * kThreads + threadIdx.x; t < a.keep; t += size * kThreads) src[t] = t < n ? t : -1;
    return;
  }

  // ---- the slots' keys (a bad page's weigh nothing) and the first pass over them, four slots
  // to a lane.  Where weights are written apart, those before `keep` are copied here (of the
  // holes too: moved rows' weights replace those) and the ones behind cleared ----
  const int cached = r_lo + room.run_keys;  // weights of the run's slots before this one are kept
  float* const run_w = reinterpret_cast<float*>(s_keys) + warp * room.run_keys - r_lo;
  auto ordered4 = [](const float4& w) {
    return make_uint4(ordered(w.x), ordered(w.y), ordered(w.z), ordered(w.w));
  };
  // Of slots t .. t + 3 of the warp's run, which only this lane asks for.  One load, wherever it
  // goes, so that those of several rows are in flight at once.
  auto keys = [&](int t) {
    const float* from = run_w + t;
    if (kLong && t >= cached) {
      const long long r = t < r_hi ? row_of(t) : -1;
      from = r < 0 ? s_zero : a.w_in + r;
    }
    return ordered4(*reinterpret_cast<const float4*>(from));
  };
  const int p_lo = a.first, p_hi = n - a.last;  // slots that nothing protects; of them `free_` stay
  const int m_lo = max(r_lo, p_lo), m_hi = min(r_hi, p_hi), m_count = max(0, m_hi - m_lo);
  const int free_ = a.keep - a.first - a.last;
  auto count = [&](int t, const uint4& x, uint32_t border, uint32_t mask, int shift, int bins) {
    const uint32_t v[4] = {x.x, x.y, x.z, x.w};
    uint32_t* const hist = s_hist[lane & 1];
    if (t >= m_lo && t + 3 < m_hi) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((v[j] & mask) == border) atomicAdd(hist + ((v[j] >> shift) & (bins - 1)), 1u);
    } else {
#pragma unroll 1
      for (int j = 0; j < 4; ++j)
        if ((unsigned)(t + j - m_lo) < (unsigned)m_count && (v[j] & mask) == border)
          atomicAdd(hist + ((v[j] >> shift) & (bins - 1)), 1u);
    }
  };
  {
    bool bad = false;
#pragma unroll 1
    for (int t0 = r_lo + 4 * lane; t0 < r_hi; t0 += 128 * kRows) {
      long long row[kRows];
      float4 w[kRows];
#pragma unroll
      for (int j = 0; j < kRows; ++j) {  // no branch but the loads': all are in flight at once
        const int t = t0 + 128 * j;
        row[j] = t < r_hi ? row_of(t) : -1;
        w[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row[j] >= 0) w[j] = __ldcg(reinterpret_cast<const float4*>(a.w_in + row[j]));
        bad |= t < r_hi && row[j] < 0;
      }
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const int t = t0 + 128 * j;
        if (t >= r_hi) break;
        const uint4 x = ordered4(w[j]);
        if (!kLong || t < cached) *reinterpret_cast<float4*>(run_w + t) = w[j];
        count(t, x, 0, 0, 21, kBins);
        if (copies && row[j] >= 0) {
          if (t + 3 < n && (t + 3 < a.keep || t >= a.keep)) {
            *reinterpret_cast<float4*>(a.w_out + row[j]) = t < a.keep ? w[j] : make_float4(0.f, 0.f, 0.f, 0.f);
          } else {
            const float v[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (t + i < n) a.w_out[row[j] + i] = t + i < a.keep ? v[i] : 0.f;
          }
        }
      }
    }
    if (bad) atomicOr(a.status, kDevBadPage);
  }

  // ---- the border: 11 bits a pass, the most significant first ----
  uint32_t border = 0, mask = 0;
  int want = free_, ties = free_;  // of the slots that begin as the border does: that stay, that there are
  for (int pass = 0; pass < 3 && free_ > 0; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
    if (pass > 0) {
#pragma unroll 1
      for (int t = r_lo + 4 * lane; t < m_hi; t += 128) count(t, keys(t), border, mask, shift, bins);
    }
    if (kLong && size > 1) {
      cluster.sync();
      // each CTA adds up its share of the bins and hands the sums to all, in the place of those
      // that it alone reads
      const int part = (bins + size - 1) / size;
      for (int i = rank * part + threadIdx.x; i < min(bins, (rank + 1) * part); i += kThreads) {
        uint32_t sum = 0;
#pragma unroll 8
        for (int r = 0; r < size; ++r) {
          const uint32_t* const theirs = cluster.map_shared_rank(&s_hist[0][0], r);
          sum += theirs[i] + theirs[kBins + i];
        }
#pragma unroll 8
        for (int r = 0; r < size; ++r) {
          uint32_t* const theirs = cluster.map_shared_rank(&s_hist[0][0], r);
          theirs[i] = sum;
          theirs[kBins + i] = 0;
        }
      }
      cluster.sync();
    } else {
      __syncthreads();
    }
    // the bin, from the top, in which the want-th slot lies: thread i has bins top, top - 1, ..
    constexpr int kEach = (kBins + kThreads - 1) / kThreads;
    const int top = bins - 1 - threadIdx.x * kEach;
    int mine = 0, all;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (top - i >= 0) mine += s_hist[0][top - i] + s_hist[1][top - i];
    int before = block_prefix<kWarps>(mine, s_scan, all);
    if (before < want && before + mine >= want) {
      int bin = top, c = s_hist[0][bin] + s_hist[1][bin];
      while (before + c < want) {
        before += c;
        --bin;
        c = s_hist[0][bin] + s_hist[1][bin];
      }
      s_pick[0] = bin;
      s_pick[1] = want - before;
      s_pick[2] = c;
    }
    __syncthreads();
    border |= s_pick[0] << shift;
    mask |= (uint32_t)(bins - 1) << shift;
    want = s_pick[1];
    ties = s_pick[2];
    if (want == ties) break;  // all that begin so stay
    if (pass < 2) {
      for (int i = threadIdx.x; i < 2 * kBins; i += kThreads) s_hist[0][i] = 0;
      __syncthreads();
    }
  }
  const bool by_slot = want < ties;  // not all of the slots at the border stay

  // exclusive prefix over the runs of all CTAs of the cluster
  auto runs_before = [&](int x, int which, int& all) {  // x: of the warp
    int before = block_prefix<kWarps>(lane == 0 ? x : 0, s_scan, all);
    before = __shfl_sync(kFull, before, 0);
    if (kLong && size > 1) {
      if (threadIdx.x == 0) s_totals[which] = all;
      cluster.sync();
      const int theirs = lane < size ? *cluster.map_shared_rank(s_totals + which, lane) : 0;
      before += __reduce_add_sync(kFull, lane < rank ? theirs : 0);
      all = __reduce_add_sync(kFull, theirs);
    }
    return before;
  };
  int seen = 0, unused;  // slots at the border before the run
  if (by_slot) {
    int mine = 0;
#pragma unroll 1
    for (int t = r_lo + 4 * lane; t < m_hi; t += 128) {
      const uint4 x = keys(t);
      const uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) mine += t + j >= m_lo && t + j < m_hi && v[j] == border;
    }
    seen = runs_before(__reduce_add_sync(kFull, mine), 0, unused);
  }

  const uint32_t least = free_ > 0 ? border : 0xffffffffu;  // which no weight has
  // ---- which slots stay: bit `lane` of word j of a row of 128 is slot 4 lane + j ----
  uint4* const run_kept = reinterpret_cast<uint4*>(s_kept) + (r_lo - lo) / 128;
  const uint32_t lower = (1u << lane) - 1;
#pragma unroll 1
  for (int t0 = r_lo; t0 < r_hi; t0 += 128) {
    const int t = t0 + 4 * lane;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (t < r_hi) x = keys(t);
    uint32_t v[4] = {x.x, x.y, x.z, x.w};
    bool stays[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in = (unsigned)(t + j - p_lo) < (unsigned)(p_hi - p_lo);
      stays[j] = t + j < r_hi && (!in || v[j] >= least);
    }
    if (by_slot) {
      bool at[4];
      uint32_t m[4];
      int before = seen;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        at[j] = t + j >= m_lo && t + j < m_hi && v[j] == border;
        m[j] = __ballot_sync(kFull, at[j]);
        before += __popc(m[j] & lower);
        seen += __popc(m[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (at[j]) stays[j] = before++ < want;
    }
    uint32_t m[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = __ballot_sync(kFull, stays[j]);
    if (lane == 0) run_kept[(t0 - r_lo) / 128] = make_uint4(m[0], m[1], m[2], m[3]);
    if (src) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // a hole's is replaced with its row
        const int i = t0 + 32 * j + lane;
        if (i < min(r_hi, a.keep)) src[i] = i;
      }
    }
  }
  __syncwarp();
  // word j of a row from t0 on: the slots below t1
  auto below = [](int t0, int t1, int j) {
    const int k = (t1 - t0 - j + 3) >> 2;
    return k >= 32 ? kFull : k <= 0 ? 0u : (1u << k) - 1;
  };
  auto listed = [&](int t0, uint32_t hm[4], uint32_t mm[4]) {  // holes and movers
    const uint4 x = run_kept[(t0 - r_lo) / 128];
    const uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      hm[j] = ~v[j] & below(t0, min(r_hi, a.keep), j);
      mm[j] = v[j] & ~below(t0, a.keep, j);
    }
  };
  int holes = 0, movers = 0;
  for (int t0 = r_lo + 128 * lane; t0 < r_hi; t0 += 128 * 32) {
    uint32_t hm[4], mm[4];
    listed(t0, hm, mm);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      holes += __popc(hm[j]);
      movers += __popc(mm[j]);
    }
  }
  int all_holes;
  holes = runs_before(__reduce_add_sync(kFull, holes), 1, all_holes);
  movers = runs_before(__reduce_add_sync(kFull, movers), 2, unused);
  if (!kMoves && rank == 0 && threadIdx.x == 0) a.counts[unit] = all_holes;
  Listed* const hole_list = kMoves ? s_listed[0] : a.holes + (long long)unit * a.keep;
  Listed* const mover_list = kMoves ? s_listed[1] : a.movers + (long long)unit * a.keep;
#pragma unroll 1
  for (int t0 = r_lo; t0 < r_hi; t0 += 128) {
    uint32_t hm[4], mm[4];
    listed(t0, hm, mm);
    auto list = [&](const uint32_t m[4], Listed* to, int& at) {
      int here = at, all = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        here += __popc(m[j] & lower);
        all += __popc(m[j]);
      }
      if ((m[0] | m[1] | m[2] | m[3]) >> lane & 1) {
        const long long r = row_of(t0 + 4 * lane);  // of the lane's four slots' first
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (m[j] >> lane & 1) to[here++] = Listed{t0 + 4 * lane + j, r < 0 ? kBadRow : (uint32_t)r + j};
      }
      at += all;
    };
    if (hm[0] | hm[1] | hm[2] | hm[3]) list(hm, hole_list, holes);
    if (mm[0] | mm[1] | mm[2] | mm[3]) list(mm, mover_list, movers);
    if (!copies && t0 + 128 > a.keep) {  // in place: weights of the slots behind that nothing moves out of
      const int t = t0 + 4 * lane;
      const long long r = t < r_hi && t + 3 >= a.keep ? row_of(t) : -1;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (r >= 0 && t + j >= a.keep && t + j < r_hi && !(mm[j] >> lane & 1)) a.w_out[r + j] = 0.f;
    }
  }
  if (kLong && size > 1) cluster.sync();  // s_totals may still be read
  if constexpr (kMoves) {
    __syncthreads();
    const int row_words = a.head_dim / 8;  // lanes 0-15 have K's row, 16-31 V's
    for (int i = warp; i < all_holes; i += kWarps) {
      const Listed hole = s_listed[0][i], mover = s_listed[1][i];
      if (lane == 0 && src) src[hole.slot] = mover.slot;
      if (hole.row == kBadRow || mover.row == kBadRow) {  // flagged before
        if (lane == 0 && mover.row != kBadRow) a.w_out[mover.row] = 0.f;
        continue;
      }
      uint4* const rows = reinterpret_cast<uint4*>(lane < 16 ? a.k : a.v) + (lane & 15);
      if ((lane & 15) < row_words)
        rows[(long long)hole.row * row_words] = __ldcg(rows + (long long)mover.row * row_words);
      if (lane == 0) {
        a.w_out[hole.row] = __ldcg(a.w_in + mover.row);
        a.w_out[mover.row] = 0.f;
      }
    }
  }
}

// Rows of all units, laid end to end; each CTA takes an equal run.  A warp copies 32
// pairs of rows (K and V) at a time through shared memory, the loads of one lot under
// way while the one before is stored: two lots of 16 KB for each of six warps keep
// about 96 KB of an SM's loads in flight, which registers had no room for.
template <int D>
__global__ void __launch_bounds__(kMoveThreads, 1) move_kernel(const __grid_constant__ Args a) {
  constexpr int kWarpsHere = kMoveThreads / 32;
  constexpr int kLanes = D / 8;               // lanes of a row
  constexpr int kAtOnce = 32 / (2 * kLanes);  // pairs of rows in one access
  constexpr int kAccesses = 32 / kAtOnce;     // of 32 pairs
  extern __shared__ uint4 s_rows[];           // [warps][2][kAccesses][32]
  __shared__ long long s_sum[kWarpsHere];
  __shared__ int s_unit;
  __shared__ long long s_at;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hkv = a.index.n_kv_heads, units = a.batch * hkv;

  allow_dependent_launch();
  grid_dependency_wait();

  const int each = (units + kMoveThreads - 1) / kMoveThreads;
  const int u_lo = min(units, (int)threadIdx.x * each), u_hi = min(units, u_lo + each);
  long long mine = 0;
  for (int u = u_lo; u < u_hi; ++u) mine += __ldcg(a.counts + u);
  long long total;
  long long before = block_prefix<kWarpsHere>(mine, s_sum, total);
  const long long per = (total + gridDim.x - 1) / gridDim.x;
  const long long lo = min(total, blockIdx.x * per), hi = min(total, lo + per);
  if (lo >= hi) return;
  if (lo >= before && lo < before + mine) {
    int u = u_lo;
    while (lo >= before + __ldcg(a.counts + u)) before += __ldcg(a.counts + u++);
    s_unit = u;
    s_at = before;
  }
  __syncthreads();
  uint4* const buffer = s_rows + warp * (2 * kAccesses * 32) + lane;
  uint16_t* const pages = lane & kLanes ? a.v : a.k;
  const int sub = lane / (2 * kLanes), chunk = lane % kLanes;
  // the lot whose loads are under way: where its rows go
  uint32_t to = kBadRow;
  int lot = 0;
  auto store = [&] {  // of the lot before the last one
    const uint4* const from = buffer + (lot & 1) * (kAccesses * 32);
#pragma unroll 8
    for (int j = 0; j < kAccesses; ++j) {
      const uint32_t d = __shfl_sync(0xffffffffu, to, j * kAtOnce + sub);
      if (d != kBadRow) reinterpret_cast<uint4*>(pages + (long long)d * D)[chunk] = from[j * 32];
    }
  };
  long long at = s_at;
  for (int u = s_unit; u < units && at < hi; ++u) {
    const int count = __ldcg(a.counts + u);
    const int i_lo = (int)(max(lo, at) - at), i_hi = (int)(min(hi, at + count) - at);
    const long long list = (long long)u * a.keep;
    auto listed = [&](const Listed* from, int i) {
      Listed x{0, kBadRow};
      if (i < i_hi) *reinterpret_cast<int2*>(&x) = __ldcg(reinterpret_cast<const int2*>(from + list + i));
      return x;
    };
    Listed hole = listed(a.holes, i_lo + warp * 32 + lane), mover = listed(a.movers, i_lo + warp * 32 + lane);
    for (int i0 = i_lo + warp * 32; i0 < i_hi; i0 += kWarpsHere * 32) {
      const int next = i0 + kWarpsHere * 32 + lane;
      const bool moves = hole.row != kBadRow && mover.row != kBadRow;  // else flagged where weights were read
      float w = 0.f;
      if (moves) w = __ldcg(a.w_in + mover.row);
      if (a.sources && i0 + lane < i_hi) a.sources[list + hole.slot] = mover.slot;
      const Listed next_hole = listed(a.holes, next), next_mover = listed(a.movers, next);
      const uint32_t from = moves ? mover.row : kBadRow;
      const uint32_t into = smem_addr(buffer + (lot & 1) * (kAccesses * 32));
#pragma unroll 8
      for (int j = 0; j < kAccesses; ++j) {
        const uint32_t f = __shfl_sync(0xffffffffu, from, j * kAtOnce + sub);
        if (f != kBadRow)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(into + j * 512),
                       "l"(reinterpret_cast<const uint4*>(pages + (long long)f * D) + chunk)
                       : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      ++lot;
      asm volatile("cp.async.wait_group 1;" ::: "memory");  // a lane reads what it copied itself
      store();
      to = moves ? hole.row : kBadRow;
      if (moves) a.w_out[to] = w;
      if (mover.row != kBadRow) a.w_out[mover.row] = 0.f;
      hole = next_hole;
      mover = next_mover;
    }
    at += count;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  ++lot;
  store();
}

struct Layout {
  size_t counts_off, holes_off, movers_off, total;
};

Layout layout(int batch, int n_kv_heads, int keep) {
  const size_t units = (size_t)batch * n_kv_heads;
  Layout w;
  w.counts_off = kStatusBytes;
  w.holes_off = w.counts_off + up256(units * sizeof(int));
  w.movers_off = w.holes_off + up256(units * keep * sizeof(Listed));
  w.total = w.movers_off + up256(units * keep * sizeof(Listed));
  return w;
}

// A kernel's shared memory (and clusters above eight), once per kernel and device.
cudaError_t opt_in(const void* fn, int smem, bool clusters) {
  static std::mutex mu;
  static std::set<std::pair<const void*, int>> done;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  if (done.count({fn, dev})) return cudaSuccess;
  e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess && clusters) e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) done.insert({fn, dev});
  return e;
}

cudaError_t launch(const Args& a, cudaStream_t stream) {
  const int units = a.batch * a.index.n_kv_heads, sms = device_sm_count();
  const long long cap = a.index.capacity();
  int size = 1;
  while (size < kMaxCluster && (cap / size > kLongSlice || (cap / size > kSlice && (long long)units * size < sms)))
    size *= 2;
  const bool long_ = size > 1 || cap > kShortSlice;
  const long long most = std::min<long long>(a.keep, std::max(0ll, cap - a.keep));  // rows of a unit to move
  const bool moves = !long_ && most <= (units <= sms ? kFewMoves : kFewMovesShared);
  // With an SM to itself a CTA has 1024 threads: 128 units cut by one slot 9.9 us, 14.0 with 512.
  const bool alone = moves && units <= sms;
  const void* const fn = long_   ? reinterpret_cast<const void*>(&select_kernel<512, 2, true, false>)
                         : alone ? reinterpret_cast<const void*>(&select_kernel<1024, 1, false, true>)
                         : moves ? reinterpret_cast<const void*>(&select_kernel<512, 3, false, true>)
                                 : reinterpret_cast<const void*>(&select_kernel<512, 3, false, false>);
  const int threads = alone ? 1024 : 512, most_smem = long_ ? kLongSmem : kShortSmem;
  // per slice: the bits, then the table, then as many keys as there is room for
  const long long run = ((cap + size - 1) / size + 4 * threads - 1) / (4 * threads) * 128, slice = run * (threads / 32);
  SliceRoom room;
  room.words = (int)(slice / 32);
  room.entries = (int)std::min<long long>(kMostEntries, slice / (1 << a.index.page_log2) + 4) / 4 * 4;
  const int left = std::max(0, most_smem / 4 - room.words - room.entries) / (4 * threads) * 128;
  room.run_keys = (int)std::min<long long>(run, left);
  const size_t smem = 4 * ((size_t)room.words + room.entries + (size_t)room.run_keys * (threads / 32));
  cudaError_t e = opt_in(fn, kMostSmem, true);
  if (e != cudaSuccess) return e;
  Args args = a;
  void* p[] = {&args, &room};
  e = launch_with_pdl(fn, dim3((unsigned)units * size), dim3(threads), p, smem, stream, size);
  if (e != cudaSuccess) return e;
  if (moves || most == 0) return cudaSuccess;
  // no more CTAs than rows can move, 32 to a CTA
  const int blocks = (int)std::min<long long>(sms, (units * most + 31) / 32);
  const void* mv = a.head_dim == 128 ? reinterpret_cast<const void*>(&move_kernel<128>)
                                     : reinterpret_cast<const void*>(&move_kernel<64>);
  const int move_smem = kMoveSmem * a.head_dim / 128;
  e = opt_in(mv, move_smem, false);
  if (e != cudaSuccess) return e;
  return launch_with_pdl(mv, dim3((unsigned)blocks), dim3(kMoveThreads), p, move_smem, stream);
}

}  // namespace

}  // namespace lara

using namespace lara;

extern "C" size_t lara_kv_evict_workspace_bytes(int batch, int n_kv_heads, int keep) {
  if (batch < 1 || n_kv_heads < 1 || keep < 1) return 0;
  return layout(batch, n_kv_heads, keep).total;
}

extern "C" int lara_kv_evict(uint16_t* k_pages, uint16_t* v_pages, const float* weights, float* weights_out,
                             const int32_t* block_table, const int32_t* seq_lens, int32_t* new_lens, int32_t* sources,
                             int batch, int n_kv_heads, int head_dim, int page_size, int pages_per_seq, int num_pages,
                             int keep, int first, int last, void* workspace, size_t workspace_bytes, void* stream) {
  LARA_NVTX("lara_kv_evict");
  Args a{};
  if (const int rc = check_paged_pool(k_pages, v_pages, block_table, n_kv_heads, head_dim, page_size, pages_per_seq,
                                      num_pages, batch, &a.index))
    return rc;
  if (keep < 1 || first < 0 || last < 0 || first > keep || last > keep - first)
    return set_last_error(LARA_ERR_BAD_CFG, "keep must be positive and at least first + last");
  if (batch == 0) return LARA_OK;
  if ((long long)batch * n_kv_heads > 0x7fffffffll / kMaxCluster)
    return set_last_error(LARA_ERR_BAD_CFG, "batch * n_kv_heads must be below 2^27");
  if (!weights || !weights_out || !seq_lens || !workspace) return set_last_error(LARA_ERR_STREAM_DEST, "null pointer");
  if (!aligned(seq_lens, 4) || !aligned(new_lens, 4) || !aligned(sources, 4) || !aligned(workspace, 256))
    return set_last_error(LARA_ERR_STREAM_DEST, "lengths and sources must be 4-byte aligned, the workspace 256-byte");
  if (a.index.capacity() > kMostSlots)
    return set_last_error(LARA_ERR_UNSUPPORTED, "eviction from sequences of at most 2^24 slots");
  if ((long long)num_pages * n_kv_heads * page_size >= (long long)kBadRow ||
      (long long)num_pages * n_kv_heads > 0x7fffffffll)
    return set_last_error(LARA_ERR_BAD_CFG, "pools of less than 2^32 - 1 rows, 2^31 pages of one head");
  // CTAs of a cluster read lengths and tables at different times, and have to agree on them
  const size_t lens_bytes = (size_t)batch * 4, table_bytes = lens_bytes * pages_per_seq,
               sources_bytes = lens_bytes * n_kv_heads * keep;
  auto apart = [](const void* x, size_t x_bytes, const void* y, size_t y_bytes) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(y);
    return !x || !y || a >= b + y_bytes || b >= a + x_bytes;
  };
  if (!apart(new_lens, lens_bytes, seq_lens, lens_bytes))
    return set_last_error(LARA_ERR_STREAM_DEST, "new_lens must lie apart from seq_lens");
  if (!apart(new_lens, lens_bytes, block_table, table_bytes) ||
      !apart(sources, sources_bytes, block_table, table_bytes) ||
      !apart(sources, sources_bytes, seq_lens, lens_bytes) || !apart(sources, sources_bytes, new_lens, lens_bytes))
    return set_last_error(LARA_ERR_STREAM_DEST,
                          "new_lens and sources must lie apart from each other, from block_table and seq_lens");
  if (const int rc = check_weights(weights, weights_out, n_kv_heads, page_size, num_pages)) return rc;
  const Layout w = layout(batch, n_kv_heads, keep);
  if (workspace_bytes < w.total) return set_last_error(LARA_ERR_RESULT_LEN, "eviction workspace too small");
  a.k = k_pages;
  a.v = v_pages;
  a.w_in = weights;
  a.w_out = weights_out;
  a.lens = seq_lens;
  a.new_lens = new_lens;
  a.sources = sources;
  a.batch = batch;
  a.head_dim = head_dim;
  a.keep = keep;
  a.first = first;
  a.last = last;
  char* base = static_cast<char*>(workspace);
  a.status = reinterpret_cast<int*>(base);
  a.counts = reinterpret_cast<int*>(base + w.counts_off);
  a.holes = reinterpret_cast<Listed*>(base + w.holes_off);
  a.movers = reinterpret_cast<Listed*>(base + w.movers_off);
  const cudaError_t e = launch(a, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess)
    return set_last_error(LARA_ERR_CUDA, std::string("evict launch: ") + cudaGetErrorString(e));
  return LARA_OK;
}
