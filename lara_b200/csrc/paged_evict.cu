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
// shared out equally over the GPU.  Bound by HBM: 8 bytes of weight per slot,
// 8 D bytes per row moved.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "paged.cuh"

namespace cg = cooperative_groups;

namespace lara {

using namespace paged;

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kKeysCached = 32768;  // keys of a CTA's slice kept in shared memory
constexpr int kMaxCluster = 8;
constexpr int kMoveThreads = 256;

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
  int slice_cached;   // keys of a slice that shared memory has room for
  int* status;
  int* counts;        // [units] rows to move
  int* holes;         // [units][keep]
  int* movers;        // [units][keep]
};

// Weights as integers of the same order: negative ones flipped, -0 as 0, NaN on top.
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int slots_of(const Args& a, int b, int* raw = nullptr) {
  const int n = __ldcg(a.lens + b);
  if (raw) *raw = n;
  return (int)min((long long)max(n, 0), a.index.capacity());
}

__global__ void __launch_bounds__(kThreads) select_kernel(const __grid_constant__ Args a) {
  extern __shared__ uint32_t s_keys[];
  __shared__ uint32_t s_hist[kBins];
  __shared__ uint32_t s_all[kBins];
  __shared__ int s_scan[kWarps + 1];
  __shared__ int s_totals[3];  // this CTA's, read by the cluster: ties, holes, movers
  __shared__ uint32_t s_pick[2];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), size = cluster.num_blocks();
  const int unit = blockIdx.x / size, hkv = a.index.n_kv_heads, b = unit / hkv, h = unit % hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  allow_dependent_launch();
  grid_dependency_wait();

  int raw;
  const int n = slots_of(a, b, &raw);
  int32_t* const src = a.sources ? a.sources + (long long)unit * a.keep : nullptr;
  if (rank == 0 && threadIdx.x == 0) {
    if (raw != n) atomicOr(a.status, kDevBadLength);
    if (h == 0 && a.new_lens) a.new_lens[b] = min(n, a.keep);
  }
  const bool copies = a.w_in != a.w_out;
  // this CTA's slots [lo, hi)
  const int per = ((n + size - 1) / size + 31) / 32 * 32;
  const int lo = min(n, rank * per), hi = min(n, lo + per);
  auto row_of = [&](int t) { return a.index.row(b, h, t, a.status); };
  if (n <= a.keep) {
    if (rank == 0 && threadIdx.x == 0) a.counts[unit] = 0;
    if (copies)
      for (int t = lo + threadIdx.x; t < hi; t += kThreads) {
        const long long r = row_of(t);
        if (r >= 0) a.w_out[r] = a.w_in[r];
      }
    if (src)
      for (int t = rank * kThreads + threadIdx.x; t < a.keep; t += size * kThreads) src[t] = t < n ? t : -1;
    return;
  }

  auto load_key = [&](int t) {
    const long long r = row_of(t);
    return ordered(r < 0 ? 0.f : __ldcg(a.w_in + r));
  };
  const bool cached = hi - lo <= a.slice_cached;
  if (cached)
    for (int t = lo + threadIdx.x; t < hi; t += kThreads) s_keys[t - lo] = load_key(t);
  auto key = [&](int t) { return cached ? s_keys[t - lo] : load_key(t); };
  // of the slots that nothing protects, `free_` stay
  const int m_lo = max(lo, a.first), m_hi = min(hi, n - a.last);
  const int free_ = a.keep - a.first - a.last;
  uint32_t border = 0xffffffffu;
  int room = 0, ties = 0;  // of the slots at the border: that stay, that there are
  if (free_ > 0) {
    uint32_t prefix = 0, mask = 0;
    int want = free_;
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11, bins = 1 << bits;
      for (int i = threadIdx.x; i < bins; i += kThreads) s_hist[i] = 0;
      __syncthreads();
      for (int t = m_lo + threadIdx.x; t < m_hi; t += kThreads) {
        const uint32_t x = key(t);
        if ((x & mask) == prefix) atomicAdd(&s_hist[(x >> shift) & (bins - 1)], 1u);
      }
      cluster.sync();
      if (size > 1) {
        for (int i = threadIdx.x; i < bins; i += kThreads) {
          uint32_t sum = 0;
          for (int r = 0; r < size; ++r) sum += cluster.map_shared_rank(s_hist, r)[i];
          s_all[i] = sum;
        }
        cluster.sync();
      }
      const uint32_t* const hist = size > 1 ? s_all : s_hist;
      // the bin, from the top, in which the want-th slot lies: thread i has bins [top - 4 i - 3, top - 4 i]
      const int each = bins / kThreads;
      int mine = 0;
      for (int i = 0; i < each; ++i) mine += hist[bins - 1 - threadIdx.x * each - i];
      int incl = mine;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += y;
      }
      if (lane == 31) s_scan[warp] = incl;
      __syncthreads();
      int before = incl - mine;
      for (int w = 0; w < warp; ++w) before += s_scan[w];
      if (before < want && before + mine >= want) {
        int bin = bins - 1 - threadIdx.x * each, c = hist[bin];
        while (before + c < want) {
          before += c;
          c = hist[--bin];
        }
        s_pick[0] = bin;
        s_pick[1] = want - before;
        s_totals[0] = c;
      }
      __syncthreads();
      prefix |= s_pick[0] << shift;
      mask |= (uint32_t)(bins - 1) << shift;
      want = s_pick[1];
      ties = s_totals[0];
      __syncthreads();
    }
    border = prefix;
    room = want;
  } else {
    __syncthreads();
  }

  // ---- each warp takes a run of the slice, 32 slots at a time, in order ----
  const int run = ((hi - lo + kWarps - 1) / kWarps + 31) / 32 * 32;
  const int r_lo = min(hi, lo + warp * run), r_hi = min(hi, r_lo + run);
  // exclusive prefix over the runs of all CTAs of the cluster
  auto runs_before = [&](int x, int which, int& all) {
    __syncthreads();
    if (lane == 0) s_scan[warp] = x;
    __syncthreads();
    int before = 0, sum = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s_scan[w];
      sum += s_scan[w];
    }
    all = sum;
    if (size > 1) {
      if (threadIdx.x == 0) s_totals[which] = sum;
      cluster.sync();
      all = 0;
      for (int r = 0; r < size; ++r) {
        const int y = *cluster.map_shared_rank(s_totals + which, r);
        if (r < rank) before += y;
        all += y;
      }
      cluster.sync();
    }
    return before;
  };
  auto is_free = [&](int t) { return t >= a.first && t < n - a.last; };
  int tie = 0, unused;
  const bool by_slot = free_ > 0 && room < ties;  // not all of the slots at the border stay
  if (by_slot) {
    int mine = 0;
    for (int t0 = r_lo; t0 < r_hi; t0 += 32) {
      const int t = t0 + lane;
      mine += __popc(__ballot_sync(0xffffffffu, t < r_hi && is_free(t) && key(t) == border));
    }
    tie = runs_before(mine, 0, unused);
  }
  auto kept_of = [&](int t, uint32_t x, int& seen) {  // seen: slots at the border before this row of 32
    const bool at = t < r_hi && is_free(t) && x == border;
    bool kept = t < r_hi && (!is_free(t) || (free_ > 0 && (x > border || (at && !by_slot))));
    if (by_slot) {
      const uint32_t m = __ballot_sync(0xffffffffu, at);
      if (at) kept = seen + __popc(m & ((1u << lane) - 1)) < room;
      seen += __popc(m);
    }
    return kept;
  };
  int holes = 0, movers = 0, seen = tie;
  for (int t0 = r_lo; t0 < r_hi; t0 += 32) {
    const int t = t0 + lane;
    const bool kept = kept_of(t, t < r_hi ? key(t) : 0, seen);
    holes += __popc(__ballot_sync(0xffffffffu, t < r_hi && t < a.keep && !kept));
    movers += __popc(__ballot_sync(0xffffffffu, kept && t >= a.keep));
  }
  int all_holes;
  holes = runs_before(holes, 1, all_holes);
  movers = runs_before(movers, 2, unused);
  if (rank == 0 && threadIdx.x == 0) a.counts[unit] = all_holes;
  int* const hole_list = a.holes + (long long)unit * a.keep;
  int* const mover_list = a.movers + (long long)unit * a.keep;
  seen = tie;
  for (int t0 = r_lo; t0 < r_hi; t0 += 32) {
    const int t = t0 + lane;
    const bool kept = kept_of(t, t < r_hi ? key(t) : 0, seen);
    const bool hole = t < r_hi && t < a.keep && !kept, mover = kept && t >= a.keep;
    const uint32_t hm = __ballot_sync(0xffffffffu, hole), mm = __ballot_sync(0xffffffffu, mover);
    const uint32_t lower = (1u << lane) - 1;
    if (hole) hole_list[holes + __popc(hm & lower)] = t;
    if (mover) mover_list[movers + __popc(mm & lower)] = t;
    holes += __popc(hm);
    movers += __popc(mm);
    if (t < r_hi && !hole && !mover) {
      if (t < a.keep) {
        if (src) src[t] = t;
        if (copies) {
          const long long r = row_of(t);
          if (r >= 0) a.w_out[r] = a.w_in[r];
        }
      } else {
        const long long r = row_of(t);
        if (r >= 0) a.w_out[r] = 0.f;
      }
    }
  }
}

// Rows of all units, laid end to end; each warp of the grid takes an equal run.
template <int D>
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const __grid_constant__ Args a) {
  constexpr int kWarpsHere = kMoveThreads / 32;
  constexpr int kLanes = D / 8;             // lanes of a row
  constexpr int kAtOnce = 32 / (2 * kLanes);  // pairs of rows (K and V) in one access
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
  long long incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += y;
  }
  if (lane == 31) s_sum[warp] = incl;
  __syncthreads();
  long long before = incl - mine, total = 0;
  for (int w = 0; w < kWarpsHere; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
  }
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
  long long at = s_at;
  for (int u = s_unit; u < units && at < hi; ++u) {
    const int count = __ldcg(a.counts + u);
    const int b = u / hkv, h = u % hkv;
    const int i_lo = (int)(max(lo, at) - at), i_hi = (int)(min(hi, at + count) - at);
    const long long list = (long long)u * a.keep;
    for (int i0 = i_lo + warp * 32; i0 < i_hi; i0 += kWarpsHere * 32) {
      const int i = i0 + lane;
      long long to = -1, from = -1;
      if (i < i_hi) {
        const int d = __ldcg(a.holes + list + i), s = __ldcg(a.movers + list + i);
        to = a.index.row(b, h, d, nullptr);  // flagged where its weight was read
        from = a.index.row(b, h, s, nullptr);
        if (a.sources) a.sources[list + d] = s;
        if (to >= 0 && from >= 0) a.w_out[to] = a.w_in[from];
        if (from >= 0) a.w_out[from] = 0.f;
        if (from < 0) to = -1;
      }
      const int pairs = min(32, i_hi - i0);
      uint16_t* const pages = lane & kLanes ? a.v : a.k;
      const int sub = lane / (2 * kLanes), chunk = lane % kLanes;
#pragma unroll 1
      for (int p0 = 0; p0 < pairs; p0 += 8 * kAtOnce) {
        uint4 x[8];
        long long dst[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int p = p0 + j * kAtOnce + sub;
          dst[j] = __shfl_sync(0xffffffffu, to, p & 31);
          const long long f = __shfl_sync(0xffffffffu, from, p & 31);
          if (p >= pairs) dst[j] = -1;
          if (dst[j] >= 0) x[j] = __ldcg(reinterpret_cast<const uint4*>(pages + f * D) + chunk);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (dst[j] >= 0) reinterpret_cast<uint4*>(pages + dst[j] * D)[chunk] = x[j];
      }
    }
    at += count;
  }
}

struct Layout {
  size_t counts_off, holes_off, movers_off, total;
};

Layout layout(int batch, int n_kv_heads, int keep) {
  const size_t units = (size_t)batch * n_kv_heads;
  Layout w;
  w.counts_off = kStatusBytes;
  w.holes_off = w.counts_off + up256(units * sizeof(int));
  w.movers_off = w.holes_off + up256(units * keep * sizeof(int));
  w.total = w.movers_off + up256(units * keep * sizeof(int));
  return w;
}

cudaError_t launch(const Args& a, cudaStream_t stream) {
  const void* fn = reinterpret_cast<const void*>(&select_kernel);
  constexpr int kMostSmem = kKeysCached * 4;
  {
    static std::mutex mu;
    static uint64_t done = 0;  // the shared-memory opt-in is per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    std::lock_guard<std::mutex> lock(mu);
    if (dev > 63 || !(done >> dev & 1)) {
      e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem);
      if (e != cudaSuccess) return e;
      if (dev <= 63) done |= 1ull << dev;
    }
  }
  const int units = a.batch * a.index.n_kv_heads, sms = device_sm_count();
  const long long cap = a.index.capacity();
  int size = 1;
  while (size < kMaxCluster && cap / size > 4096 && (long long)units * size < sms) size *= 2;
  Args args = a;
  const long long slice = ((cap + size - 1) / size + 31) / 32 * 32;
  args.slice_cached = (int)std::min<long long>(slice, kKeysCached);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)units * size);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)args.slice_cached * 4;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* p[] = {&args};
  cudaError_t e = cudaLaunchKernelExC(&cfg, fn, p);
  if (e != cudaSuccess) return e;
  // no more CTAs than rows can move, 256 to a CTA
  const long long most = (long long)units * std::min<long long>(a.keep, std::max(0ll, cap - a.keep));
  if (most == 0) return cudaSuccess;
  const int blocks = (int)std::min<long long>(sms * 8, (most + 31) / 32);
  const void* mv = a.head_dim == 128 ? reinterpret_cast<const void*>(&move_kernel<128>)
                                     : reinterpret_cast<const void*>(&move_kernel<64>);
  return launch_with_pdl(mv, dim3((unsigned)blocks), dim3(kMoveThreads), p, 0, stream);
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
    return set_last_error(LARA_ERR_BAD_CFG, "batch * n_kv_heads must be below 2^28");
  if (!weights || !weights_out || !seq_lens || !workspace) return set_last_error(LARA_ERR_STREAM_DEST, "null pointer");
  if (!aligned(weights, 4) || !aligned(weights_out, 4) || !aligned(seq_lens, 4) || !aligned(workspace, 256))
    return set_last_error(LARA_ERR_STREAM_DEST, "the workspace must be 256-byte aligned, all else 4-byte");
  if (kvq::overlap(new_lens, seq_lens, (size_t)batch * 4))
    return set_last_error(LARA_ERR_STREAM_DEST, "new_lens must lie apart from seq_lens");
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
  a.holes = reinterpret_cast<int*>(base + w.holes_off);
  a.movers = reinterpret_cast<int*>(base + w.movers_off);
  const cudaError_t e = launch(a, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess)
    return set_last_error(LARA_ERR_CUDA, std::string("evict launch: ") + cudaGetErrorString(e));
  return LARA_OK;
}
