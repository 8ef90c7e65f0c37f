// Writing and reading the paged 8-bit KV pool (declared in include/lara_b200.h;
// the write replaces the K/V cache write of hw/rtl/mem/kv_cache_ram.sv:45-91
// for a quantised cache).
//
// Both are bound by HBM: append reads 2 D bytes of bf16 per row and writes
// D + 4, read the reverse.  D / 16 lanes hold a row, 32 bytes of bf16 each (one
// access where it is so aligned).  A warp takes as many consecutive tokens of
// one (sequence, kv head) as it has lane groups, K and V: the length, the start
// and the pages (two at most) are looked up once per warp, not once per row.
// 8192 tokens of 8 x 8 heads (head_dim 128) are read back in 63 us, 0.98 of the
// copy rate (16-byte accesses: 70 us; several rows per lane: 64-65 us), 2048 of
// 8 x 8 appended and read in 33 us (0.94; 43 us).
#include <algorithm>

#include "kvq.cuh"

namespace lara {

namespace kvq {

int check_pool(const lara_kvq_pool* pool, const void* block_table, int pages_per_seq, int batch, PoolIndex* index) {
  if (!pool) return set_last_error(LARA_ERR_STREAM_DEST, "null pool");
  if (pool->format != LARA_KVQ_INT8 && pool->format != LARA_KVQ_FP8_E4M3)
    return set_last_error(LARA_ERR_UNSUPPORTED, "unknown code format");
  if (pool->head_dim != 64 && pool->head_dim != 128)
    return set_last_error(LARA_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  const int ps = pool->page_size;
  if (ps < 16 || ps > 65536 || (ps & (ps - 1)))
    return set_last_error(LARA_ERR_BAD_CFG, "page_size must be a power of two in [16, 65536]");
  if (pool->num_pages < 1 || pool->n_kv_heads < 1 || pages_per_seq < 1 || (long long)pages_per_seq * ps > 0x7fffffffll)
    return set_last_error(LARA_ERR_BAD_CFG, "bad pool geometry");
  if (!pool->k_codes || !pool->v_codes || !pool->k_scales || !pool->v_scales || (!block_table && batch > 0))
    return set_last_error(LARA_ERR_STREAM_DEST, "null pool or block table pointer");
  if (!aligned(pool->k_codes, 16) || !aligned(pool->v_codes, 16) || !aligned(pool->k_scales, 16) ||
      !aligned(pool->v_scales, 16) || !aligned(block_table, 4))
    return set_last_error(LARA_ERR_STREAM_DEST, "pool buffers must be 16-byte aligned, the block table 4-byte");
  int lg = 0;
  while ((1 << lg) < ps) ++lg;
  index->block_table = static_cast<const int32_t*>(block_table);
  index->pages_per_seq = pages_per_seq;
  index->page_log2 = lg;
  index->num_pages = pool->num_pages;
  index->n_kv_heads = pool->n_kv_heads;
  return LARA_OK;
}

}  // namespace kvq

using namespace kvq;

namespace {

constexpr int kThreads = 128;

struct RowArgs {
  lara_kvq_pool pool;
  PoolIndex index;
  const int32_t* starts;
  const int32_t* counts;  // append: rows per sequence; read: seq_lens
  int32_t* new_lens;
  Heads<const uint16_t> k, v;
  Heads<uint16_t> ko, vo;
  int batch, n;
  uint32_t tiles;          // warps' worth of work
  FastDiv div_tiles, div_h;  // tiles per (sequence, kv head); kv heads
  int* status;
};

// A warp's tokens t0 .. t0 + kTokens - 1 of (b, h), and where their rows lie in
// the pool: row p (a position in the sequence) is base + p, on its second page
// base2 + p; a negative base is a bad page.
template <int kTokens>
struct WarpRows {
  uint32_t b, h;
  int t0, cross;
  long long start, base, base2;
  __device__ __forceinline__ bool init(const RowArgs& a) {
    const uint32_t w = blockIdx.x * (uint32_t)(kThreads / 32) + threadIdx.x / 32;  // below 2^31, unlike the thread's index
    if (w >= a.tiles) return false;
    uint32_t tile;
    const uint32_t bh = a.div_tiles.div(w, tile);
    b = a.div_h.div(bh, h);
    t0 = tile * kTokens;
    start = a.starts ? a.starts[b] : 0;
    return true;
  }
  // The pages of positions [lo, hi], which span at most kTokens.
  __device__ __forceinline__ void find(const RowArgs& a, long long lo, long long hi) {
    const int log2 = a.index.page_log2;
    cross = (int)((lo >> log2) + 1) << log2;
    const long long first = a.index.row(b, h, (int)lo, a.status);
    const long long second = hi >= cross ? a.index.row(b, h, cross, a.status) : 0;
    base = first < 0 ? kBad : first - lo;
    base2 = second < 0 ? kBad : second - cross;
  }
  __device__ __forceinline__ long long row(long long pos) const { return (pos < cross ? base : base2) + pos; }
  static constexpr long long kBad = -(1ll << 62);
};

// How a lane's 16 bf16 values may be accessed: by element, in 16-byte halves, whole.
enum Access { kElement, kHalf, kFull };

template <Access kA>
__device__ __forceinline__ void load16(const uint16_t* p, uint32_t w[8]) {
  if constexpr (kA == kFull) {
    load32(p, w);
  } else if constexpr (kA == kHalf) {
    *reinterpret_cast<uint4*>(w) = __ldcs(reinterpret_cast<const uint4*>(p));
    *reinterpret_cast<uint4*>(w + 4) = __ldcs(reinterpret_cast<const uint4*>(p) + 1);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
  }
}
template <Access kA>
__device__ __forceinline__ void store16(uint16_t* p, const uint32_t w[8]) {
  if constexpr (kA == kFull) {
    store32(p, w);
  } else if constexpr (kA == kHalf) {
    reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
  }
}

template <int D, int FMT, Access kA>
__global__ void __launch_bounds__(kThreads) kvq_append_kernel(const __grid_constant__ RowArgs a) {
  constexpr int kLanes = D / 16, kGroups = 32 / kLanes;
  allow_dependent_launch();
  grid_dependency_wait();
  // a large grid has more than 2^31 threads: those of the first blocks write the lengths
  if (a.new_lens && blockIdx.x <= (uint32_t)(a.batch - 1) / kThreads) {
    const uint32_t b = blockIdx.x * (uint32_t)kThreads + threadIdx.x;
    if (b < (uint32_t)a.batch) {
      const int start = a.starts[b];
      const long long end = (long long)start + (a.counts ? min(max(a.counts[b], 0), a.n) : a.n);
      a.new_lens[b] = start < 0 ? start : (int)min(end, max(a.index.capacity(), (long long)start));
    }
  }
  WarpRows<kGroups> rows;
  if (!rows.init(a)) return;
  const int l = threadIdx.x % kLanes, t = rows.t0 + (threadIdx.x & 31) / kLanes;
  uint32_t w[2][8];
#pragma unroll
  for (int i = 0; i < 2; ++i) load16<kA>((i ? a.v : a.k).row(rows.b, min(t, a.n - 1), rows.h) + 16 * l, w[i]);
  int count = a.n;
  if (a.counts) {
    count = a.counts[rows.b];
    if ((count < 0 || count > a.n) && a.status) atomicOr(a.status, kDevBadLength);
    count = min(max(count, 0), a.n);
  }
  // tokens [t0, end) have a place in the sequence
  int end = min(rows.t0 + kGroups, count);
  if (end > rows.t0 && (rows.start < 0 || rows.start + end > a.index.capacity())) {
    if (a.status) atomicOr(a.status, kDevAppendOverflow);
    end = rows.start < 0 ? rows.t0 : (int)min((long long)end, a.index.capacity() - rows.start);
  }
  if (end <= rows.t0) return;
  rows.find(a, rows.start + rows.t0, rows.start + end - 1);
  const long long dst = rows.row(rows.start + t);
  const bool store = t < end && dst >= 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t codes[4];
    const float scale = quantise_row<kLanes, 8, FMT>(w[i], codes);
    if (store) {
      *reinterpret_cast<uint4*>((i ? a.pool.v_codes : a.pool.k_codes) + dst * D + 16 * l) =
          make_uint4(codes[0], codes[1], codes[2], codes[3]);
      if (l == 0) (i ? a.pool.v_scales : a.pool.k_scales)[dst] = scale;
    }
  }
}

template <int D, int FMT, Access kA>
__global__ void __launch_bounds__(kThreads) kvq_read_kernel(const __grid_constant__ RowArgs a) {
  constexpr int kLanes = D / 16, kGroups = 32 / kLanes;
  allow_dependent_launch();
  grid_dependency_wait();
  WarpRows<kGroups> rows;
  if (!rows.init(a)) return;
  const int l = threadIdx.x % kLanes, t = rows.t0 + (threadIdx.x & 31) / kLanes;
  const int given = a.counts[rows.b];
  const int len = min(max(given, 0), (int)a.index.capacity());
  if (given != len && a.status) atomicOr(a.status, kDevBadLength);
  // positions [lo, hi) of the warp's tokens are cached
  const long long lo = max(rows.start + rows.t0, 0ll), hi = min(rows.start + rows.t0 + kGroups, (long long)len);
  if (lo < hi) rows.find(a, lo, hi - 1);
  const long long pos = rows.start + t;
  const long long src = pos >= lo && pos < hi ? rows.row(pos) : -1;
  uint4 c[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  float scale[2] = {0.f, 0.f};
  if (src >= 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      c[i] = *reinterpret_cast<const uint4*>((i ? a.pool.v_codes : a.pool.k_codes) + src * D + 16 * l);
      scale[i] = (i ? a.pool.v_scales : a.pool.k_scales)[src];
    }
  }
  if (t >= a.n) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t cw[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
    uint32_t w[8];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      float2 f[2];
      codes_to_f32<FMT>(cw[m], f);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        f[k] = mul2(f[k], make_float2(scale[i], scale[i]));
        w[2 * m + k] = pack2_rn(f[k].x, f[k].y);
      }
    }
    store16<kA>((i ? a.vo : a.ko).row(rows.b, t, rows.h) + 16 * l, w);
  }
}

Access access_of(const void* p, long long sb, int batch, long long sh, int heads, long long st, int n) {
  const int bytes = row_alignment(p, sb, batch, st, n, sh, heads);
  return bytes >= 32 ? kFull : bytes >= 16 ? kHalf : kElement;
}

// Whether the rows of a call fit one launch: warps are counted in 31 bits, and so
// are the positions up to a warp's last.
bool set_rows(RowArgs* a, const lara_kvq_pool& pool, int batch, int n) {
  a->pool = pool;
  a->batch = batch;
  a->n = n;
  a->div_h = FastDiv((uint32_t)pool.n_kv_heads);
  const int tokens = 512 / pool.head_dim;  // a warp's
  const uint32_t tiles = ((uint32_t)n + tokens - 1) / tokens;
  if (n > 1 << 30 || (tiles > 0 && (long long)batch * pool.n_kv_heads > 0x7fffffffll / tiles)) return false;
  a->div_tiles = FastDiv(std::max(tiles, 1u));
  a->tiles = (uint32_t)batch * (uint32_t)pool.n_kv_heads * tiles;
  return true;
}

cudaError_t launch_rows(const void* kernel, RowArgs a, void* stream) {
  // a thread for each length: without rows they alone are written
  const unsigned blocks = std::max(((unsigned)a.batch + kThreads - 1) / kThreads,
                                   (a.tiles + kThreads / 32 - 1) / (kThreads / 32));
  void* args[] = {&a};
  return launch_with_pdl(kernel, dim3(blocks), dim3(kThreads), args, 0, static_cast<cudaStream_t>(stream));
}

#define LARA_KVQ_LAUNCH(kernel, d, f, v)                            \
  if (pool->head_dim == d && pool->format == f && access == v)     \
    e = launch_rows(reinterpret_cast<const void*>(&kernel<d, f, v>), a, stream);
#define LARA_KVQ_LAUNCH_ACCESS(kernel, d, f) \
  LARA_KVQ_LAUNCH(kernel, d, f, kElement) LARA_KVQ_LAUNCH(kernel, d, f, kHalf) LARA_KVQ_LAUNCH(kernel, d, f, kFull)
#define LARA_KVQ_LAUNCH_ALL(kernel)                                                                       \
  LARA_KVQ_LAUNCH_ACCESS(kernel, 128, LARA_KVQ_INT8) LARA_KVQ_LAUNCH_ACCESS(kernel, 128, LARA_KVQ_FP8_E4M3) \
  LARA_KVQ_LAUNCH_ACCESS(kernel, 64, LARA_KVQ_INT8) LARA_KVQ_LAUNCH_ACCESS(kernel, 64, LARA_KVQ_FP8_E4M3)

}  // namespace

}  // namespace lara

using namespace lara;

extern "C" int lara_kvq_append(const lara_kvq_pool* pool, const int32_t* block_table, int pages_per_seq,
                               const int32_t* starts, const int32_t* counts, int32_t* new_lens, const uint16_t* k_new,
                               long long k_sb, long long k_sh, long long k_st, const uint16_t* v_new, long long v_sb,
                               long long v_sh, long long v_st, int batch, int n_new, void* workspace, void* stream) {
  LARA_NVTX("lara_kvq_append");
  RowArgs a{};
  if (const int rc = check_pool(pool, block_table, pages_per_seq, batch, &a.index)) return rc;
  if (batch < 0 || n_new < 0) return set_last_error(LARA_ERR_BAD_CFG, "batch and n_new must not be negative");
  if (batch == 0) return LARA_OK;
  if (!starts || (n_new > 0 && (!k_new || !v_new))) return set_last_error(LARA_ERR_STREAM_DEST, "null pointer");
  if (!aligned(k_new, 2) || !aligned(v_new, 2) || !aligned(starts, 4) || !aligned(counts, 4) ||
      !aligned(new_lens, 4) || !aligned(workspace, 4))
    return set_last_error(LARA_ERR_STREAM_DEST, "misaligned buffer");
  if (overlap(new_lens, starts, 4 * (size_t)batch) || overlap(new_lens, counts, 4 * (size_t)batch))
    return set_last_error(LARA_ERR_STREAM_DEST, "new_lens must not overlap starts or counts");
  a.starts = starts;
  a.counts = counts;
  a.new_lens = new_lens;
  a.k = {k_new, k_sb, k_st, k_sh};
  a.v = {v_new, v_sb, v_st, v_sh};
  a.status = static_cast<int*>(workspace);
  if (!set_rows(&a, *pool, batch, n_new)) return set_last_error(LARA_ERR_BAD_CFG, "too many rows for one launch");
  if (n_new == 0 && !new_lens) return LARA_OK;
  const int heads = pool->n_kv_heads;
  const Access access = std::min(access_of(k_new, k_sb, batch, k_sh, heads, k_st, n_new),
                                 access_of(v_new, v_sb, batch, v_sh, heads, v_st, n_new));
  cudaError_t e = cudaErrorInvalidValue;
  LARA_KVQ_LAUNCH_ALL(kvq_append_kernel)
  if (e != cudaSuccess)
    return set_last_error(LARA_ERR_CUDA, std::string("kvq_append launch: ") + cudaGetErrorString(e));
  return LARA_OK;
}

extern "C" int lara_kvq_read(const lara_kvq_pool* pool, const int32_t* block_table, int pages_per_seq,
                             const int32_t* seq_lens, const int32_t* starts, uint16_t* k_out, long long k_sb,
                             long long k_sh, long long k_st, uint16_t* v_out, long long v_sb, long long v_sh,
                             long long v_st, int batch, int n_tokens, void* workspace, void* stream) {
  LARA_NVTX("lara_kvq_read");
  RowArgs a{};
  if (const int rc = check_pool(pool, block_table, pages_per_seq, batch, &a.index)) return rc;
  if (batch < 0 || n_tokens < 0) return set_last_error(LARA_ERR_BAD_CFG, "batch and n_tokens must not be negative");
  if (batch == 0 || n_tokens == 0) return LARA_OK;
  if (!seq_lens || !k_out || !v_out) return set_last_error(LARA_ERR_STREAM_DEST, "null pointer");
  if (!aligned(k_out, 2) || !aligned(v_out, 2) || !aligned(starts, 4) || !aligned(seq_lens, 4) ||
      !aligned(workspace, 4))
    return set_last_error(LARA_ERR_STREAM_DEST, "misaligned buffer");
  a.starts = starts;
  a.counts = seq_lens;
  a.ko = {k_out, k_sb, k_st, k_sh};
  a.vo = {v_out, v_sb, v_st, v_sh};
  a.status = static_cast<int*>(workspace);
  if (!set_rows(&a, *pool, batch, n_tokens)) return set_last_error(LARA_ERR_BAD_CFG, "too many rows for one launch");
  const int heads = pool->n_kv_heads;
  const Access access = std::min(access_of(k_out, k_sb, batch, k_sh, heads, k_st, n_tokens),
                                 access_of(v_out, v_sb, batch, v_sh, heads, v_st, n_tokens));
  cudaError_t e = cudaErrorInvalidValue;
  LARA_KVQ_LAUNCH_ALL(kvq_read_kernel)
  if (e != cudaSuccess)
    return set_last_error(LARA_ERR_CUDA, std::string("kvq_read launch: ") + cudaGetErrorString(e));
  return LARA_OK;
}
