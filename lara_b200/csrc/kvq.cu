// Writing and reading the paged 8-bit KV pool (declared in include/lara_b200.h;
// the write replaces the K/V cache write of hw/rtl/mem/kv_cache_ram.sv:45-91
// for a quantised cache).
//
// Both are bound by HBM: append reads 2 D bytes of bf16 per row and writes
// D + 4, read the reverse.  D / 8 lanes hold a row, and a lane group takes the
// K and the V row of one (token, kv head), so both loads are in flight.
#include "kvq.cuh"

namespace lara {

namespace kvq {

int check_pool(const lara_kvq_pool* pool, const void* block_table, int pages_per_seq, PoolIndex* index) {
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
  if (!pool->k_codes || !pool->v_codes || !pool->k_scales || !pool->v_scales || !block_table)
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
  uint32_t rows;
  int* status;
};

template <int D, int FMT, bool kVec>
__global__ void __launch_bounds__(kThreads) kvq_append_kernel(const __grid_constant__ RowArgs a) {
  constexpr int kLanes = D / 8;
  const uint32_t tid = blockIdx.x * (uint32_t)kThreads + threadIdx.x;
  if (a.new_lens)
    for (uint32_t b = tid; b < (uint32_t)a.batch; b += gridDim.x * (uint32_t)kThreads) {
      const int start = a.starts[b];
      const long long end = (long long)start + (a.counts ? min(max(a.counts[b], 0), a.n) : a.n);
      a.new_lens[b] = start < 0 ? start : (int)min(end, max(a.index.capacity(), (long long)start));
    }
  const uint32_t row = tid / kLanes;
  if (row - (threadIdx.x & 31) / kLanes >= a.rows) return;  // the whole warp is past the end
  const uint32_t r = min(row, a.rows - 1);
  const int l = threadIdx.x % kLanes;
  const int t = (int)(r % (uint32_t)a.n);
  const uint32_t bh = r / (uint32_t)a.n;
  const int h = (int)(bh % (uint32_t)a.pool.n_kv_heads), b = (int)(bh / (uint32_t)a.pool.n_kv_heads);
  int count = a.n;
  if (a.counts) {
    count = a.counts[b];
    if ((count < 0 || count > a.n) && a.status) atomicOr(a.status, kDevBadLength);
  }
  const int start = a.starts[b];
  const long long pos = (long long)start + t;
  long long dst = -1;
  if (row < a.rows && t < count) {
    if (start < 0 || pos >= a.index.capacity()) {
      if (a.status) atomicOr(a.status, kDevAppendOverflow);
    } else {
      dst = a.index.row(b, h, (int)pos, a.status);
    }
  }
  uint32_t w[2][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint16_t* src = (i ? a.v : a.k).row(b, t, h) + 8 * l;
    if constexpr (kVec) {
      *reinterpret_cast<uint4*>(w[i]) = *reinterpret_cast<const uint4*>(src);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[i][j] = (uint32_t)src[2 * j] | ((uint32_t)src[2 * j + 1] << 16);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t codes[2];
    const float scale = quantise_row<D, FMT>(w[i], codes);
    if (dst >= 0) {
      *reinterpret_cast<uint2*>((i ? a.pool.v_codes : a.pool.k_codes) + dst * D + 8 * l) =
          make_uint2(codes[0], codes[1]);
      if (l == 0) (i ? a.pool.v_scales : a.pool.k_scales)[dst] = scale;
    }
  }
}

template <int D, int FMT, bool kVec>
__global__ void __launch_bounds__(kThreads) kvq_read_kernel(const __grid_constant__ RowArgs a) {
  constexpr int kLanes = D / 8;
  const uint32_t row = (blockIdx.x * (uint32_t)kThreads + threadIdx.x) / kLanes;
  if (row >= a.rows) return;
  const int l = threadIdx.x % kLanes;
  const int t = (int)(row % (uint32_t)a.n);
  const uint32_t bh = row / (uint32_t)a.n;
  const int h = (int)(bh % (uint32_t)a.pool.n_kv_heads), b = (int)(bh / (uint32_t)a.pool.n_kv_heads);
  const int len = a.counts[b];
  if ((len < 0 || len > a.index.capacity()) && a.status) atomicOr(a.status, kDevBadLength);
  const long long pos = (a.starts ? (long long)a.starts[b] : 0) + t;
  long long src = -1;
  if (pos >= 0 && pos < len && pos < a.index.capacity()) src = a.index.row(b, h, (int)pos, a.status);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t w[4] = {0, 0, 0, 0};
    if (src >= 0) {
      const uint2 c = *reinterpret_cast<const uint2*>((i ? a.pool.v_codes : a.pool.k_codes) + src * D + 8 * l);
      const float scale = (i ? a.pool.v_scales : a.pool.k_scales)[src];
      float f[8];
      codes_to_f32<FMT>(c.x, f);
      codes_to_f32<FMT>(c.y, f + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = pack2_rn(f[2 * j] * scale, f[2 * j + 1] * scale);
    }
    uint16_t* dst = (i ? a.vo : a.ko).row(b, t, h) + 8 * l;
    if constexpr (kVec) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) dst[j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
    }
  }
}

// 16-byte accesses: the base and every stride that is taken (an extent of 1
// takes none).
bool vec_ok(const void* p, long long sb, int batch, long long sh, int heads, long long st, int n) {
  return aligned(p, 16) && (((batch > 1 ? sb : 0) | (heads > 1 ? sh : 0) | (n > 1 ? st : 0)) & 7) == 0;
}

// rows = batch * Hkv * n as a launch over D / 8 lanes each, or 0 when it does not fit one.
long long row_blocks(const lara_kvq_pool& pool, int batch, int n, uint32_t* rows) {
  const long long bh = (long long)batch * pool.n_kv_heads;
  if (bh > 0x7fffffffll || bh * n > 0x7fffffffll / (pool.head_dim / 8)) return -1;
  *rows = (uint32_t)(bh * n);
  return (bh * n * (pool.head_dim / 8) + kThreads - 1) / kThreads;
}

template <typename F>
cudaError_t launch_rows(F kernel, long long blocks, const RowArgs& a, void* stream) {
  kernel<<<(unsigned)blocks, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return cudaGetLastError();
}

bool overlap(const void* a, const void* b, size_t bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a && b && x < y + bytes && y < x + bytes;
}

}  // namespace

}  // namespace lara

using namespace lara;

extern "C" int lara_kvq_append(const lara_kvq_pool* pool, const int32_t* block_table, int pages_per_seq,
                               const int32_t* starts, const int32_t* counts, int32_t* new_lens, const uint16_t* k_new,
                               long long k_sb, long long k_sh, long long k_st, const uint16_t* v_new, long long v_sb,
                               long long v_sh, long long v_st, int batch, int n_new, void* workspace, void* stream) {
  LARA_NVTX("lara_kvq_append");
  RowArgs a{};
  if (const int rc = check_pool(pool, block_table, pages_per_seq, &a.index)) return rc;
  if (batch < 0 || n_new < 0) return set_last_error(LARA_ERR_BAD_CFG, "batch and n_new must not be negative");
  if (batch == 0) return LARA_OK;
  if (!starts || (n_new > 0 && (!k_new || !v_new))) return set_last_error(LARA_ERR_STREAM_DEST, "null pointer");
  if (!aligned(k_new, 2) || !aligned(v_new, 2) || !aligned(starts, 4) || !aligned(counts, 4) ||
      !aligned(new_lens, 4) || !aligned(workspace, 4))
    return set_last_error(LARA_ERR_STREAM_DEST, "misaligned buffer");
  if (overlap(new_lens, starts, 4 * (size_t)batch) || overlap(new_lens, counts, 4 * (size_t)batch))
    return set_last_error(LARA_ERR_STREAM_DEST, "new_lens must not overlap starts or counts");
  a.pool = *pool;
  a.starts = starts;
  a.counts = counts;
  a.new_lens = new_lens;
  a.k = {k_new, k_sb, k_st, k_sh};
  a.v = {v_new, v_sb, v_st, v_sh};
  a.batch = batch;
  a.n = n_new;
  a.status = static_cast<int*>(workspace);
  long long blocks = row_blocks(*pool, batch, n_new, &a.rows);
  if (blocks < 0) return set_last_error(LARA_ERR_BAD_CFG, "too many rows for one launch");
  if (blocks == 0) {
    if (!new_lens) return LARA_OK;
    blocks = 1;
  }
  const int heads = pool->n_kv_heads;
  const bool vec = vec_ok(k_new, k_sb, batch, k_sh, heads, k_st, n_new) &&
                   vec_ok(v_new, v_sb, batch, v_sh, heads, v_st, n_new);
  cudaError_t e = cudaErrorInvalidValue;
#define LARA_CASE(d, f)                                                                        \
  if (pool->head_dim == d && pool->format == f)                                                \
    e = vec ? launch_rows(kvq_append_kernel<d, f, true>, blocks, a, stream)                    \
            : launch_rows(kvq_append_kernel<d, f, false>, blocks, a, stream);
  LARA_CASE(128, LARA_KVQ_INT8) LARA_CASE(128, LARA_KVQ_FP8_E4M3)
  LARA_CASE(64, LARA_KVQ_INT8) LARA_CASE(64, LARA_KVQ_FP8_E4M3)
#undef LARA_CASE
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
  if (const int rc = check_pool(pool, block_table, pages_per_seq, &a.index)) return rc;
  if (batch < 0 || n_tokens < 0) return set_last_error(LARA_ERR_BAD_CFG, "batch and n_tokens must not be negative");
  if (batch == 0 || n_tokens == 0) return LARA_OK;
  if (!seq_lens || !k_out || !v_out) return set_last_error(LARA_ERR_STREAM_DEST, "null pointer");
  if (!aligned(k_out, 2) || !aligned(v_out, 2) || !aligned(starts, 4) || !aligned(seq_lens, 4) ||
      !aligned(workspace, 4))
    return set_last_error(LARA_ERR_STREAM_DEST, "misaligned buffer");
  a.pool = *pool;
  a.starts = starts;
  a.counts = seq_lens;
  a.ko = {k_out, k_sb, k_st, k_sh};
  a.vo = {v_out, v_sb, v_st, v_sh};
  a.batch = batch;
  a.n = n_tokens;
  a.status = static_cast<int*>(workspace);
  const long long blocks = row_blocks(*pool, batch, n_tokens, &a.rows);
  if (blocks < 0) return set_last_error(LARA_ERR_BAD_CFG, "too many rows for one launch");
  const int heads = pool->n_kv_heads;
  const bool vec = vec_ok(k_out, k_sb, batch, k_sh, heads, k_st, n_tokens) &&
                   vec_ok(v_out, v_sb, batch, v_sh, heads, v_st, n_tokens);
  cudaError_t e = cudaErrorInvalidValue;
#define LARA_CASE(d, f)                                                                        \
  if (pool->head_dim == d && pool->format == f)                                                \
    e = vec ? launch_rows(kvq_read_kernel<d, f, true>, blocks, a, stream)                      \
            : launch_rows(kvq_read_kernel<d, f, false>, blocks, a, stream);
  LARA_CASE(128, LARA_KVQ_INT8) LARA_CASE(128, LARA_KVQ_FP8_E4M3)
  LARA_CASE(64, LARA_KVQ_INT8) LARA_CASE(64, LARA_KVQ_FP8_E4M3)
#undef LARA_CASE
  if (e != cudaSuccess)
    return set_last_error(LARA_ERR_CUDA, std::string("kvq_read launch: ") + cudaGetErrorString(e));
  return LARA_OK;
}
