// The row work of a serving step in one launch (declared in include/lara_b200.h):
// q and k heads are normed and rotated, k and v quantised into the paged pool.
//
// Bound by latency at a decode step (a few hundred rows; one launch in place of
// two, and k does not go to memory as bf16 in between), by HBM for prompts:
// q 4 D bytes per head, k and v 2 D + D + 4.  Heads are held, normed and
// rotated as in qk_rope.cu; k is rounded to bf16 and quantised from there, so
// the pool gets the words of the two calls.  A block takes q, k or v alone, a
// lane group kHeads heads of one token.
#include <algorithm>

#include "kvq.cuh"

namespace lara {

using namespace kvq;

namespace {

constexpr int kThreads = 128;

struct QkvArgs {
  lara_kvq_pool pool;
  PoolIndex index;
  const int32_t* starts;
  const int32_t* counts;
  int32_t* new_lens;
  Heads<const uint16_t> q, k, v;
  Heads<uint16_t> qo;
  int batch, n, hq;
  uint32_t tokens, blocks[2];  // blocks of q, of k (and of v)
  FastDiv chunks[2], div_n;    // chunks of heads per token: of q, of k and v
  const int32_t* positions;
  const float* cos_sin;
  int max_pos, rot;
  const uint16_t* qw;
  const uint16_t* kw;
  float eps;
  int* status;
};

template <int D, int W, int FMT, bool kInter, bool kNorm, bool kVec, int kHeads>
__global__ void __launch_bounds__(kThreads) kvq_append_qkv_kernel(const __grid_constant__ QkvArgs a) {
  constexpr int kLanes = D / (2 * W);
  allow_dependent_launch();
  grid_dependency_wait();
  const long long cap = a.index.capacity();
  // a large grid has more than 2^31 threads: those of the first blocks write the lengths
  if (a.new_lens && blockIdx.x <= (uint32_t)(a.batch - 1) / kThreads) {
    const uint32_t b = blockIdx.x * (uint32_t)kThreads + threadIdx.x;
    if (b < (uint32_t)a.batch) {
      const int start = a.starts[b];
      const long long end = (long long)start + (a.counts ? min(max(a.counts[b], 0), a.n) : a.n);
      a.new_lens[b] = start < 0 ? start : (int)min(end, max(cap, (long long)start));
    }
  }
  if (a.tokens == 0) return;
  const uint32_t x = blockIdx.x;
  const int kind = x < a.blocks[0] ? 0 : x < a.blocks[0] + a.blocks[1] ? 1 : 2;  // q, k, v
  const uint32_t block = x - (kind == 0 ? 0 : a.blocks[0] + (kind == 1 ? 0 : a.blocks[1]));
  const FastDiv& chunks = a.chunks[kind == 0 ? 0 : 1];
  const uint32_t group = block * (uint32_t)(kThreads / kLanes) + threadIdx.x / kLanes;
  const int l = threadIdx.x % kLanes;
  const bool active = group < a.tokens * chunks.d;
  uint32_t t, chunk;
  const uint32_t tok = chunks.div(active ? group : 0, chunk);
  const uint32_t b = a.div_n.div(tok, t);
  const int h0 = (int)chunk * kHeads;
  const int heads = active ? (kind == 0 ? a.hq : a.pool.n_kv_heads) - h0 : 0;  // to store, at most kHeads
  const HeadLane<W> ld(l, kind == 2 ? 0 : a.rot, kInter);  // v is not turned

  const Heads<const uint16_t>& in = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
  const uint16_t* src = in.row(b, t, h0);
  uint32_t w[kHeads][W];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) load_words<W, kInter, kVec>(src + (i < heads ? i : 0) * in.sh, ld, w[i]);
  const int start = a.starts[b];
  // tokens past the count are padding: nothing is stored or reported for them
  auto given_count = [&] { return a.counts ? a.counts[b] : a.n; };
  if (kind != 2) {
    const float* row = nullptr;
    if (ld.rotated) {
      long long pos = a.positions ? a.positions[tok] : (long long)start + t;
      if (pos < 0 || pos >= a.max_pos) {
        if (a.status && (int)t < given_count()) atomicOr(a.status, kDevBadPosition);
        pos = pos < 0 ? 0 : a.max_pos - 1;
      }
      row = a.cos_sin + pos * a.rot;
    }
    const Turn<W> turn = make_turn<W, kInter>(row, a.rot, l, kNorm ? (kind == 0 ? a.qw : a.kw) : nullptr, ld);
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
      words_of<W, kInter>(turn_head<D, W, kNorm>(pairs_of<W, kInter>(w[i]), turn, ld.rotated, a.eps), w[i]);
  }
  if (kind == 0) {
    uint16_t* dst = a.qo.row(b, t, h0);
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
      if (i < heads) store_words<W, kInter, kVec>(dst + i * a.qo.sh, ld, w[i]);
    return;
  }
  // where the token's first row lies: its heads are a page's rows apart
  long long dst = -1;
  if (heads > 0) {
    const int count = given_count();
    if ((count < 0 || count > a.n) && a.status) atomicOr(a.status, kDevBadLength);
    if ((int)t < count) {
      const long long pos = (long long)start + t;
      if (start < 0 || pos >= cap) {
        if (a.status) atomicOr(a.status, kDevAppendOverflow);
      } else {
        dst = a.index.row((int)b, h0, (int)pos, a.status);
      }
    }
  }
  uint8_t* const codes_out = kind == 1 ? a.pool.k_codes : a.pool.v_codes;
  float* const scales_out = kind == 1 ? a.pool.k_scales : a.pool.v_scales;
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    uint32_t codes[W / 2];
    const float scale = quantise_row<kLanes, W, FMT>(w[i], codes);
    if (i < heads && dst >= 0) {
      const long long row = dst + ((long long)i << a.index.page_log2);
      uint8_t *c0 = codes_out + row * D + ld.o0, *c1 = codes_out + row * D + ld.o1;
      if constexpr (W == 8) {
        *reinterpret_cast<uint2*>(c0) = make_uint2(codes[0], codes[1]);
        *reinterpret_cast<uint2*>(c1) = make_uint2(codes[2], codes[3]);
      } else {
        *reinterpret_cast<uint32_t*>(c0) = codes[0];
        *reinterpret_cast<uint32_t*>(c1) = codes[1];
      }
      if (l == 0) scales_out[row] = scale;
    }
  }
}

template <int D, int W, int FMT, bool kInter, bool kNorm, bool kVec, int kHeads>
cudaError_t launch_heads(QkvArgs a, uint32_t tokens, cudaStream_t stream) {
  const uint32_t per_block = kThreads / (D / (2 * W));
  const int heads[2] = {a.hq, a.pool.n_kv_heads};
  for (int i = 0; i < 2; ++i) {
    const uint32_t chunks = (heads[i] + kHeads - 1) / kHeads;
    a.chunks[i] = FastDiv(chunks);
    a.blocks[i] = (tokens * chunks + per_block - 1) / per_block;
  }
  a.tokens = tokens;
  // a thread for each length: without tokens they alone are written
  const dim3 grid(std::max(((unsigned)a.batch + kThreads - 1) / kThreads, a.blocks[0] + 2 * a.blocks[1]));
  void* args[] = {&a};
  return launch_with_pdl(reinterpret_cast<const void*>(&kvq_append_qkv_kernel<D, W, FMT, kInter, kNorm, kVec, kHeads>),
                         grid, dim3(kThreads), args, 0, stream);
}

// Heads per lane group, on the grounds of qk_rope.cu; the boundary by 32 + 8 + 8
// heads (head_dim 128, int8) that would fill the GPU 0.6, 0.75, 1.2, 2 times: one each 3.5,
// 3.5, 3.9, 5.5 us, four 3.9, 4.2, 4.6, 4.9 (8 + 2 + 2 heads of 64 dims: 3.3, 3.3, 3.8, 5.3
// and 4.1, 3.7, 4.4, 5.4).  Those heads of 64 single tokens take 2.7 us (the two
// calls 4.1), of 2000 tokens 8.4 us (10.2), of 8192 tokens 36 us (39; 0.78 of the
// copy rate).
template <int D, int W, int FMT, bool kInter, bool kNorm, bool kVec>
cudaError_t launch(const QkvArgs& a, uint32_t tokens, cudaStream_t stream) {
  const double fill = (double)tokens * (a.hq + 2 * a.pool.n_kv_heads) * (D / 8) / (device_sm_count() * 2048.0);
  return fill < 1.5 ? launch_heads<D, W, FMT, kInter, kNorm, kVec, 1>(a, tokens, stream)
                    : launch_heads<D, W, FMT, kInter, kNorm, kVec, 4>(a, tokens, stream);
}

// W by the rule of qk_rope.cu.
template <int D, int FMT, bool kInter, bool kNorm>
cudaError_t launch(const QkvArgs& a, uint32_t tokens, int alignment, cudaStream_t st) {
  if (alignment >= 32 && a.rot % 16 == 0) return launch<D, 8, FMT, kInter, kNorm, true>(a, tokens, st);
  return alignment >= 16 ? launch<D, 4, FMT, kInter, kNorm, true>(a, tokens, st)
                         : launch<D, 4, FMT, kInter, kNorm, false>(a, tokens, st);
}

template <int D, int FMT>
cudaError_t launch(const QkvArgs& a, uint32_t tokens, bool inter, int alignment, cudaStream_t st) {
  if (a.qw)
    return inter ? launch<D, FMT, true, true>(a, tokens, alignment, st)
                 : launch<D, FMT, false, true>(a, tokens, alignment, st);
  return inter ? launch<D, FMT, true, false>(a, tokens, alignment, st)
               : launch<D, FMT, false, false>(a, tokens, alignment, st);
}

}  // namespace

}  // namespace lara

using namespace lara;

extern "C" int lara_kvq_append_qkv(const lara_kvq_pool* pool, const int32_t* block_table, int pages_per_seq,
                                   const int32_t* starts, const int32_t* counts, int32_t* new_lens, const uint16_t* q,
                                   long long q_sb, long long q_st, long long q_sh, const uint16_t* k, long long k_sb,
                                   long long k_st, long long k_sh, const uint16_t* v, long long v_sb, long long v_st,
                                   long long v_sh, uint16_t* q_out, long long qo_sb, long long qo_st, long long qo_sh,
                                   int batch, int n_new, int n_q_heads, const int32_t* positions, const float* cos_sin,
                                   int max_pos, int rot_dim, int interleaved, const uint16_t* q_weight,
                                   const uint16_t* k_weight, float eps, void* workspace, void* stream) {
  LARA_NVTX("lara_kvq_append_qkv");
  QkvArgs a{};
  if (const int rc = check_pool(pool, block_table, pages_per_seq, batch, &a.index)) return rc;
  const int hkv = pool->n_kv_heads;
  if (batch < 0 || n_new < 0 || n_q_heads < 1 || n_q_heads > 65535 || hkv > 65535 ||
      (long long)batch * n_new > 0x7fffffffll / (n_q_heads + 2 * hkv))
    return set_last_error(LARA_ERR_BAD_CFG, "bad geometry: batch, n_new >= 0, below 2^31 heads in all");
  if (!q_weight != !k_weight) return set_last_error(LARA_ERR_BAD_CFG, "q_weight and k_weight go together");
  if (cos_sin && (rot_dim < 8 || rot_dim > pool->head_dim || rot_dim % 8 || max_pos < 1))
    return set_last_error(LARA_ERR_BAD_CFG, "rot_dim must be a multiple of 8 up to head_dim, max_pos >= 1");
  if (!(eps >= 0.f)) return set_last_error(LARA_ERR_BAD_CFG, "eps must not be negative");
  if (batch == 0) return LARA_OK;
  if (!starts || (n_new > 0 && (!q || !k || !v || !q_out))) return set_last_error(LARA_ERR_STREAM_DEST, "null pointer");
  if (!aligned(q, 2) || !aligned(k, 2) || !aligned(v, 2) || !aligned(q_out, 2) || !aligned(starts, 4) ||
      !aligned(counts, 4) || !aligned(new_lens, 4) || !aligned(positions, 4) || !aligned(cos_sin, 16) ||
      !aligned(q_weight, 16) || !aligned(k_weight, 16) || !aligned(workspace, 4))
    return set_last_error(LARA_ERR_STREAM_DEST, "cos_sin and the weights must be 16-byte aligned");
  if (overlap(new_lens, starts, 4 * (size_t)batch) || overlap(new_lens, counts, 4 * (size_t)batch))
    return set_last_error(LARA_ERR_STREAM_DEST, "new_lens must not overlap starts or counts");
  if (n_new == 0 && !new_lens) return LARA_OK;
  const int alignment = std::min({row_alignment(q, q_sb, batch, q_st, n_new, q_sh, n_q_heads),
                                  row_alignment(k, k_sb, batch, k_st, n_new, k_sh, hkv),
                                  row_alignment(v, v_sb, batch, v_st, n_new, v_sh, hkv),
                                  row_alignment(q_out, qo_sb, batch, qo_st, n_new, qo_sh, n_q_heads)});
  a.pool = *pool;
  a.starts = starts;
  a.counts = counts;
  a.new_lens = new_lens;
  a.q = {q, q_sb, q_st, q_sh};
  a.k = {k, k_sb, k_st, k_sh};
  a.v = {v, v_sb, v_st, v_sh};
  a.qo = {q_out, qo_sb, qo_st, qo_sh};
  a.batch = batch;
  a.n = n_new;
  a.hq = n_q_heads;
  a.div_n = FastDiv((uint32_t)n_new);
  a.positions = positions;
  a.cos_sin = cos_sin;
  a.max_pos = max_pos;
  a.rot = cos_sin ? rot_dim : 0;
  a.qw = q_weight;
  a.kw = k_weight;
  a.eps = eps;
  a.status = static_cast<int*>(workspace);
  const uint32_t tokens = (uint32_t)batch * (uint32_t)n_new;
  const bool inter = interleaved || !cos_sin;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaErrorInvalidValue;
#define LARA_CASE(d, f) \
  if (pool->head_dim == d && pool->format == f) e = launch<d, f>(a, tokens, inter, alignment, st);
  LARA_CASE(128, LARA_KVQ_INT8) LARA_CASE(128, LARA_KVQ_FP8_E4M3)
  LARA_CASE(64, LARA_KVQ_INT8) LARA_CASE(64, LARA_KVQ_FP8_E4M3)
#undef LARA_CASE
  if (e != cudaSuccess)
    return set_last_error(LARA_ERR_CUDA, std::string("kvq_append_qkv launch: ") + cudaGetErrorString(e));
  return LARA_OK;
}
