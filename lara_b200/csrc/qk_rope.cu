// RMS norm of query and key heads with the position rotation, in one pass
// (declared in include/lara_b200.h).  The rotation's dim pairs are those of
// hw/rtl/core/rope_engine.sv:1-11 (interleaved) or half a rotation apart.
//
//   y = x w / sqrt(mean(x^2) + eps);  (y_a, y_b) -> (y_a c - y_b s, y_a s + y_b c)
//
// Bound by HBM: every head is read and written once (4 D bytes), the table row
// of a token once from HBM (4 rot bytes) and from L2 after that.  D / 16 lanes
// hold a head in registers between the load and the store.  A lane group takes
// kHeads heads of one token, all of q or all of k: it folds the weights into
// the token's cosines and sines once, and has kHeads loads in flight.
#include <algorithm>

#include "kvq.cuh"

namespace lara {

using namespace kvq;

namespace {

constexpr int kThreads = 128;

struct NormRopeArgs {
  Heads<const uint16_t> q, k;
  Heads<uint16_t> qo, ko;
  int hq, hkv, q_chunks;
  uint32_t groups;   // tokens * chunks
  FastDiv chunks, n;
  const int32_t* positions;
  const float* cos_sin;
  int max_pos, rot;
  const uint16_t* qw;
  const uint16_t* kw;
  float eps;
  int* status;
};

// Lane group i takes chunk i % chunks (kHeads heads, of q first) of token
// i / chunks, so that neighbours in the grid are neighbours in memory.
template <int D, int W, bool kInter, bool kNorm, bool kVec, int kHeads>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const __grid_constant__ NormRopeArgs a) {
  constexpr int kLanes = D / (2 * W);
  allow_dependent_launch();
  grid_dependency_wait();
  const uint32_t group = blockIdx.x * (uint32_t)(kThreads / kLanes) + threadIdx.x / kLanes;
  const int l = threadIdx.x % kLanes;
  uint32_t t, chunk;
  const uint32_t tok = a.chunks.div(min(group, a.groups - 1), chunk);
  const uint32_t b = a.n.div(tok, t);
  const bool is_k = (int)chunk >= a.q_chunks;
  const int h0 = ((int)chunk - (is_k ? a.q_chunks : 0)) * kHeads;
  const int heads = group < a.groups ? (is_k ? a.hkv : a.hq) - h0 : 0;  // to store, at most kHeads of them
  const HeadLane<W> ld(l, a.rot, kInter);

  const long long sh = is_k ? a.k.sh : a.q.sh;
  const uint16_t* src = is_k ? a.k.row(b, t, h0) : a.q.row(b, t, h0);
  uint32_t x[kHeads][W];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) load_words<W, kInter, kVec>(src + (i < heads ? i : 0) * sh, ld, x[i]);
  const float* row = nullptr;
  if (ld.rotated) {
    int pos = a.positions[tok];
    if (pos < 0 || pos >= a.max_pos) {
      if (a.status) atomicOr(a.status, kDevBadPosition);
      pos = pos < 0 ? 0 : a.max_pos - 1;
    }
    row = a.cos_sin + (long long)pos * a.rot;
  }
  const Turn<W> turn = make_turn<W, kInter>(row, a.rot, l, kNorm ? (is_k ? a.kw : a.qw) : nullptr, ld);
  const long long osh = is_k ? a.ko.sh : a.qo.sh;
  uint16_t* dst = is_k ? a.ko.row(b, t, h0) : a.qo.row(b, t, h0);
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const Pairs<W> y = turn_head<D, W, kNorm>(pairs_of<W, kInter>(x[i]), turn, ld.rotated, a.eps);
    uint32_t w[W];
    words_of<W, kInter>(y, w);
    if (i < heads) store_words<W, kInter, kVec>(dst + i * osh, ld, w);
  }
}

template <int D, int W, bool kInter, bool kNorm, bool kVec, int kHeads>
cudaError_t launch_heads(NormRopeArgs a, uint32_t tokens, cudaStream_t stream) {
  a.q_chunks = (a.hq + kHeads - 1) / kHeads;
  const uint32_t chunks = a.q_chunks + (a.hkv + kHeads - 1) / kHeads;
  a.groups = tokens * chunks;
  a.chunks = FastDiv(chunks);
  const uint32_t per_block = kThreads / (D / (2 * W));
  const dim3 grid((a.groups + per_block - 1) / per_block);
  void* args[] = {&a};
  return launch_with_pdl(reinterpret_cast<const void*>(&qk_norm_rope_kernel<D, W, kInter, kNorm, kVec, kHeads>), grid,
                         dim3(kThreads), args, 0, stream);
}

// Heads per lane group.  More of them share a token's turn and keep more loads
// in flight, fewer spread a small call over more lanes; what counts is how often
// the call would fill the GPU's threads with eight dims each.  72 heads
// (head_dim 128) of 128, 512, 1024, 16384 tokens: one each 2.8, 5.0, 8.2,
// 143 us; two 2.8, 4.6, 7.2, 132; four 2.8, 3.9, 6.2, 101; eight 3.0, 4.8, 5.4,
// 93 us (1.0 of the copy rate; 102 us with inputs that no earlier call left in
// L2).  8 dims per lane instead of 16: 1024 tokens 6.3, 2048 10.8 against 9.5 us.
// Heads that leave the last group short lose by more of them: 8 + 2 heads of 64
// dims at eight times the GPU's threads 13.4 us with two, 14.6, 15.7 with eight.
template <int D, int W, bool kInter, bool kNorm, bool kVec>
cudaError_t launch(const NormRopeArgs& a, uint32_t tokens, cudaStream_t stream) {
  const double fill = (double)tokens * (a.hq + a.hkv) * (D / 8) / (device_sm_count() * 2048.0);
  if (fill < 0.5) return launch_heads<D, W, kInter, kNorm, kVec, 1>(a, tokens, stream);
  if (fill < 1.5) return launch_heads<D, W, kInter, kNorm, kVec, 2>(a, tokens, stream);
  if (fill < 3.5) return launch_heads<D, W, kInter, kNorm, kVec, 4>(a, tokens, stream);
  return launch_heads<D, W, kInter, kNorm, kVec, 8>(a, tokens, stream);
}

// W = 8 where rows start on 32-byte boundaries and rot allows it.
template <int D, bool kInter, bool kNorm>
cudaError_t launch(const NormRopeArgs& a, uint32_t tokens, int alignment, cudaStream_t stream) {
  if (alignment >= 32 && a.rot % 16 == 0) return launch<D, 8, kInter, kNorm, true>(a, tokens, stream);
  return alignment >= 16 ? launch<D, 4, kInter, kNorm, true>(a, tokens, stream)
                         : launch<D, 4, kInter, kNorm, false>(a, tokens, stream);
}

template <int D, bool kInter>
cudaError_t launch(const NormRopeArgs& a, uint32_t tokens, int alignment, cudaStream_t stream) {
  return a.qw ? launch<D, kInter, true>(a, tokens, alignment, stream)
              : launch<D, kInter, false>(a, tokens, alignment, stream);
}

}  // namespace

}  // namespace lara

using namespace lara;

extern "C" int lara_qk_norm_rope(const uint16_t* q, long long q_sb, long long q_st, long long q_sh, const uint16_t* k,
                                 long long k_sb, long long k_st, long long k_sh, uint16_t* q_out, long long qo_sb,
                                 long long qo_st, long long qo_sh, uint16_t* k_out, long long ko_sb, long long ko_st,
                                 long long ko_sh, int batch, int n, int n_q_heads, int n_kv_heads, int head_dim,
                                 const int32_t* positions, const float* cos_sin, int max_pos, int rot_dim,
                                 int interleaved, const uint16_t* q_weight, const uint16_t* k_weight, float eps,
                                 void* workspace, void* stream) {
  LARA_NVTX("lara_qk_norm_rope");
  if (head_dim != 64 && head_dim != 128)
    return set_last_error(LARA_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  if (batch < 0 || n < 0 || n_q_heads < 1 || n_kv_heads < 1 || n_q_heads > 65535 || n_kv_heads > 65535 ||
      (long long)batch * n > 0x7fffffffll / (n_q_heads + n_kv_heads))
    return set_last_error(LARA_ERR_BAD_CFG, "bad geometry: batch, n >= 0, head counts in [1, 65535], below 2^31 heads in all");
  if (!q_weight != !k_weight) return set_last_error(LARA_ERR_BAD_CFG, "q_weight and k_weight go together");
  if (!q_weight && !cos_sin) return set_last_error(LARA_ERR_BAD_CFG, "neither norm weights nor a rotation table");
  if (cos_sin && (rot_dim < 8 || rot_dim > head_dim || rot_dim % 8 || max_pos < 1))
    return set_last_error(LARA_ERR_BAD_CFG, "rot_dim must be a multiple of 8 up to head_dim, max_pos >= 1");
  if (!(eps >= 0.f)) return set_last_error(LARA_ERR_BAD_CFG, "eps must not be negative");
  if (batch == 0 || n == 0) return LARA_OK;
  if (!q || !k || !q_out || !k_out || (cos_sin && !positions))
    return set_last_error(LARA_ERR_STREAM_DEST, "null pointer");
  if (!aligned(q, 2) || !aligned(k, 2) || !aligned(q_out, 2) || !aligned(k_out, 2) || !aligned(positions, 4) ||
      !aligned(cos_sin, 16) || !aligned(q_weight, 16) || !aligned(k_weight, 16) || !aligned(workspace, 4))
    return set_last_error(LARA_ERR_STREAM_DEST, "cos_sin and the weights must be 16-byte aligned");
  const int alignment = std::min({row_alignment(q, q_sb, batch, q_st, n, q_sh, n_q_heads),
                                  row_alignment(k, k_sb, batch, k_st, n, k_sh, n_kv_heads),
                                  row_alignment(q_out, qo_sb, batch, qo_st, n, qo_sh, n_q_heads),
                                  row_alignment(k_out, ko_sb, batch, ko_st, n, ko_sh, n_kv_heads)});
  NormRopeArgs a{};
  a.q = {q, q_sb, q_st, q_sh};
  a.k = {k, k_sb, k_st, k_sh};
  a.qo = {q_out, qo_sb, qo_st, qo_sh};
  a.ko = {k_out, ko_sb, ko_st, ko_sh};
  const uint32_t tokens = (uint32_t)batch * (uint32_t)n;
  a.hq = n_q_heads;
  a.hkv = n_kv_heads;
  a.n = FastDiv((uint32_t)n);
  a.positions = positions;
  a.cos_sin = cos_sin;
  a.max_pos = max_pos;
  a.rot = cos_sin ? rot_dim : 0;
  a.qw = q_weight;
  a.kw = k_weight;
  a.eps = eps;
  a.status = static_cast<int*>(workspace);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // without a rotation nothing is paired: side by side is the wider access
  const bool inter = interleaved || !cos_sin;
  const cudaError_t e = head_dim == 128 ? (inter ? launch<128, true>(a, tokens, alignment, st) : launch<128, false>(a, tokens, alignment, st))
                                        : (inter ? launch<64, true>(a, tokens, alignment, st) : launch<64, false>(a, tokens, alignment, st));
  if (e != cudaSuccess)
    return set_last_error(LARA_ERR_CUDA, std::string("qk_norm_rope launch: ") + cudaGetErrorString(e));
  return LARA_OK;
}
