// RMS norm of query and key heads with the position rotation, in one pass
// (declared in include/lara_b200.h).  The rotation's dim pairs are those of
// hw/rtl/core/rope_engine.sv:1-11 (interleaved) or half a rotation apart.
//
//   y = x w / sqrt(mean(x^2) + eps);  (y_a, y_b) -> (y_a c - y_b s, y_a s + y_b c)
//
// Bound by HBM: every head is read and written once (4 D bytes), the table row
// of a token once from HBM (4 rot bytes) and from L2 after that.  D / 8 lanes
// hold a head in registers between the load and the store; a lane group takes
// kHeads heads of one token, so it loads its cosines, sines and weights once
// and has kHeads loads in flight.
#include "kvq.cuh"

namespace lara {

using namespace kvq;

namespace {

constexpr int kHeads = 4;
constexpr int kThreads = 128;

struct NormRopeArgs {
  Heads<const uint16_t> q, k;
  Heads<uint16_t> qo, ko;
  int n, hq, heads, groups_per_token;
  long long groups;
  const int32_t* positions;
  const float* cos_sin;
  int max_pos, rot, interleaved;
  const uint16_t* qw;
  const uint16_t* kw;
  float eps;
  int* status;
};

template <int D, bool kVec>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const __grid_constant__ NormRopeArgs a) {
  constexpr int kLanes = D / 8;
  const long long gid = ((long long)blockIdx.x * kThreads + threadIdx.x) / kLanes;
  const int l = threadIdx.x % kLanes;
  const bool active = gid < a.groups;
  const long long g = active ? gid : a.groups - 1;
  const long long tok = g / a.groups_per_token;
  const int h0 = (int)(g % a.groups_per_token) * kHeads;
  const int b = (int)(tok / a.n), t = (int)(tok % a.n);
  const LaneDims ld(l, a.cos_sin ? a.rot : 0, a.interleaved);

  float x[kHeads][8];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = min(h0 + i, a.heads - 1);
    load8<kVec>(h < a.hq ? a.q.row(b, t, h) : a.k.row(b, t, h - a.hq), ld.o0, ld.o1, x[i]);
  }
  float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (ld.rotated) {
    int pos = a.positions[tok];
    if (pos < 0 || pos >= a.max_pos) {
      if (a.status) atomicOr(a.status, kDevBadPosition);
      pos = pos < 0 ? 0 : a.max_pos - 1;
    }
    const float* row = a.cos_sin + (long long)pos * a.rot + 4 * l;
    c = *reinterpret_cast<const float4*>(row);
    s = *reinterpret_cast<const float4*>(row + a.rot / 2);
  }
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = h0 + i;
    if (a.qw) {
      float w[8];
      load8<true>(h < a.hq ? a.qw : a.kw, ld.o0, ld.o1, w);
      norm_row<D>(x[i], w, a.eps);
    }
    if (ld.rotated) rotate_row(x[i], c, s, a.interleaved);
    if (active && h < a.heads) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = pack2_rn(x[i][2 * j], x[i][2 * j + 1]);
      store8<kVec>(h < a.hq ? a.qo.row(b, t, h) : a.ko.row(b, t, h - a.hq), ld.o0, ld.o1, w);
    }
  }
}

// 8-byte accesses: the base and every stride that is taken (an extent of 1
// takes none).
bool vec_ok(const void* p, long long sb, int batch, long long st, int n, long long sh, int heads) {
  return aligned(p, 8) && (((batch > 1 ? sb : 0) | (n > 1 ? st : 0) | (heads > 1 ? sh : 0)) & 3) == 0;
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
  if (batch < 0 || n < 0 || n_q_heads < 1 || n_kv_heads < 1 || (long long)batch * n > 0x7fffffffll ||
      (long long)n_q_heads + n_kv_heads > 65535)
    return set_last_error(LARA_ERR_BAD_CFG, "bad geometry: batch, n >= 0 and head counts >= 1");
  if (!q_weight != !k_weight) return set_last_error(LARA_ERR_BAD_CFG, "q_weight and k_weight go together");
  if (!q_weight && !cos_sin) return set_last_error(LARA_ERR_BAD_CFG, "neither norm weights nor a rotation table");
  if (cos_sin && (rot_dim < 8 || rot_dim > head_dim || rot_dim % 8 || max_pos < 1))
    return set_last_error(LARA_ERR_BAD_CFG, "rot_dim must be a multiple of 8 up to head_dim, max_pos >= 1");
  if (!(eps >= 0.f)) return set_last_error(LARA_ERR_BAD_CFG, "eps must not be negative");
  if (batch == 0 || n == 0) return LARA_OK;
  if (!q || !k || !q_out || !k_out || (cos_sin && !positions))
    return set_last_error(LARA_ERR_STREAM_DEST, "null pointer");
  if (!aligned(q, 2) || !aligned(k, 2) || !aligned(q_out, 2) || !aligned(k_out, 2) || !aligned(positions, 4) ||
      !aligned(cos_sin, 16) || !aligned(q_weight, 8) || !aligned(k_weight, 8) || !aligned(workspace, 4))
    return set_last_error(LARA_ERR_STREAM_DEST, "cos_sin must be 16-byte aligned, the weights 8-byte");
  const bool vec = vec_ok(q, q_sb, batch, q_st, n, q_sh, n_q_heads) && vec_ok(k, k_sb, batch, k_st, n, k_sh, n_kv_heads) &&
                   vec_ok(q_out, qo_sb, batch, qo_st, n, qo_sh, n_q_heads) &&
                   vec_ok(k_out, ko_sb, batch, ko_st, n, ko_sh, n_kv_heads);
  NormRopeArgs a{};
  a.q = {q, q_sb, q_st, q_sh};
  a.k = {k, k_sb, k_st, k_sh};
  a.qo = {q_out, qo_sb, qo_st, qo_sh};
  a.ko = {k_out, ko_sb, ko_st, ko_sh};
  a.n = n;
  a.hq = n_q_heads;
  a.heads = n_q_heads + n_kv_heads;
  a.groups_per_token = (a.heads + kHeads - 1) / kHeads;
  a.groups = (long long)batch * n * a.groups_per_token;
  a.positions = positions;
  a.cos_sin = cos_sin;
  a.max_pos = max_pos;
  a.rot = cos_sin ? rot_dim : 0;
  a.interleaved = interleaved;
  a.qw = q_weight;
  a.kw = k_weight;
  a.eps = eps;
  a.status = static_cast<int*>(workspace);
  const long long per_block = kThreads / (head_dim / 8);
  const long long blocks = (a.groups + per_block - 1) / per_block;
  if (blocks > 0x7fffffffll) return set_last_error(LARA_ERR_BAD_CFG, "too many heads for one launch");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 128) {
    if (vec) qk_norm_rope_kernel<128, true><<<(unsigned)blocks, kThreads, 0, st>>>(a);
    else qk_norm_rope_kernel<128, false><<<(unsigned)blocks, kThreads, 0, st>>>(a);
  } else {
    if (vec) qk_norm_rope_kernel<64, true><<<(unsigned)blocks, kThreads, 0, st>>>(a);
    else qk_norm_rope_kernel<64, false><<<(unsigned)blocks, kThreads, 0, st>>>(a);
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    return set_last_error(LARA_ERR_CUDA, std::string("qk_norm_rope launch: ") + cudaGetErrorString(e));
  return LARA_OK;
}
