// GQA decode over the paged 8-bit KV pool (declared in include/lara_b200.h).
//
//   o[b,h,:] = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q.k_t - m),
//   k_t = ks_t ck_t, v_t = vs_t cv_t  (codes c, one fp32 scale per row)
//
// One CTA per (sequence, query head); a warp takes every kWarps-th token, a
// lane D / 32 dims, with a running maximum and sum in fp32; the warps are
// joined at the end.
#include <cmath>

#include "kvq.cuh"

namespace lara {

using namespace kvq;

namespace {

constexpr int kWarps = 8;
constexpr size_t kStatusBytes = 256;

struct KvqDecodeArgs {
  lara_kvq_pool pool;
  PoolIndex index;
  const uint16_t* q;
  const int32_t* lens;
  uint16_t* o;
  int n_q_heads;
  float scale_log2;
  int* status;
};

template <int D, int FMT>
__global__ void __launch_bounds__(kWarps * 32) kvq_decode_kernel(const __grid_constant__ KvqDecodeArgs a) {
  constexpr int V = D / 32;
  __shared__ float sm[kWarps], sl[kWarps], sacc[kWarps][D];
  const int h = blockIdx.x, b = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int kvh = h / (a.n_q_heads / a.pool.n_kv_heads);
  int len = a.lens[b];
  if (len < 0 || len > a.index.capacity()) {
    if (threadIdx.x == 0) atomicOr(a.status, kDevBadLength);
    len = len < 0 ? 0 : (int)a.index.capacity();
  }
  const long long qrow = ((long long)b * a.n_q_heads + h) * D;
  float q[V], acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    q[j] = __uint_as_float((uint32_t)a.q[qrow + lane * V + j] << 16);
    acc[j] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int t = warp; t < len; t += kWarps) {
    long long row = a.index.row(b, kvh, t, a.status);
    if (row < 0) row = 0;
    uint32_t ck = 0, cv = 0;
    if constexpr (V == 4) {
      ck = *reinterpret_cast<const uint32_t*>(a.pool.k_codes + row * D + lane * V);
      cv = *reinterpret_cast<const uint32_t*>(a.pool.v_codes + row * D + lane * V);
    } else {
      ck = *reinterpret_cast<const uint16_t*>(a.pool.k_codes + row * D + lane * V);
      cv = *reinterpret_cast<const uint16_t*>(a.pool.v_codes + row * D + lane * V);
    }
    float kf[4], vf[4];
    codes_to_f32<FMT>(ck, kf);
    codes_to_f32<FMT>(cv, vf);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) s = fmaf(q[j], kf[j], s);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    s = s * a.pool.k_scales[row] * a.scale_log2;
    const float mn = fmaxf(m, s);
    const float corr = exp2f(m - mn), p = exp2f(s - mn);
    const float pv = p * a.pool.v_scales[row];
    m = mn;
    l = fmaf(l, corr, p);
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = fmaf(acc[j], corr, pv * vf[j]);
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) sacc[warp][lane * V + j] = acc[j];
  __syncthreads();
  if (threadIdx.x < D) {
    float M = -INFINITY, L = 0.f, x = 0.f;
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm[w]);
    for (int w = 0; w < kWarps; ++w) {
      if (sm[w] == -INFINITY) continue;
      const float c = exp2f(sm[w] - M);
      L = fmaf(sl[w], c, L);
      x = fmaf(sacc[w][threadIdx.x], c, x);
    }
    a.o[qrow + threadIdx.x] = (uint16_t)pack2_rn(len > 0 ? x / L : 0.f, 0.f);
  }
}

}  // namespace

}  // namespace lara

using namespace lara;

extern "C" size_t lara_kvq_decode_workspace_bytes(int batch, int n_q_heads, int n_kv_heads, int head_dim) {
  if (batch < 1 || n_q_heads < 1 || n_kv_heads < 1 || head_dim < 1) return 0;
  return kStatusBytes;
}

extern "C" int lara_gqa_decode_kvq(const uint16_t* q, const lara_kvq_pool* pool, const int32_t* block_table,
                                   int pages_per_seq, const int32_t* seq_lens, uint16_t* o, int batch, int n_q_heads,
                                   float scale, void* workspace, size_t workspace_bytes, void* stream) {
  LARA_NVTX("lara_gqa_decode_kvq");
  KvqDecodeArgs a{};
  if (const int rc = check_pool(pool, block_table, pages_per_seq, &a.index)) return rc;
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
  if (workspace_bytes < lara_kvq_decode_workspace_bytes(batch, n_q_heads, pool->n_kv_heads, pool->head_dim))
    return set_last_error(LARA_ERR_RESULT_LEN, "decode workspace too small");
  a.pool = *pool;
  a.q = q;
  a.lens = seq_lens;
  a.o = o;
  a.n_q_heads = n_q_heads;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.status = static_cast<int*>(workspace);
  const dim3 grid(n_q_heads, batch);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define LARA_CASE(d, f) \
  if (pool->head_dim == d && pool->format == f) kvq_decode_kernel<d, f><<<grid, kWarps * 32, 0, st>>>(a);
  LARA_CASE(128, LARA_KVQ_INT8) LARA_CASE(128, LARA_KVQ_FP8_E4M3)
  LARA_CASE(64, LARA_KVQ_INT8) LARA_CASE(64, LARA_KVQ_FP8_E4M3)
#undef LARA_CASE
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    return set_last_error(LARA_ERR_CUDA, std::string("kvq decode launch: ") + cudaGetErrorString(e));
  return LARA_OK;
}
