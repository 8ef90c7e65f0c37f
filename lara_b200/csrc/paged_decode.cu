// Decode over the paged bf16 cache, with each slot's attention weight gathered
// (lara_gqa_decode_scored) or behind a prefix that the batch shares
// (lara_gqa_decode_shared); declared in include/lara_b200.h.
//
//   s_t = scale log2(e) q.k_t,  o = sum_t 2^(s_t - R) v_t / sum_t 2^(s_t - R)
//   w_t += sum over the group's heads of 2^(s_t - M) / L   (M, L: the whole row's R and sum)
//
// Two launches (of a decode behind a prefix the first is in paged_shared.cu).  The
// first reads every cached row once and leaves partial results (R, l, acc) of each
// unit, a (sequence, kv head), or of the parts that several CTAs take of it; the
// second joins them, and, scoring, turns the scores that the first left into
// weights (G fp32 numbers per token and kv head written and read beside the 4 D
// bytes of its rows: at G = 4, D = 128 6 % of them, against 50 % for reading K twice).
//
// Bound by HBM.  Measured, scored, one state replayed in a graph and, in brackets,
// inputs that change from pass to pass: 64 x 4096 tokens (32 heads on 8) 175 us (180 to
// 184), of which the first launch takes 168 (6.4 TB/s, 0.97 of the copy rate) and the
// second 8 to 16 beside the next call; 524288 tokens (64 heads) 397 us (391 to 404; 351
// and 46); 33 sequences of up to 9000, head_dim 64, 7 heads to a kv head 48 us (48 to
// 51; 30 and 13); 500 tokens 9 us (9).  What is left is in the second launch: a chain of loads per unit,
// and of long contexts scores that L2 no longer holds.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "paged_own.cuh"

namespace lara {

using namespace paged;

namespace {

// Small rings, so that three CTAs share an SM (two with more than eight heads to a unit): 64 x 4096
// tokens 179 us, 188 with two CTAs and rings of three stages; one sequence of 524288 tokens 413 against 404.
template <int D, int NG>
struct Cfg {
  static constexpr int kCtasPerSm = NG == 1 ? 3 : 2;
  using Pass = OwnTokens<D, NG, 4, D == 64 ? 4 : NG == 1 ? 2 : 3, true>;
  static_assert(kCtasPerSm * Pass::C::kWarps <= kMostPerSm);
};

template <int D, int NG>
__global__ void __launch_bounds__(Cfg<D, NG>::Pass::C::kThreads, Cfg<D, NG>::kCtasPerSm)
    own_tokens_kernel(const __grid_constant__ DecodeArgs a) {
  using Pass = typename Cfg<D, NG>::Pass;
  extern __shared__ uint8_t smem_raw[];
  __shared__ typename Pass::Shared shared;
  grid_dependency_wait();
  Pass pass(a, shared);
  pass.totals();
  pass.run(blockIdx.x, gridDim.x, smem_raw + (-smem_addr(smem_raw) & 127));
  allow_dependent_launch();  // not before: the join's blocks would take the room of this grid's
}

// ---- the second launch ----
constexpr int kJoinThreads = 256;
constexpr int kJoinWarps = kJoinThreads / 32;
constexpr int kAhead = 2;      // times four tokens of a thread whose scores are in flight
constexpr int kFewParts = 32;  // parts of a row that one warp joins (more: the block, row after row),
constexpr int kAtOnce = 8;     // from registers, all loads at once: 64 x 4096 181 us without, 177 with

// What a row's result is joined from.
struct Parts {
  long long prefix_row;
  int h, slot0, prefix, all;
};

// Joins the parts of kJoinWarps output rows: a warp to a row, and the rows of many
// parts by the whole block, one after the other.
template <int D>
__device__ __forceinline__ void join_rows(const DecodeArgs& a, int block) {
  constexpr int kLanes = D / 4, kSub = kJoinThreads / kLanes;  // lanes of a row, parts in flight
  __shared__ float4 s_x[kSub][kLanes];
  __shared__ float s_l[kSub];
  __shared__ Parts s_many[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.group;
  const long long rows = (long long)a.batch * a.n_q_heads, row0 = (long long)block * kJoinWarps;
  // part i of a row: of the prefix, then of the unit
  auto ml_of = [&](const Parts& up, int i) {
    return i < up.prefix ? a.prefix_ml + up.prefix_row + (long long)i * a.prefix.rows
                         : a.part_ml + (long long)(up.slot0 + i - up.prefix) * G + up.h;
  };
  auto acc_of = [&](const Parts& up, int i) {
    return i < up.prefix ? a.prefix_acc + (up.prefix_row + (long long)i * a.prefix.rows) * D
                         : a.part_acc + ((long long)(up.slot0 + i - up.prefix) * G + up.h) * D;
  };
  auto largest = [&](const Parts& up) {
    float M = -INFINITY;
    for (int i = lane; i < up.all; i += 32) M = fmaxf(M, __ldcg(ml_of(up, i)).x);
#pragma unroll
    for (int off = 16; off; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
    return M;
  };
  auto add = [](const float2& ml, const float4& y, float M, float& L, float4& x) {
    const float f = ml.x == M ? 1.f : ex2_ftz(ml.x - M);
    L = fmaf(ml.y, f, L);
    x.x = fmaf(y.x, f, x.x);
    x.y = fmaf(y.y, f, x.y);
    x.z = fmaf(y.z, f, x.z);
    x.w = fmaf(y.w, f, x.w);
  };
  // parts i0, i0 + step, ..
  auto sum = [&](const Parts& up, float M, int i0, int step, int at, float& L) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = i0; i < up.all; i += step) {
      const float2 ml = __ldcg(ml_of(up, i));
      const float4 y = __ldcg(reinterpret_cast<const float4*>(acc_of(up, i)) + at);
      add(ml, y, M, L, x);
    }
    return x;
  };
  auto store = [&](long long row, int at, const float4& x, float L) {
    const float inv = L == 0.f ? 0.f : 1.f / L;  // scores of -inf alone: zeros, as the other decodes give
    reinterpret_cast<uint2*>(a.o + row * D)[at] =
        make_uint2(pack2_rn(x.x * inv, x.y * inv), pack2_rn(x.z * inv, x.w * inv));
  };
  {
    const long long row = row0 + warp;
    Parts up{0, 0, 0, 0, 0};
    if (row < rows) {
      const int b = (int)(row / a.n_q_heads), hq = (int)(row % a.n_q_heads);
      up.h = hq % G;
      // what there may be of parts, whatever the length is: one round of loads for all
      const int raw = __ldcg(a.lens + b);
      UnitParts unit = a.units[b * a.index.n_kv_heads + hq / G], prefix{0, 0};
      int in = 0;
      if (a.shared_tokens > 0) {
        const int seqs = a.prefix.seqs * (a.prefix.rows / 128);  // of a unit of the prefix
        prefix = a.prefix_units[hq / G * a.prefix.units + b / seqs];
        in = b % seqs;
      }
      const int len = (int)min((long long)raw, a.index.capacity());
      const Own own = own_tokens(a, len);
      if (own.start > 0) {
        up.prefix = up.all = prefix.parts;
        const int tile = in / a.prefix.seqs;
        up.prefix_row = (long long)prefix.slot0 * a.prefix.rows + tile * 128 + in % a.prefix.seqs * G + up.h;
      }
      if (own.len > 0) {
        up.slot0 = unit.slot0;
        up.all += unit.parts;
      }
      const int at = lane % kLanes;
      if (len <= 0) {
        if (lane < kLanes) reinterpret_cast<uint2*>(a.o + row * D)[at] = make_uint2(0, 0);
      } else if (up.all <= kAtOnce) {
        float2 ml[kAtOnce];
        float4 y[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          ml[i] = make_float2(-INFINITY, 0.f);
          y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (i < up.all) {
            ml[i] = __ldcg(ml_of(up, i));
            y[i] = __ldcg(reinterpret_cast<const float4*>(acc_of(up, i)) + at);
          }
        }
        float M = -INFINITY, L = 0.f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) M = fmaxf(M, ml[i].x);
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
          if (i < up.all) add(ml[i], y[i], M, L, x);
        if (lane < kLanes) store(row, at, x, L);
      } else if (up.all <= kFewParts) {
        float L = 0.f;
        const float4 x = sum(up, largest(up), 0, 1, at, L);
        if (lane < kLanes) store(row, at, x, L);
      }
    }
    if (lane == 0) s_many[warp] = up;
  }
  __syncthreads();
  for (int r = 0; r < kJoinWarps; ++r) {
    const Parts up = s_many[r];
    if (up.all <= kFewParts) continue;
    const int sub = threadIdx.x / kLanes, at = threadIdx.x % kLanes;
    float L = 0.f;
    const float4 part = sum(up, largest(up), sub, kSub, at, L);
    s_x[sub][at] = part;
    if (at == 0) s_l[sub] = L;
    __syncthreads();
    if (threadIdx.x < kLanes) {
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      L = 0.f;
#pragma unroll
      for (int i = 0; i < kSub; ++i) {
        const float4 y = s_x[i][at];
        L += s_l[i];
        x.x += y.x;
        x.y += y.y;
        x.z += y.z;
        x.w += y.w;
      }
      store(row0 + r, at, x, L);
    }
    __syncthreads();
  }
}

// Adds the weights of an equal run of all groups, four tokens to a thread, from its end to its
// start: the scores written last are still in L2, and those read are dropped there, which spares
// writing them to memory.
__device__ __forceinline__ void add_weights(const DecodeArgs& a, int block, int blocks) {
  __shared__ float2 s_ml[16];  // each head's (M, 1 / L)
  __shared__ int s_seq;
  __shared__ long long s_first[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.group, hkv = a.index.n_kv_heads, log2 = a.index.page_log2;
  const long long total = __ldcg(a.seq_groups + a.batch) * hkv;
  const long long room = min(total, a.score_groups);
  if (room < total && block == 0 && threadIdx.x == 0) atomicOr(a.status, kDevScoreRoom);
  const long long per = (room + blocks - 1) / blocks;
  const long long lo = block * per, hi = min(room, lo + per);
  if (lo >= hi) return;
  for (int b = threadIdx.x; b < a.batch; b += kJoinThreads) {  // the sequence with group hi - 1
    const long long from = __ldcg(a.seq_groups + b), to = __ldcg(a.seq_groups + b + 1);
    if (from * hkv < hi && hi <= to * hkv) {
      s_seq = b;
      s_first[0] = from;
      s_first[1] = to;
    }
  }
  __syncthreads();
  int b = s_seq;
  long long first = s_first[0];
  int groups = (int)(s_first[1] - first);
  int kvh = (int)quotient(hi - 1 - first * hkv, groups);
  long long at = first * hkv + (long long)kvh * groups;  // the unit's first group
  while (true) {
    const UnitParts up = a.units[b * hkv + kvh];
    const int len = (int)min((long long)__ldcg(a.lens + b), a.index.capacity());
    const int t0 = (int)(max(lo, at) - at) * kGroup, t1 = min((int)(min(hi, at + groups) - at) * kGroup, len);
    const int32_t* const pages = a.index.block_table + (long long)b * a.index.pages_per_seq;
    auto page_of = [&](int t) { return t < t1 ? __ldg(pages + (t >> log2)) : -1; };
    constexpr int kStep = 4 * kJoinThreads;
    const int last = t0 + (max(0, t1 - t0 - 1)) / (kStep * kAhead) * (kStep * kAhead);
    int page[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) page[j] = page_of(last + kStep * j + 4 * threadIdx.x);
    for (int h = warp; h < G; h += kJoinWarps) {
      float M = -INFINITY, L = 0.f;
      auto join = [&](float m, float l) {
        const float to = fmaxf(M, m);
        L = L * (M == to ? 1.f : ex2_ftz(M - to)) + l * (m == to ? 1.f : ex2_ftz(m - to));
        M = to;
      };
      for (int p = lane; p < up.parts; p += 32) {
        const float2 x = __ldcg(a.part_ml + (long long)(up.slot0 + p) * G + h);
        join(x.x, x.y);
      }
#pragma unroll
      for (int off = 16; off; off >>= 1)
        join(__shfl_xor_sync(0xffffffffu, M, off), __shfl_xor_sync(0xffffffffu, L, off));
      if (lane == 0) s_ml[h] = L == 0.f ? make_float2(0.f, 0.f) : make_float2(M, 1.f / L);  // scores of -inf alone
    }
    __syncthreads();
    for (int base = last; base >= t0; base -= kStep * kAhead) {
      const int t = base + 4 * threadIdx.x;
      const float4* s[kAhead];
      long long row[kAhead];
      float4 w[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int x = t + kStep * j;
        const bool there = x < t1 && (unsigned)page[j] < (unsigned)a.index.num_pages;  // else flagged before
        row[j] = there ? (((long long)page[j] * hkv + kvh) << log2) + (x & ((1 << log2) - 1)) : -1;
        s[j] = reinterpret_cast<const float4*>(
            a.scores + (there ? (at + x / kGroup) * (G * kGroup) + x % kGroup : 0));
        w[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (there) w[j] = __ldcg(reinterpret_cast<const float4*>(a.w_in + row[j]));
        page[j] = base > t0 ? page_of(x - kStep * kAhead) : -1;
      }
      float4 sum[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) sum[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int i = 0; i < G; ++i) {
        const float2 x = s_ml[i];
        float4 y[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) y[j] = __ldcg(s[j] + i * (kGroup / 4));
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          sum[j].x = fmaf(ex2_ftz(y[j].x - x.x), x.y, sum[j].x);
          sum[j].y = fmaf(ex2_ftz(y[j].y - x.x), x.y, sum[j].y);
          sum[j].z = fmaf(ex2_ftz(y[j].z - x.x), x.y, sum[j].z);
          sum[j].w = fmaf(ex2_ftz(y[j].w - x.x), x.y, sum[j].w);
        }
      }
      __syncwarp();  // every lane's scores are read: what is discarded may be written at once
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (row[j] < 0) continue;
        if (lane % 8 == 0) {  // a group's line, which this warp alone has read, eight lanes together
#pragma unroll 1
          for (int i = 0; i < G; ++i)
            asm volatile("discard.global.L2 [%0], 128;" ::"l"(s[j] + i * (kGroup / 4)), "f"(sum[j].x) : "memory");
        }
        const int left = t1 - (t + kStep * j);
        const float4 v =
            make_float4(w[j].x + sum[j].x, w[j].y + sum[j].y, w[j].z + sum[j].z, w[j].w + sum[j].w);
        float* const to = a.w_out + row[j];
        if (left >= 4) {
          *reinterpret_cast<float4*>(to) = v;
        } else {
          to[0] = v.x;
          if (left > 1) to[1] = v.y;
          if (left > 2) to[2] = v.z;
        }
      }
    }
    if (at <= lo) return;
    if (--kvh < 0) {
      kvh = hkv - 1;
      do {
        --b;
        first = __ldcg(a.seq_groups + b);
        groups = (int)(__ldcg(a.seq_groups + b + 1) - first);
      } while (groups == 0);
    }
    at -= groups;
    __syncthreads();  // s_ml is free again
  }
}

// The blocks of weights, of one wave, come first: they take longer than the others.
template <int D, bool kScored>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ DecodeArgs a, int weight_blocks) {
  allow_dependent_launch();
  grid_dependency_wait();
  if constexpr (kScored) {
    if ((int)blockIdx.x < weight_blocks) {
      add_weights(a, blockIdx.x, weight_blocks);
      return;
    }
  }
  join_rows<D>(a, blockIdx.x - weight_blocks);
}

// Workspace: status word | units | partial results | scores, or the prefix's results.
struct Layout {
  size_t units_off, seq_off, ml_off, acc_off, scores_off, prefix_units_off, prefix_ml_off, prefix_acc_off, total;
  long long score_groups;
};

Layout layout(int batch, int n_kv_heads, int group, int head_dim, long long score_tokens, bool shared) {
  const size_t units = (size_t)batch * n_kv_heads, sms = std::max(1, device_sm_count());
  const size_t slots = units + kMostPerSm * sms;
  Layout w;
  w.units_off = kStatusBytes;
  w.seq_off = w.units_off + up256(units * sizeof(UnitParts));
  w.ml_off = w.seq_off + up256(((size_t)batch + 1) * sizeof(long long));
  w.acc_off = w.ml_off + up256(slots * group * sizeof(float2));
  w.scores_off = w.acc_off + up256(slots * group * head_dim * sizeof(float));
  // every sequence's scores start in a group of their own
  w.score_groups = score_tokens ? (score_tokens / kGroup + batch) * n_kv_heads : 0;
  w.prefix_units_off = w.scores_off + up256((size_t)w.score_groups * kGroup * group * sizeof(float));
  const PrefixPlan plan = prefix_plan(batch, group);
  const size_t prefix_units = shared ? (size_t)plan.units * n_kv_heads : 0;
  const size_t prefix_rows = shared ? (prefix_units + sms) * plan.rows : 0;
  w.prefix_ml_off = w.prefix_units_off + up256(prefix_units * sizeof(UnitParts));
  w.prefix_acc_off = w.prefix_ml_off + up256(prefix_rows * sizeof(float2));
  w.total = w.prefix_acc_off + up256(prefix_rows * head_dim * sizeof(float));
  return w;
}

// The second launch: weights, where there are scores, and the join.
template <int D, bool kScored>
cudaError_t launch_join(const DecodeArgs& a, cudaStream_t stream) {
  DecodeArgs args = a;
  const long long rows = (long long)a.batch * a.n_q_heads;
  const long long groups = (long long)a.batch * a.index.n_kv_heads * ((a.index.capacity() + kGroup - 1) / kGroup);
  int weight_blocks = kScored ? (int)std::min<long long>(device_sm_count() * 3, (groups + 15) / 16) : 0;
  const int blocks = weight_blocks + (int)((rows + kJoinWarps - 1) / kJoinWarps);
  void* p[] = {&args, &weight_blocks};
  return launch_with_pdl(reinterpret_cast<const void*>(&join_kernel<D, kScored>), dim3((unsigned)blocks),
                         dim3(kJoinThreads), p, 0, stream);
}

template <int D, int NG>
cudaError_t launch_scored(const DecodeArgs& a, cudaStream_t stream) {
  using Pass = typename Cfg<D, NG>::Pass;
  using C = typename Pass::C;
  const void* fn = reinterpret_cast<const void*>(&own_tokens_kernel<D, NG>);
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
  const long long units = (long long)a.batch * a.index.n_kv_heads;
  const long long tiles = units * ((a.index.capacity() + kTile - 1) / kTile);
  const long long ctas = std::min<long long>(device_sm_count() * Cfg<D, NG>::kCtasPerSm,
                                             std::max(units, (tiles + C::kMinTiles - 1) / C::kMinTiles));
  DecodeArgs args = a;
  void* p[] = {&args};
  const cudaError_t e = launch_with_pdl(fn, dim3((unsigned)ctas), dim3(C::kThreads), p, C::kSmemBytes, stream);
  return e == cudaSuccess ? launch_join<D, true>(a, stream) : e;
}

}  // namespace

namespace paged {

int check_paged_pool(const void* k_pages, const void* v_pages, const void* block_table, int n_kv_heads, int head_dim,
                     int page_size, int pages_per_seq, int num_pages, int batch, PoolIndex* index) {
  if (head_dim != 64 && head_dim != 128) return set_last_error(LARA_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  if (page_size < 16 || page_size > 65536 || (page_size & (page_size - 1)))
    return set_last_error(LARA_ERR_BAD_CFG, "page_size must be a power of two in [16, 65536]");
  if (batch < 0 || batch > 65535) return set_last_error(LARA_ERR_BAD_CFG, "batch must be in [0, 65535]");
  if (n_kv_heads < 1 || n_kv_heads > 65535 || num_pages < 1 || pages_per_seq < 1 ||
      (long long)pages_per_seq * page_size > 0x3fffffffll || (long long)batch * n_kv_heads > 0x3fffffffll ||
      (double)batch * n_kv_heads * pages_per_seq * page_size > 0x1p40)
    return set_last_error(LARA_ERR_BAD_CFG,
                          "bad paged-cache geometry (at most 2^30 - 1 tokens a sequence, 2^40 rows in all)");
  if (batch == 0) return LARA_OK;
  if (!k_pages || !v_pages || !block_table) return set_last_error(LARA_ERR_STREAM_DEST, "null pointer");
  if (!aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(block_table, 4))
    return set_last_error(LARA_ERR_STREAM_DEST, "k_pages and v_pages must be 16-byte aligned");
  index->block_table = static_cast<const int32_t*>(block_table);
  index->pages_per_seq = pages_per_seq;
  index->page_log2 = __builtin_ctz(page_size);
  index->num_pages = num_pages;
  index->n_kv_heads = n_kv_heads;
  return LARA_OK;
}

int check_weights(const float* in, const float* out, int n_kv_heads, int page_size, int num_pages) {
  if (!in || !out) return set_last_error(LARA_ERR_STREAM_DEST, "null pointer");
  if (!aligned(in, 16) || !aligned(out, 16))
    return set_last_error(LARA_ERR_STREAM_DEST, "weights must be 16-byte aligned");
  if (in != out && kvq::overlap(in, out, (size_t)num_pages * n_kv_heads * page_size * 4))
    return set_last_error(LARA_ERR_STREAM_DEST, "weights_out must be weights or lie apart from them");
  return LARA_OK;
}

}  // namespace paged

}  // namespace lara

using namespace lara;

namespace {

// The checks and arguments that the two decodes have in common.
int decode_args(DecodeArgs& a, const uint16_t* q, const uint16_t* k_pages, const uint16_t* v_pages,
                const int32_t* block_table, const int32_t* seq_lens, uint16_t* o, int batch, int n_q_heads,
                int n_kv_heads, int head_dim, int page_size, int pages_per_seq, int num_pages, float scale,
                const void* workspace) {
  if (const int rc = check_paged_pool(k_pages, v_pages, block_table, n_kv_heads, head_dim, page_size, pages_per_seq,
                                      num_pages, batch, &a.index))
    return rc;
  if (n_q_heads < 1 || n_q_heads % n_kv_heads)
    return set_last_error(LARA_ERR_BAD_CFG, "n_q_heads must be a multiple of n_kv_heads");
  if (n_q_heads / n_kv_heads > 16)
    return set_last_error(LARA_ERR_UNSUPPORTED, "groups of at most 16 query heads per kv head");
  if (!(scale > 0.f) || !std::isfinite(scale))
    return set_last_error(LARA_ERR_BAD_CFG, "scale must be positive and finite");
  if (batch == 0) return LARA_OK;
  if (!q || !seq_lens || !o || !workspace) return set_last_error(LARA_ERR_STREAM_DEST, "null pointer");
  if (!aligned(q, 16) || !aligned(o, 16) || !aligned(seq_lens, 4) || !aligned(workspace, 256))
    return set_last_error(LARA_ERR_STREAM_DEST, "q and o must be 16-byte aligned, the workspace 256-byte");
  a.q = q;
  a.k = k_pages;
  a.v = v_pages;
  a.lens = seq_lens;
  a.o = o;
  a.batch = batch;
  a.n_q_heads = n_q_heads;
  a.group = n_q_heads / n_kv_heads;
  a.scale_log2 = scale * 1.4426950408889634f;
  return LARA_OK;
}

void place(DecodeArgs& a, const Layout& w, void* workspace) {
  char* base = static_cast<char*>(workspace);
  a.status = reinterpret_cast<int*>(base);
  a.units = reinterpret_cast<UnitParts*>(base + w.units_off);
  a.seq_groups = reinterpret_cast<long long*>(base + w.seq_off);
  a.part_ml = reinterpret_cast<float2*>(base + w.ml_off);
  a.part_acc = reinterpret_cast<float*>(base + w.acc_off);
  a.scores = reinterpret_cast<float*>(base + w.scores_off);
  a.prefix_units = reinterpret_cast<UnitParts*>(base + w.prefix_units_off);
  a.prefix_ml = reinterpret_cast<float2*>(base + w.prefix_ml_off);
  a.prefix_acc = reinterpret_cast<float*>(base + w.prefix_acc_off);
  a.score_groups = w.score_groups;
}

// Tokens whose scores a call can leave: those of every page its tables can name.
long long score_tokens(int batch, int page_size, int pages_per_seq, int num_pages) {
  return std::min<long long>((long long)batch * pages_per_seq, num_pages) * page_size;
}

}  // namespace

extern "C" size_t lara_decode_scored_workspace_bytes(int batch, int n_q_heads, int n_kv_heads, int head_dim,
                                                     int page_size, int pages_per_seq, int num_pages) {
  if (batch < 1 || n_q_heads < 1 || n_kv_heads < 1 || head_dim < 1 || page_size < 1 || pages_per_seq < 1 ||
      num_pages < 1)
    return 0;
  return layout(batch, n_kv_heads, (n_q_heads + n_kv_heads - 1) / n_kv_heads, head_dim,
                score_tokens(batch, page_size, pages_per_seq, num_pages), false)
      .total;
}

extern "C" int lara_gqa_decode_scored(const uint16_t* q, const uint16_t* k_pages, const uint16_t* v_pages,
                                      const float* weights, float* weights_out, const int32_t* block_table,
                                      const int32_t* seq_lens, uint16_t* o, int batch, int n_q_heads, int n_kv_heads,
                                      int head_dim, int page_size, int pages_per_seq, int num_pages, float scale,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  LARA_NVTX("lara_gqa_decode_scored");
  DecodeArgs a{};
  if (const int rc = decode_args(a, q, k_pages, v_pages, block_table, seq_lens, o, batch, n_q_heads, n_kv_heads,
                                 head_dim, page_size, pages_per_seq, num_pages, scale, workspace))
    return rc;
  if (batch == 0) return LARA_OK;
  if (const int rc = check_weights(weights, weights_out, n_kv_heads, page_size, num_pages)) return rc;
  const Layout w = layout(batch, n_kv_heads, a.group, head_dim,
                          score_tokens(batch, page_size, pages_per_seq, num_pages), false);
  if (workspace_bytes < w.total) return set_last_error(LARA_ERR_RESULT_LEN, "scored decode workspace too small");
  place(a, w, workspace);
  a.w_in = weights;
  a.w_out = weights_out;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = head_dim == 128 ? (a.group <= 8 ? launch_scored<128, 1>(a, st) : launch_scored<128, 2>(a, st))
                                        : (a.group <= 8 ? launch_scored<64, 1>(a, st) : launch_scored<64, 2>(a, st));
  if (e != cudaSuccess)
    return set_last_error(LARA_ERR_CUDA, std::string("scored decode launch: ") + cudaGetErrorString(e));
  return LARA_OK;
}

extern "C" size_t lara_decode_shared_workspace_bytes(int batch, int n_q_heads, int n_kv_heads, int head_dim) {
  if (batch < 1 || n_q_heads < 1 || n_kv_heads < 1 || head_dim < 1) return 0;
  const int group = std::min(16, (n_q_heads + n_kv_heads - 1) / n_kv_heads);
  return layout(batch, n_kv_heads, group, head_dim, 0, true).total;
}

extern "C" int lara_gqa_decode_shared(const uint16_t* q, const uint16_t* k_pages, const uint16_t* v_pages,
                                      const int32_t* block_table, const int32_t* seq_lens, uint16_t* o, int batch,
                                      int n_q_heads, int n_kv_heads, int head_dim, int page_size, int pages_per_seq,
                                      int num_pages, int shared_pages, float scale, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  LARA_NVTX("lara_gqa_decode_shared");
  DecodeArgs a{};
  if (const int rc = decode_args(a, q, k_pages, v_pages, block_table, seq_lens, o, batch, n_q_heads, n_kv_heads,
                                 head_dim, page_size, pages_per_seq, num_pages, scale, workspace))
    return rc;
  if (shared_pages < 0 || shared_pages > pages_per_seq)
    return set_last_error(LARA_ERR_BAD_CFG, "shared_pages must be in [0, pages_per_seq]");
  if (batch == 0) return LARA_OK;
  const Layout w = layout(batch, n_kv_heads, a.group, head_dim, 0, true);
  if (workspace_bytes < w.total) return set_last_error(LARA_ERR_RESULT_LEN, "shared decode workspace too small");
  place(a, w, workspace);
  a.shared_tokens = shared_pages * page_size;
  a.prefix = prefix_plan(batch, a.group);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = shared_launch(a, head_dim, st);
  if (e == cudaSuccess) e = head_dim == 128 ? launch_join<128, false>(a, st) : launch_join<64, false>(a, st);
  if (e != cudaSuccess)
    return set_last_error(LARA_ERR_CUDA, std::string("shared decode launch: ") + cudaGetErrorString(e));
  return LARA_OK;
}
