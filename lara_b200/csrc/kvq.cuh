// Rows of the 8-bit KV pool and of the q/k head pass (sm_100a).
//
// A row is the D values of one (token, head).  D / 16 lanes hold it, sixteen
// values each, and reduce over it with shuffles.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "../../include/lara_b200.h"
#include "common.cuh"
#include "lara_internal.h"

namespace lara {
namespace kvq {

// A strided [batch][token][head][D] bf16 tensor; strides in elements.
template <typename T>
struct Heads {
  T* p;
  long long sb, st, sh;
  __device__ __forceinline__ T* row(int b, int t, int h) const { return p + b * sb + t * st + h * sh; }
};

// Round to nearest even; NaN stays NaN (the reference packer's carry could
// turn a NaN's payload over, and a NaN row has to read as one).
__device__ __forceinline__ uint32_t pack2_rn(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return reinterpret_cast<const uint32_t&>(v);
}

// Two fp32 values that one instruction works on.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)),
        "l"(reinterpret_cast<const unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)));
  return d;
}

// n / d for 0 <= n < 2^31 by one multiplication: with s = 31 + ceil(log2 d) and
// m = floor(2^s / d) + 1, n m / 2^s exceeds n / d by less than 1 / d.
struct FastDiv {
  uint32_t d, m, shift;
  FastDiv() = default;
  explicit FastDiv(uint32_t divisor) : d(divisor), m(0), shift(0) {
    if (d > 1) {
      uint32_t lg = 0;
      while ((1ull << lg) < d) ++lg;
      shift = lg - 1;
      m = (uint32_t)((1ull << (31 + lg)) / d + 1);
    }
  }
  __device__ __forceinline__ uint32_t div(uint32_t n, uint32_t& rest) const {
    const uint32_t q = d > 1 ? __umulhi(n, m) >> shift : n;
    rest = n - q * d;
    return q;
  }
};

// A lane's 32 bytes in one access.
__device__ __forceinline__ void load32(const void* p, uint32_t w[8]) {
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void store32(void* p, const uint32_t w[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// How the q/k pass holds a head: D / 2W lanes, 2W dims each (W = 8, or 4 where
// rot or the addresses are not so divisible), kept as W rotation pairs: a[j]
// and b[j] make pair W * lane + j of the table.  Pairs (2i, 2i+1) lie side by
// side in memory; pairs (i, i + rot/2) meet in one lane because the first
// rot / 2W lanes take W dims of each half, so the rotation needs no exchange.
// Lanes past rot hold 2W dims in a row and do not rotate.
template <int W>
struct HeadLane {
  int o0, o1;      // the lane's two runs of W dims
  bool rotated;
  __device__ __forceinline__ HeadLane(int lane, int rot, bool interleaved) {
    rotated = 2 * W * lane < rot;
    const bool split = rotated && !interleaved;
    o0 = split ? W * lane : 2 * W * lane;
    o1 = split ? rot / 2 + W * lane : 2 * W * lane + W;
  }
};

// The lane's values: a[i] = (x_a of pairs 2i, 2i + 1), b alike.
template <int W>
struct Pairs {
  float2 a[W / 2], b[W / 2];
};

// The lane's 2W values as words in memory order: run o0, then run o1.
template <int W, bool kInter, bool kVec>
__device__ __forceinline__ void load_words(const uint16_t* row, const HeadLane<W>& ld, uint32_t w[W]) {
  if constexpr (kVec && kInter && W == 8) {
    load32(row + ld.o0, w);
  } else if constexpr (kVec && (kInter || W == 8)) {
    *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(row + ld.o0);
    if constexpr (W == 8) *reinterpret_cast<uint4*>(w + 4) = *reinterpret_cast<const uint4*>(row + ld.o1);
  } else if constexpr (kVec) {
    *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(row + ld.o0);
    *reinterpret_cast<uint2*>(w + 2) = *reinterpret_cast<const uint2*>(row + ld.o1);
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const uint16_t* p = row + (j < W / 2 ? ld.o0 + 2 * j : ld.o1 + 2 * j - W);
      w[j] = (uint32_t)p[0] | ((uint32_t)p[1] << 16);
    }
  }
}

template <int W, bool kInter, bool kVec>
__device__ __forceinline__ void store_words(uint16_t* row, const HeadLane<W>& ld, const uint32_t w[W]) {
  if constexpr (kVec && kInter && W == 8) {
    store32(row + ld.o0, w);
  } else if constexpr (kVec && (kInter || W == 8)) {
    *reinterpret_cast<uint4*>(row + ld.o0) = make_uint4(w[0], w[1], w[2], w[3]);
    if constexpr (W == 8) *reinterpret_cast<uint4*>(row + ld.o1) = make_uint4(w[4], w[5], w[6], w[7]);
  } else if constexpr (kVec) {
    *reinterpret_cast<uint2*>(row + ld.o0) = make_uint2(w[0], w[1]);
    *reinterpret_cast<uint2*>(row + ld.o1) = make_uint2(w[2], w[3]);
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      uint16_t* p = row + (j < W / 2 ? ld.o0 + 2 * j : ld.o1 + 2 * j - W);
      p[0] = (uint16_t)w[j];
      p[1] = (uint16_t)(w[j] >> 16);
    }
  }
}

template <int W, bool kInter>
__device__ __forceinline__ Pairs<W> pairs_of(const uint32_t w[W]) {
  Pairs<W> x;
#pragma unroll
  for (int i = 0; i < W / 2; ++i) {
    if constexpr (kInter) {
      x.a[i] = make_float2(bf16lo(w[2 * i]), bf16lo(w[2 * i + 1]));
      x.b[i] = make_float2(bf16hi(w[2 * i]), bf16hi(w[2 * i + 1]));
    } else {
      x.a[i] = make_float2(bf16lo(w[i]), bf16hi(w[i]));
      x.b[i] = make_float2(bf16lo(w[W / 2 + i]), bf16hi(w[W / 2 + i]));
    }
  }
  return x;
}

template <int W, bool kInter>
__device__ __forceinline__ void words_of(const Pairs<W>& x, uint32_t w[W]) {
#pragma unroll
  for (int i = 0; i < W / 2; ++i) {
    if constexpr (kInter) {
      w[2 * i] = pack2_rn(x.a[i].x, x.b[i].x);
      w[2 * i + 1] = pack2_rn(x.a[i].y, x.b[i].y);
    } else {
      w[i] = pack2_rn(x.a[i].x, x.a[i].y);
      w[W / 2 + i] = pack2_rn(x.b[i].x, x.b[i].y);
    }
  }
}

// What a token and a weight vector make of a pair, (a', b') = inv * (a ac - b bs,
// a as + b bc): the weights are folded into the cosines and sines once per
// token, so a head costs four products per pair and one with inv.
template <int W>
struct Turn {
  float2 ac[W / 2], bs[W / 2], as[W / 2], bc[W / 2];  // bs holds -w_b s
};

// row: the token's row of the table (cosines, then sines), null for no rotation.
template <int W, bool kInter>
__device__ __forceinline__ Turn<W> make_turn(const float* row, int rot, int lane, const uint16_t* weight,
                                             const HeadLane<W>& ld) {
  Turn<W> t;
  float c[W], s[W];
#pragma unroll
  for (int i = 0; i < W; i += 4) {
    float4 c4 = make_float4(1.f, 1.f, 1.f, 1.f), s4 = make_float4(0.f, 0.f, 0.f, 0.f);
    if (ld.rotated) {
      c4 = *reinterpret_cast<const float4*>(row + W * lane + i);
      s4 = *reinterpret_cast<const float4*>(row + rot / 2 + W * lane + i);
    }
    *reinterpret_cast<float4*>(c + i) = c4;
    *reinterpret_cast<float4*>(s + i) = s4;
  }
#pragma unroll
  for (int i = 0; i < W / 2; ++i) {
    t.ac[i] = t.bc[i] = make_float2(c[2 * i], c[2 * i + 1]);
    t.as[i] = make_float2(s[2 * i], s[2 * i + 1]);
    t.bs[i] = make_float2(-s[2 * i], -s[2 * i + 1]);
  }
  if (weight) {
    uint32_t w[W];
    load_words<W, false, true>(weight, ld, w);
    const Pairs<W> x = pairs_of<W, kInter>(w);
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      t.ac[i] = mul2(t.ac[i], x.a[i]);
      t.as[i] = mul2(t.as[i], x.a[i]);
      t.bs[i] = mul2(t.bs[i], x.b[i]);
      t.bc[i] = mul2(t.bc[i], x.b[i]);
    }
  }
  return t;
}

// One head: the norm's factor (sum of squares in fp32) and the turn.  Every
// step is an operation with its rounding, and the sum a tree over runs of eight
// dims, so every kernel and either W give the same words.
template <int D, int W, bool kNorm>
__device__ __forceinline__ Pairs<W> turn_head(const Pairs<W>& x, const Turn<W>& t, bool rotated, float eps) {
  Pairs<W> y;
#pragma unroll
  for (int i = 0; i < W / 2; ++i) {
    y.a[i] = fma2(x.a[i], t.ac[i], mul2(x.b[i], t.bs[i]));
    y.b[i] = fma2(x.a[i], t.as[i], mul2(x.b[i], t.bc[i]));
  }
  if (!rotated)  // an infinity in one dim stays out of its neighbour's
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      y.a[i] = mul2(x.a[i], t.ac[i]);
      y.b[i] = mul2(x.b[i], t.bc[i]);
    }
  if constexpr (kNorm) {
    float part[W / 4];
#pragma unroll
    for (int j = 0; j < W / 4; ++j) {
      float2 q = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 2 * j; i < 2 * j + 2; ++i) q = fma2(x.b[i], x.b[i], fma2(x.a[i], x.a[i], q));
      part[j] = __fadd_rn(q.x, q.y);
    }
    float ss = part[0];
    if constexpr (W == 8) ss = __fadd_rn(part[0], part[1]);
#pragma unroll
    for (int off = 1; off < D / (2 * W); off <<= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, off));
    const float inv = rsqrtf(__fmaf_rn(ss, 1.f / D, eps));
    const float2 inv2 = make_float2(inv, inv);
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      y.a[i] = mul2(y.a[i], inv2);
      y.b[i] = mul2(y.b[i], inv2);
    }
  }
  return y;
}

constexpr uint32_t kTinyBits = 0x0D800000u;  // 2^-100 as fp32

// Largest |x| of a row of bf16 values as its 15 magnitude bits (which order
// like the magnitudes, with infinities and NaN above every number); kLanes
// lanes hold the row, kWords words each.
template <int kLanes, int kWords>
__device__ __forceinline__ uint32_t row_amax(const uint32_t* w) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kWords; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
#pragma unroll
  for (int off = kLanes / 2; off > 0; off >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, off));
  return max(m & 0xffffu, m >> 16);
}

// The row's scale and the lane's codes, in the order of its words.
template <int kLanes, int kWords, int FMT>
__device__ __forceinline__ float quantise_row(const uint32_t* w, uint32_t* codes) {
  const uint32_t am = row_amax<kLanes, kWords>(w);
  float scale;
  if constexpr (FMT == LARA_KVQ_INT8) {
    // rint of the exact quotient 127 x / a, ties to even, as x r rounded by
    // adding 1.5 * 2^23 (the integer is the sum's low byte).  For bf16 x and a a
    // quotient that is not a tie is at least 2^-17 of itself away from one.  Ties
    // are x = a / 2 (63.5, to 64) and, where a's significand is 254, any half:
    // there 127 / a is a power of two and x r exact.  Elsewhere r is taken a few
    // units in the last place above 127 / a, which settles a / 2 as it should.
    const uint32_t ab = max(am << 16, kTinyBits), expo = (ab & 0x7f800000u) - 0x3f800000u, sig = ab & 0x7fffffu;
    const float a = __uint_as_float(ab);
    float rcp;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(rcp) : "f"(__uint_as_float(sig | 0x3f800000u)));  // off by 2^-23 at most
    const uint32_t r127 = sig == 0x7e0000u ? 0x42800000u : __float_as_uint(127.f * rcp) + 6u;
    const float r = __uint_as_float(r127 - expo);
    // a / 127, rounded once: the product's error is put right by a fused step
    constexpr float kInv127 = 1.f / 127.f;
    const float q = __fmul_rn(a, kInv127);
    scale = __fmaf_rn(__fmaf_rn(-127.f, q, a), kInv127, q);
    const float2 r2 = make_float2(r, r), magic = make_float2(0x1.8p23f, 0x1.8p23f);
#pragma unroll
    for (int i = 0; i < kWords; i += 2) {
      uint32_t c[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        // the product is rounded by itself: a fused step could see past a tie
        const float2 n = add2(mul2(make_float2(bf16lo(w[i + k]), bf16hi(w[i + k])), r2), magic);
        c[k] = __byte_perm(__float_as_uint(n.x), __float_as_uint(n.y), 0x0040);
      }
      codes[i / 2] = __byte_perm(c[0], c[1], 0x5410);
    }
  } else {
    // a = (1 + m/128) 2^(E-127); 448 = 1.75 * 2^8, and 1 + m/128 <= 1.75 at m <= 96.
    const int e = max((int)(am >> 7) - 135 + ((am & 0x7fu) > 96u ? 1 : 0), -100);
    scale = __uint_as_float((uint32_t)(e + 127) << 23);
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);  // exact: a power of two
    const float2 inv2 = make_float2(inv, inv);
#pragma unroll
    for (int i = 0; i < kWords; i += 2) {
      uint32_t h[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        h[k] = __nv_cvt_float2_to_fp8x2(mul2(make_float2(bf16lo(w[i + k]), bf16hi(w[i + k])), inv2), __NV_SATFINITE,
                                        __NV_E4M3);
      codes[i / 2] = __byte_perm(h[0], h[1], 0x5410);
    }
  }
  if (am >= 0x7f80u) {
#pragma unroll
    for (int i = 0; i < kWords / 2; ++i) codes[i] = 0;
    scale = __uint_as_float(0x7fffffffu);
  }
  return scale;
}

// Four codes as fp32, as pairs (0, 1) and (2, 3).
template <int FMT>
__device__ __forceinline__ void codes_to_f32(uint32_t w, float2 f[2]) {
  if constexpr (FMT == LARA_KVQ_INT8) {
    // 2^23 + code + 128 by setting the upper bytes, minus 2^23 + 128
    const uint32_t x = w ^ 0x80808080u;
    const float2 bias = make_float2(-8388736.f, -8388736.f);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      f[i] = add2(make_float2(__uint_as_float(__byte_perm(x, 0x4b000000u, 0x7650 + 2 * i)),
                              __uint_as_float(__byte_perm(x, 0x4b000000u, 0x7651 + 2 * i))),
                  bias);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * i)), __NV_E4M3);
      f[i] = __half22float2(*reinterpret_cast<const __half2*>(&h));
    }
  }
}

// Where a token's row lies in the pool: index of the (page, kv head, row), or
// -1 for a bad page (flagged).
struct PoolIndex {
  const int32_t* block_table;
  int pages_per_seq, page_log2, num_pages, n_kv_heads;
  __device__ __forceinline__ long long row(int b, int h, int pos, int* status) const {
    const int page = __ldg(block_table + (long long)b * pages_per_seq + (pos >> page_log2));
    if (page < 0 || page >= num_pages) {
      if (status) atomicOr(status, kDevBadPage);
      return -1;
    }
    return ((((long long)page * n_kv_heads + h) << page_log2) + (pos & ((1 << page_log2) - 1)));
  }
  __host__ __device__ __forceinline__ long long capacity() const { return (long long)pages_per_seq << page_log2; }
};

// Host: the pool's pointers and geometry, checked; LARA_OK or an error code.
// Without sequences the block table may be null.
int check_pool(const lara_kvq_pool* pool, const void* block_table, int pages_per_seq, int batch, PoolIndex* index);

inline bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Whether two arrays of `bytes` bytes overlap (a null one overlaps nothing).
inline bool overlap(const void* a, const void* b, size_t bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a && b && x < y + bytes && y < x + bytes;
}

// The alignment in bytes, up to 32, of every row of a strided tensor (an extent
// of 1 takes no stride).
inline int row_alignment(const void* p, long long sb, int batch, long long st, int n, long long sh, int heads) {
  const long long bytes = 2 * ((batch > 1 ? sb : 0) | (n > 1 ? st : 0) | (heads > 1 ? sh : 0)) |
                          (long long)reinterpret_cast<uintptr_t>(p) | 32;
  return (int)(bytes & -bytes);
}

}  // namespace kvq
}  // namespace lara
