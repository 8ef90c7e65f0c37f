// Rows of the 8-bit KV pool and of the q/k head pass (sm_100a).
//
// A row is the D values of one (token, head).  D / 8 lanes hold it, eight
// values each, and reduce over it with shuffles; a warp holds 256 / D rows.
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

// Eight values as two runs of four at element offsets o0 and o1.  kVec: 8-byte
// accesses (the row is 8-byte aligned), else one element at a time.
template <bool kVec>
__device__ __forceinline__ void load8(const uint16_t* row, int o0, int o1, float x[8]) {
  if constexpr (kVec) {
    bf16x4_to_f32(*reinterpret_cast<const uint2*>(row + o0), x);
    bf16x4_to_f32(*reinterpret_cast<const uint2*>(row + o1), x + 4);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = __uint_as_float((uint32_t)row[o0 + j] << 16);
      x[4 + j] = __uint_as_float((uint32_t)row[o1 + j] << 16);
    }
  }
}

// Round to nearest even; NaN stays NaN (the reference packer's carry could
// turn a NaN's payload over, and a NaN row has to read as one).
__device__ __forceinline__ uint32_t pack2_rn(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return reinterpret_cast<const uint32_t&>(v);
}

template <bool kVec>
__device__ __forceinline__ void store8(uint16_t* row, int o0, int o1, const uint32_t w[4]) {
  if constexpr (kVec) {
    *reinterpret_cast<uint2*>(row + o0) = make_uint2(w[0], w[1]);
    *reinterpret_cast<uint2*>(row + o1) = make_uint2(w[2], w[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      row[o0 + j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
      row[o1 + j] = (uint16_t)(w[2 + j / 2] >> (16 * (j & 1)));
    }
  }
}

// Which dims a lane of a row holds: pairs (2i, 2i+1) lie side by side; pairs
// (i, i + rot/2) are brought together in one lane by giving the first rot/8
// lanes four dims of each half, so the rotation needs no exchange.
struct LaneDims {
  int o0, o1;
  bool rotated;
  __device__ __forceinline__ LaneDims(int lane_in_row, int rot, bool interleaved) {
    rotated = 8 * lane_in_row < rot;
    const bool split = rotated && !interleaved;
    o0 = split ? 4 * lane_in_row : 8 * lane_in_row;
    o1 = split ? rot / 2 + 4 * lane_in_row : 8 * lane_in_row + 4;
  }
};

// Norm of one row: the sum of squares and every product in fp32, each step
// written out so that all kernels that norm a row round alike.
template <int D>
__device__ __forceinline__ void norm_row(float x[8], const float w[8], float eps) {
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) ss = __fmaf_rn(x[j], x[j], ss);
#pragma unroll
  for (int off = D / 16; off > 0; off >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, off));
  const float inv = __frsqrt_rn(__fmaf_rn(ss, 1.f / D, eps));
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = __fmul_rn(__fmul_rn(x[j], inv), w[j]);
}

__device__ __forceinline__ void rotate_pair(float& a, float& b, float c, float s) {
  const float y = __fmaf_rn(a, c, -__fmul_rn(b, s));
  b = __fmaf_rn(a, s, __fmul_rn(b, c));
  a = y;
}

// Pair j of the lane has table index 4 * lane_in_row + j in either pairing.
__device__ __forceinline__ void rotate_row(float x[8], const float4& c, const float4& s, bool interleaved) {
  if (interleaved) {
    rotate_pair(x[0], x[1], c.x, s.x);
    rotate_pair(x[2], x[3], c.y, s.y);
    rotate_pair(x[4], x[5], c.z, s.z);
    rotate_pair(x[6], x[7], c.w, s.w);
  } else {
    rotate_pair(x[0], x[4], c.x, s.x);
    rotate_pair(x[1], x[5], c.y, s.y);
    rotate_pair(x[2], x[6], c.z, s.z);
    rotate_pair(x[3], x[7], c.w, s.w);
  }
}

constexpr uint32_t kTinyBits = 0x0D800000u;  // 2^-100 as fp32

// Largest |x| of a row of bf16 values as its 15 magnitude bits (which order
// like the magnitudes, with infinities and NaN above every number).
template <int D>
__device__ __forceinline__ uint32_t row_amax(const uint32_t w[4]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
#pragma unroll
  for (int off = D / 16; off > 0; off >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, off));
  return max(m & 0xffffu, m >> 16);
}

// The row's scale and the lane's eight codes.
template <int D, int FMT>
__device__ __forceinline__ float quantise_row(const uint32_t w[4], uint32_t codes[2]) {
  const uint32_t am = row_amax<D>(w);
  const bool finite = am < 0x7f80u;
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16lo(w[i]);
    x[2 * i + 1] = bf16hi(w[i]);
  }
  float scale;
  if constexpr (FMT == LARA_KVQ_INT8) {
    // 127 x is exact in fp32 (8 + 7 bits; rows past 2^100 are brought down by
    // 2^-16 first, so that it stays finite) and the quotient is rounded once,
    // so a code sits on a tie only where 127 x / a itself does.
    const float down = am >= 0x7180u ? 0x1p-16f : 1.f;
    const float a = __uint_as_float(max(am << 16, kTinyBits)) * down;
    scale = __fdiv_rn(a, 127.f) / down;
    uint32_t c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = (uint32_t)__float2int_rn(__fdiv_rn(127.f * (x[j] * down), a)) & 0xffu;
    codes[0] = c[0] | (c[1] << 8) | (c[2] << 16) | (c[3] << 24);
    codes[1] = c[4] | (c[5] << 8) | (c[6] << 16) | (c[7] << 24);
  } else {
    // a = (1 + m/128) 2^(E-127); 448 = 1.75 * 2^8, and 1 + m/128 <= 1.75 at m <= 96.
    const int e = max((int)(am >> 7) - 135 + ((am & 0x7fu) > 96u ? 1 : 0), -100);
    scale = __uint_as_float((uint32_t)(e + 127) << 23);
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);  // exact: a power of two
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      h[i] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * i] * inv, x[2 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    codes[0] = h[0] | (h[1] << 16);
    codes[1] = h[2] | (h[3] << 16);
  }
  if (!finite) {
    codes[0] = codes[1] = 0;
    scale = __uint_as_float(0x7fffffffu);
  }
  return scale;
}

// Four codes as fp32.
template <int FMT>
__device__ __forceinline__ void codes_to_f32(uint32_t w, float f[4]) {
  if constexpr (FMT == LARA_KVQ_INT8) {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = (float)(int8_t)(w >> (8 * j));
  } else {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * j)), __NV_E4M3);
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&h));
      f[2 * j] = p.x;
      f[2 * j + 1] = p.y;
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
int check_pool(const lara_kvq_pool* pool, const void* block_table, int pages_per_seq, PoolIndex* index);

inline bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

}  // namespace kvq
}  // namespace lara
