// Operators of the paged bf16 cache beyond append and plain decode (sm_100a):
// what their kernels share.
#pragma once

#include <cuda_bf16.h>

#include "../../include/lara_b200.h"
#include "common.cuh"
#include "kvq.cuh"
#include "lara_internal.h"

namespace lara {
namespace paged {

using kvq::aligned;
using kvq::pack2_rn;
using kvq::PoolIndex;

constexpr size_t kStatusBytes = 256;

// What the own-token pass leaves of a unit, a (sequence, kv head): `parts`
// partial results from slot `slot0` on.
struct UnitParts {
  int slot0, parts;
};

// Host: geometry of a paged bf16 cache, checked; LARA_OK or an error code.
// Without sequences the pointers may be null.
int check_paged_pool(const void* k_pages, const void* v_pages, const void* block_table, int n_kv_heads, int head_dim,
                     int page_size, int pages_per_seq, int num_pages, int batch, PoolIndex* index);

// Weights may be updated in place or written elsewhere, not half over themselves.
int check_weights(const float* in, const float* out, int n_kv_heads, int page_size, int num_pages);

// The pass over a shared prefix: row tiles of `seqs` sequences, taken in pairs
// where there are two; `units` of them (pairs) to a kv head, of `rows` rows each.
struct PrefixPlan {
  int seqs, units, rows;
};
PrefixPlan prefix_plan(int batch, int group);

inline size_t up256(size_t x) { return (x + 255) / 256 * 256; }

}  // namespace paged
}  // namespace lara
