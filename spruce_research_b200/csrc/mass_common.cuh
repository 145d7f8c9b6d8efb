// Pieces shared by the kernels that sum softmax weights over keys (mass*.cu).
#pragma once

#include "paged_common.cuh"

namespace spruce {

struct KeyMassParams {
  PagedParams v;            // the batch: rows, keys and pages as the attention sees them
  const float* lse;         // [N, Hq]
  int64_t ln, lh;
  const float* mass;        // [num_pages, Hkv, page_size]
  float* out;
  int64_t ms[3], os[3];
  float decay;
  int key_tiles;            // of the longest sequence allowed
};

inline KeyMassParams key_mass_params(const KeyMassArgs& a, int tile) {
  KeyMassParams p{};
  p.v = paged_params(a.a, 16, 1, 0);
  p.lse = a.lse;
  p.ln = a.ln;
  p.lh = a.lh;
  p.mass = a.mass;
  p.out = a.out;
  for (int i = 0; i < 3; ++i) {
    p.ms[i] = a.ms[i];
    p.os[i] = a.os[i];
  }
  p.decay = a.decay;
  p.key_tiles = (p.v.kv_cap + tile - 1) / tile;
  return p;
}

// Key mass of more than kKmFewRows query rows a sequence and KV head, in 16 bits (key_mass_sm100.cu).
constexpr int kKmFewRows = 32, kKmFewRowsF32 = 16;
cudaError_t launch_key_mass_sm100(const KeyMassArgs& a, int dtype, cudaStream_t stream);
// At most that many (key_mass_rows.cu).
cudaError_t launch_key_mass_rows(const KeyMassArgs& a, int dtype, cudaStream_t stream);

// Block mass in 16 bits (block_mass_sm100.cu).
int64_t block_mass_sm100_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t T);
cudaError_t launch_block_mass_sm100(const BlockMassArgs& a, int dtype, cudaStream_t stream);

// Page of the 16 keys from `key` on; -1 past the sequence's keys, or where the table names no page of the cache.
__device__ __forceinline__ int mass_page(const KeyMassParams& p, int s, int key, int kv) {
  if (key >= kv) return -1;
  return paged_page(p.v, p.v.a.block_table + s * p.v.a.table_stride, key / p.v.a.page_size);
}

// Keys that the new tokens see.  All the sequence holds, but where its tokens are cut to max_q.
__device__ __forceinline__ int mass_keys(const PagedSeq& q) { return min(max(q.first + q.qlen, 0), q.kv); }

// A row's lse in log2 units.  A row that saw nothing (-inf) counts for nothing.
__device__ __forceinline__ float mass_row_lse(float lse) {
  return lse == -INFINITY ? INFINITY : lse * 1.4426950408889634f;
}

// A key's new weight; one that was there before the new tokens keeps a part of its old one.
__device__ __forceinline__ void mass_store(const KeyMassParams& p, int page, int g, int row, bool before, float sum) {
  if (before && p.decay != 0.0f) sum = fmaf(p.decay, p.mass[page * p.ms[0] + g * p.ms[1] + row * p.ms[2]], sum);
  p.out[page * p.os[0] + g * p.os[1] + row * p.os[2]] = sum;
}

// log2 of a row's total from its maximum and sum; +inf (all weights 0) where nothing is above -inf.
__device__ __forceinline__ float mass_total(float m, float l) { return l == 0.0f ? INFINITY : m + log2f(l); }

}  // namespace spruce
