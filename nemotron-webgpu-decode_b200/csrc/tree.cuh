// Trees of drafted tokens, as the speculative-decoding kernels read them.
//
// A tree of n <= 64 nodes is parents[0..n): parents[i] < i, or -1 for a root.
// Nodes at or past tree_len[b] are absent.  A parent outside [-1, i) is
// recorded as NWD_DEVERR_TREE and read as -1, so every walk towards the root
// descends strictly and ends.
#pragma once

#include <stdint.h>

#include "nwd.h"

namespace nwd {

constexpr uint32_t TREE_MAX_NODES = 64;  // one 64-bit mask per node

// Node i's parent, or -1.
static __device__ __forceinline__ int tree_parent(const int32_t* parents, int i, uint32_t* err) {
  const int p = parents[i];
  if (p >= -1 && p < i) return p;
  if (err) atomicOr(err, NWD_DEVERR_TREE);
  return -1;
}

// Bit j: node i sees node j (its ancestors and itself).
static __device__ __forceinline__ uint64_t tree_mask(const int32_t* parents, int i, uint32_t* err) {
  uint64_t m = 0;
  for (; i >= 0; i = tree_parent(parents, i, err)) m |= 1ull << i;
  return m;
}

// The rows that each of n nodes sees, for a warp whose lane i has the parents of
// nodes i and i + 32 (anything for those past n): seen[0] is node i's, seen[1]
// node i + 32's.
// The lanes walk up in doubling steps, so a chain takes as many as the logarithm
// of its depth.
static __device__ __forceinline__ void tree_closure(int2 par, uint32_t n, uint32_t* err,
                                                    uint64_t (&seen)[2]) {
  const int lane = (int)(threadIdx.x & 31);
  int up[2] = {par.x, par.y};
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const int i = lane + 32 * k;
    if (up[k] < -1 || up[k] >= i) {
      if (i < (int)n && err) atomicOr(err, NWD_DEVERR_TREE);
      up[k] = -1;
    }
    seen[k] = 1ull << i;
  }
  while (__any_sync(0xffffffffu, up[0] >= 0 || up[1] >= 0)) {
    uint64_t more[2];
    int far[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const int from = up[k] & 31;
      const uint64_t lo = __shfl_sync(0xffffffffu, seen[0], from);
      const uint64_t hi = __shfl_sync(0xffffffffu, seen[1], from);
      const int flo = __shfl_sync(0xffffffffu, up[0], from);
      const int fhi = __shfl_sync(0xffffffffu, up[1], from);
      more[k] = up[k] < 0 ? 0 : up[k] < 32 ? lo : hi;
      far[k] = up[k] < 0 ? -1 : up[k] < 32 ? flo : fhi;
    }
#pragma unroll
    for (int k = 0; k < 2; k++) {
      seen[k] |= more[k];
      up[k] = far[k];
    }
  }
}

// Present nodes of sequence b: tree_len[b] (nullptr: all), held to [0, n].
static __device__ __forceinline__ uint32_t tree_nodes(const int32_t* tree_len, uint32_t b,
                                                      uint32_t n, uint32_t* err) {
  if (!tree_len) return n;
  const int32_t l = tree_len[b];
  if (l >= 0 && (uint32_t)l <= n) return (uint32_t)l;
  if (err) atomicOr(err, NWD_DEVERR_TREE);
  return l < 0 ? 0u : n;
}

// The rows of a sequence: ctx context rows from pool row row0, then its nodes'.
// A sequence whose rows leave the pool, or its region of `capacity` rows where
// those are given, is recorded as NWD_DEVERR_ROW_RANGE and has no rows and no
// nodes.
struct TreeSeq {
  int64_t row0;
  uint32_t ctx, nodes;
};
struct TreeRaw {
  int64_t row_offset;
  int32_t seq_len, tree_len, capacity;
};
static __device__ __forceinline__ TreeRaw tree_raw(const int64_t* row_offset,
                                                   const int32_t* seq_len, const int32_t* tree_len,
                                                   const int32_t* capacity, uint32_t b,
                                                   uint32_t n) {
  return TreeRaw{row_offset[b], seq_len[b], tree_len ? tree_len[b] : (int32_t)n,
                 capacity ? capacity[b] : 0x7fffffff};
}
static __device__ __forceinline__ TreeSeq tree_seq(const TreeRaw& raw, uint64_t pool_rows,
                                                   uint32_t n, uint32_t* err) {
  TreeSeq s;
  s.row0 = raw.row_offset;
  s.ctx = (uint32_t)raw.seq_len;
  s.nodes = min((uint32_t)max(raw.tree_len, 0), n);
  if ((uint32_t)raw.tree_len > n && err) atomicOr(err, NWD_DEVERR_TREE);
  if (s.row0 < 0 || raw.seq_len < 0 || (uint64_t)s.row0 > pool_rows ||
      (uint64_t)s.ctx + s.nodes > pool_rows - (uint64_t)s.row0 ||
      (int64_t)s.ctx + s.nodes > raw.capacity) {
    if (err) atomicOr(err, NWD_DEVERR_ROW_RANGE);
    s.row0 = 0;
    s.ctx = s.nodes = 0;
  }
  return s;
}
static __device__ __forceinline__ TreeSeq tree_seq(const int64_t* row_offset,
                                                   const int32_t* seq_len, const int32_t* tree_len,
                                                   const int32_t* capacity, uint64_t pool_rows,
                                                   uint32_t b, uint32_t n, uint32_t* err) {
  return tree_seq(tree_raw(row_offset, seq_len, tree_len, capacity, b, n), pool_rows, n, err);
}

}  // namespace nwd
