// The accepted path's cache rows, moved to the end of the context: row
// seq + path[j] of a sequence becomes row seq + j, for up to 16 pools (K and V
// of several layers) in one launch.  Bit-exact.
//
// path is strictly increasing and path[j] >= j, so in the order of j a row is
// overwritten only after it has been read.  A thread owns 16 bytes of a row
// (a column of the pool) and moves them for every j, a batch of loads before
// its stores (the rows a batch writes, j0 .. j0 + 7, lie before every row
// that a later batch reads): columns are independent, so no thread waits for
// another.
//
// Bound by the rows' bytes, read and written once: 128 sequences, 8 pools, 8 of
// 64 rows each, 33.6 MB in 5.8 us (5.8 TB/s); one sequence by its launch, 2.5 us.
#include "nwd_common.h"
#include "tree.cuh"

namespace {

constexpr uint32_t MAX_POOLS = 16;
constexpr int THREADS = 128;
constexpr int AHEAD = 8;  // rows of a column in flight

struct Pools {
  uint4* p[MAX_POOLS];
};

__global__ void __launch_bounds__(THREADS)
    kv_commit_kernel(const __grid_constant__ Pools pools, uint64_t pool_rows,
                     const int64_t* __restrict__ row_offset, const int32_t* __restrict__ pos,
                     const int32_t* __restrict__ path, const int32_t* __restrict__ n_accepted,
                     uint32_t n_nodes, uint32_t row_vec, uint32_t* err) {
  const uint32_t b = blockIdx.y;
  __shared__ int32_t s_path[nwd::TREE_MAX_NODES];
  const int32_t n = n_accepted[b];
  if (threadIdx.x < n_nodes) s_path[threadIdx.x] = path[(uint64_t)b * n_nodes + threadIdx.x];
  __syncthreads();
  // a path that does not ascend, or leaves the tree, moves nothing
  bool bad = n < 0 || n > (int32_t)n_nodes;
  int last = -1;
  if (!bad) {
    for (int j = 0; j < n; j++) {
      bad |= s_path[j] <= last || s_path[j] >= (int32_t)n_nodes;
      last = s_path[j];
    }
  }
  if (bad) {
    if (err && threadIdx.x == 0) atomicOr(err, NWD_DEVERR_TREE);
    return;
  }
  const int64_t base = row_offset[b] + (int64_t)pos[b];
  if (n > 0 && (row_offset[b] < 0 || pos[b] < 0 || (uint64_t)base + last >= pool_rows)) {
    if (err && threadIdx.x == 0) atomicOr(err, NWD_DEVERR_ROW_RANGE);
    return;
  }
  const uint32_t c = blockIdx.x * THREADS + threadIdx.x;
  if (c >= row_vec) return;
  uint4* col = pools.p[blockIdx.z] + (uint64_t)base * row_vec + c;
  for (int j0 = 0; j0 < n; j0 += AHEAD) {
    uint4 x[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
      if (j0 + i < n) x[i] = col[(uint64_t)s_path[j0 + i] * row_vec];
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
      if (j0 + i < n && s_path[j0 + i] != j0 + i) col[(uint64_t)(j0 + i) * row_vec] = x[i];
  }
}

}  // namespace

using namespace nwd;

extern "C" int nwd_kv_commit(uint16_t* const* pools, uint32_t n_pools, uint64_t pool_rows,
                             const int64_t* row_offset, const int32_t* pos, const int32_t* path,
                             const int32_t* n_accepted, uint32_t batch, uint32_t n_nodes,
                             uint32_t n_kv, uint32_t hd, uint32_t* err, void* stream) {
  const char* who = "nwd_kv_commit";
  if (n_pools > MAX_POOLS)
    return fail(NWD_ERR_INVALID, "%s: %u pools (at most %u)", who, n_pools, MAX_POOLS);
  if ((n_pools && !pools) || !row_offset || !pos || !path || !n_accepted)
    return fail(NWD_ERR_INVALID, "%s: null pointer", who);
  if (n_kv == 0 || hd == 0) return fail(NWD_ERR_INVALID, "%s: zero shape", who);
  if (n_nodes > TREE_MAX_NODES)
    return fail(NWD_ERR_UNSUPPORTED, "%s: %u nodes (at most %u)", who, n_nodes, TREE_MAX_NODES);
  if (batch > 65535u) return fail(NWD_ERR_UNSUPPORTED, "%s: batch > 65535", who);
  const uint64_t row = (uint64_t)n_kv * hd;
  if (row > (1ull << 30)) return fail(NWD_ERR_INVALID, "%s: row of %llu halves is too large", who,
                                      (unsigned long long)row);
  Pools pp{};
  for (uint32_t i = 0; i < n_pools; i++) {
    if (!pools[i]) return fail(NWD_ERR_INVALID, "%s: pool %u is NULL", who, i);
    if (row % 8 || !aligned16(pools[i]))
      return fail(NWD_ERR_UNSUPPORTED,
                  "%s: rows must be a multiple of 8 halves, pools 16-byte aligned", who);
    for (uint32_t j = 0; j < i; j++)
      if (pools[j] == pools[i])
        return fail(NWD_ERR_INVALID, "%s: pools %u and %u are the same", who, j, i);
    pp.p[i] = reinterpret_cast<uint4*>(pools[i]);
  }
  if (batch == 0 || n_pools == 0 || n_nodes == 0) return ok();
  const uint32_t row_vec = (uint32_t)(row / 8);
  kv_commit_kernel<<<dim3((row_vec + THREADS - 1) / THREADS, batch, n_pools), THREADS, 0,
                     (cudaStream_t)stream>>>(pp, pool_rows, row_offset, pos, path, n_accepted,
                                             n_nodes, row_vec, err);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, who);
  return ok();
}
