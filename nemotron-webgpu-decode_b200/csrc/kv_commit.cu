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
// Bound by latency, then by the rows' bytes, read and written once.  128 sequences,
// 8 pools, 8 of 64 rows each, 33.6 MB: 9.0 us with rows that L2 does not hold (3.7
// TB/s, where the bytes alone take 5.2: the path, the places and the first rows
// are loads that wait for one another, and the ninth node is a second round of
// them); 5.4 us in replays, from L2.  One sequence: its launch, 1.9 us.
#include "nwd_common.h"
#include "tree.cuh"

namespace {

constexpr uint32_t MAX_POOLS = 16;   // of nwd_kv_commit
constexpr uint32_t MAX_LAYERS = 32;  // of nwd_kv_commit_layers: a lane each
constexpr int THREADS = 128;
constexpr int AHEAD = 8;  // rows of a column in flight

// Pools, pools_per_layer to a layer, and where each layer's sequences are: one
// place for all pools, or K and V of each layer at the layer's own.
template <uint32_t POOLS, uint32_t LAYERS>
struct Args {
  uint4* pools[POOLS];
  const int64_t* row_offset[LAYERS];
  const int32_t* pos[LAYERS];
  const int32_t* capacity[LAYERS];  // or nullptr: the pool alone bounds a region
  const int32_t* tree_len[LAYERS];  // or nullptr: all nodes are present
  int32_t* lengths[LAYERS];         // what grows: pos, once where layers share it
  const int32_t* path;
  const int32_t* n_accepted;
  uint64_t pool_rows;
  uint32_t n_layers, pools_per_layer, batch, n_nodes, row_vec;
  bool whole_tree;  // the region has to hold the whole tree, not just the path
  uint32_t* err;
};
using OnePlace = Args<MAX_POOLS, 1>;
using OwnPlaces = Args<2 * MAX_LAYERS, MAX_LAYERS>;

// A sequence's move, as a warp has it: lane l holds nodes l and l + 32 of the
// path, and layer l's place.
struct Move {
  int32_t n, lo, hi, pos, capacity, tree_len;
  int64_t off;
};
template <typename A>
__device__ __forceinline__ Move load_move(const A& a, uint32_t b) {
  const uint32_t lane = threadIdx.x & 31;
  const int32_t* path = a.path + (uint64_t)b * a.n_nodes;
  Move m{a.n_accepted[b], -1, -1, 0, 0x7fffffff, (int32_t)a.n_nodes, 0};
  if (lane < a.n_nodes) m.lo = path[lane];
  if (lane + 32 < a.n_nodes) m.hi = path[lane + 32];
  if (lane < a.n_layers) {
    m.pos = a.pos[lane][b];
    m.off = a.row_offset[lane][b];
    if (a.capacity[lane]) m.capacity = a.capacity[lane][b];
    if (a.tree_len[lane]) m.tree_len = a.tree_len[lane][b];
  }
  return m;
}

// What speaks against a move, for the whole warp (error bits; 0:
// nothing): a path that does not ascend or leaves the tree, or rows outside the
// pool or the region in any of the layers, which a lane each looks at.  With
// whole_tree the rows are those that the attention asked for, so a tree that it
// refused, and whose rows it did not write, is refused here too.
template <typename A>
__device__ __forceinline__ uint32_t refusal(const A& a, const Move& p) {
  const uint32_t all = 0xffffffffu, lane = threadIdx.x & 31;
  const int32_t up = __shfl_up_sync(all, p.lo, 1), end = __shfl_sync(all, p.lo, 31);
  const int32_t up_hi = __shfl_up_sync(all, p.hi, 1);
  bool bad = p.n < 0 || p.n > (int32_t)a.n_nodes;
  if ((int32_t)lane < p.n)
    bad |= p.lo <= (lane ? up : -1) || p.lo >= (int32_t)a.n_nodes;
  if ((int32_t)lane + 32 < p.n)
    bad |= p.hi <= (lane ? up_hi : end) || p.hi >= (int32_t)a.n_nodes;
  if (__any_sync(all, bad)) return NWD_DEVERR_TREE;
  if (p.n == 0) return 0;
  const uint32_t at = (uint32_t)p.n - 1;
  uint32_t rows = (uint32_t)__shfl_sync(all, at < 32 ? p.lo : p.hi, (int)(at & 31)) + 1;
  if (a.whole_tree) {
    const uint32_t nodes = min((uint32_t)max(p.tree_len, 0), a.n_nodes);
    if (__any_sync(all, lane < a.n_layers && rows > nodes)) return NWD_DEVERR_TREE;
    rows = nodes;
  }
  const bool out = lane < a.n_layers &&
                   (p.off < 0 || p.pos < 0 || (uint64_t)p.off > a.pool_rows ||
                    (uint64_t)p.pos + rows > a.pool_rows - (uint64_t)p.off ||
                    (int64_t)p.pos + rows > p.capacity);
  return __any_sync(all, out) ? NWD_DEVERR_ROW_RANGE : 0u;
}

template <typename A>
__global__ void __launch_bounds__(THREADS) kv_commit_kernel(const __grid_constant__ A a) {
  const uint32_t b = blockIdx.y, layer = blockIdx.z / a.pools_per_layer;
  const Move p = load_move(a, b);
  const uint32_t bad = refusal(a, p);
  if (bad) {
    if (a.err && (blockIdx.x | blockIdx.z | threadIdx.x) == 0) atomicOr(a.err, bad);
    return;
  }
  const int64_t base = __shfl_sync(0xffffffffu, p.off + p.pos, (int)layer);
  const uint32_t c = blockIdx.x * THREADS + threadIdx.x;
  const bool mine = c < a.row_vec;  // (the others' lanes still hold path nodes)
  uint4* col = a.pools[blockIdx.z] + (uint64_t)base * a.row_vec + c;
  for (int j0 = 0; j0 < p.n; j0 += AHEAD) {
    const int32_t half = j0 < 32 ? p.lo : p.hi;
    uint4 x[AHEAD];
    int32_t from[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; i++) {
      from[i] = __shfl_sync(0xffffffffu, half, (j0 + i) & 31);
      if (mine && j0 + i < p.n) x[i] = col[(uint64_t)from[i] * a.row_vec];
    }
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
      if (mine && j0 + i < p.n && from[i] != j0 + i) col[(uint64_t)(j0 + i) * a.row_vec] = x[i];
  }
}

// The lengths that grow by what was accepted, behind the moves: a warp per
// sequence, a lane per layer.  A launch of its own, because every block of the
// moves reads the lengths.
constexpr uint32_t GROW_THREADS = 128;
__global__ void __launch_bounds__(GROW_THREADS)
    kv_commit_lengths_kernel(const __grid_constant__ OwnPlaces a) {
  nwd::pdl_wait();
  const uint32_t b = (blockIdx.x * GROW_THREADS + threadIdx.x) / 32, lane = threadIdx.x & 31;
  if (b >= a.batch) return;
  const Move p = load_move(a, b);
  if (refusal(a, p)) return;
  if (lane < a.n_layers && a.lengths[lane]) a.lengths[lane][b] = p.pos + p.n;
}

// The arguments that both calls have, checked in the order that their errors have.
int check_commit(const char* who, bool null, uint16_t* const* pools, uint32_t n_pools,
                 uint32_t max_pools, uint32_t batch, uint32_t n_nodes, uint32_t n_kv, uint32_t hd) {
  using namespace nwd;
  if (n_pools > max_pools)
    return fail(NWD_ERR_INVALID, "%s: %u pools (at most %u)", who, n_pools, max_pools);
  if (null || (n_pools && !pools)) return fail(NWD_ERR_INVALID, "%s: null pointer", who);
  if (n_kv == 0 || hd == 0) return fail(NWD_ERR_INVALID, "%s: zero shape", who);
  if (n_nodes > TREE_MAX_NODES)
    return fail(NWD_ERR_UNSUPPORTED, "%s: %u nodes (at most %u)", who, n_nodes, TREE_MAX_NODES);
  if (batch > 65535u) return fail(NWD_ERR_UNSUPPORTED, "%s: batch > 65535", who);
  const uint64_t row = (uint64_t)n_kv * hd;
  if (row > (1ull << 30)) return fail(NWD_ERR_INVALID, "%s: row of %llu halves is too large", who,
                                      (unsigned long long)row);
  for (uint32_t i = 0; i < n_pools; i++) {
    if (!pools[i]) return fail(NWD_ERR_INVALID, "%s: pool %u is NULL", who, i);
    if (row % 8 || !aligned16(pools[i]))
      return fail(NWD_ERR_UNSUPPORTED,
                  "%s: rows must be a multiple of 8 halves, pools 16-byte aligned", who);
    for (uint32_t j = 0; j < i; j++)
      if (pools[j] == pools[i])
        return fail(NWD_ERR_INVALID, "%s: pools %u and %u are the same", who, j, i);
  }
  return NWD_OK;
}

template <typename A>
int launch_commit(const char* who, const A& a, uint32_t n_pools, cudaStream_t stream) {
  kv_commit_kernel<<<dim3((a.row_vec + THREADS - 1) / THREADS, a.batch, n_pools), THREADS, 0,
                     stream>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return nwd::cuda_fail(e, who);
  return nwd::ok();
}

}  // namespace

using namespace nwd;

extern "C" int nwd_kv_commit(uint16_t* const* pools, uint32_t n_pools, uint64_t pool_rows,
                             const int64_t* row_offset, const int32_t* pos, const int32_t* path,
                             const int32_t* n_accepted, uint32_t batch, uint32_t n_nodes,
                             uint32_t n_kv, uint32_t hd, uint32_t* err, void* stream) {
  const char* who = "nwd_kv_commit";
  int st = check_commit(who, !row_offset || !pos || !path || !n_accepted, pools, n_pools, MAX_POOLS,
                        batch, n_nodes, n_kv, hd);
  if (st) return st;
  if (batch == 0 || n_pools == 0 || n_nodes == 0) return ok();
  OnePlace a{};
  for (uint32_t i = 0; i < n_pools; i++) a.pools[i] = reinterpret_cast<uint4*>(pools[i]);
  a.row_offset[0] = row_offset;
  a.pos[0] = pos;
  a.path = path;
  a.n_accepted = n_accepted;
  a.pool_rows = pool_rows;
  a.n_layers = 1;
  a.pools_per_layer = n_pools;
  a.batch = batch;
  a.n_nodes = n_nodes;
  a.row_vec = (uint32_t)((uint64_t)n_kv * hd / 8);
  a.err = err;
  return launch_commit(who, a, n_pools, (cudaStream_t)stream);
}

extern "C" int nwd_kv_commit_layers(uint16_t* const* pools, uint32_t n_layers, uint64_t pool_rows,
                                    const int64_t* const* row_offset, int32_t* const* lengths,
                                    const int32_t* const* capacity, const int32_t* const* tree_len,
                                    const int32_t* path, const int32_t* n_accepted, uint32_t batch,
                                    uint32_t n_nodes, uint32_t n_kv, uint32_t hd, uint32_t* err,
                                    void* stream) {
  const char* who = "nwd_kv_commit_layers";
  if (n_layers > MAX_LAYERS)
    return fail(NWD_ERR_INVALID, "%s: %u layers (at most %u)", who, n_layers, MAX_LAYERS);
  bool null = !path || !n_accepted || (n_layers && (!row_offset || !lengths));
  for (uint32_t i = 0; !null && i < n_layers; i++) null = !row_offset[i] || !lengths[i];
  int st = check_commit(who, null, pools, 2 * n_layers, 2 * MAX_LAYERS, batch, n_nodes, n_kv, hd);
  if (st) return st;
  if (batch == 0 || n_layers == 0 || n_nodes == 0) return ok();
  OwnPlaces a{};
  for (uint32_t i = 0; i < n_layers; i++) {
    a.pools[2 * i] = reinterpret_cast<uint4*>(pools[2 * i]);
    a.pools[2 * i + 1] = reinterpret_cast<uint4*>(pools[2 * i + 1]);
    a.row_offset[i] = row_offset[i];
    a.pos[i] = a.lengths[i] = lengths[i];
    for (uint32_t j = 0; j < i; j++)
      if (lengths[j] == lengths[i]) a.lengths[i] = nullptr;
    a.capacity[i] = capacity ? capacity[i] : nullptr;
    a.tree_len[i] = tree_len ? tree_len[i] : nullptr;
  }
  a.whole_tree = true;
  a.path = path;
  a.n_accepted = n_accepted;
  a.pool_rows = pool_rows;
  a.n_layers = n_layers;
  a.pools_per_layer = 2;
  a.batch = batch;
  a.n_nodes = n_nodes;
  a.row_vec = (uint32_t)((uint64_t)n_kv * hd / 8);
  a.err = err;
  st = launch_commit(who, a, 2 * n_layers, (cudaStream_t)stream);
  if (st) return st;
  const cudaError_t e =
      launch_pdl(kv_commit_lengths_kernel, dim3((batch + GROW_THREADS / 32 - 1) / (GROW_THREADS / 32)),
                 dim3(GROW_THREADS), 0, (cudaStream_t)stream, a);
  if (e != cudaSuccess) return cuda_fail(e, who);
  return ok();
}
