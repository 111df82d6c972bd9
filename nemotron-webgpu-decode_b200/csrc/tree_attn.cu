// Attention for a tree of drafted tokens over the KV pool.
//
// Node i of sequence b sits at pool row row_offset[b] + seq_len[b] + i and
// attends the seq_len[b] context rows, its ancestors' rows and its own:
//   O[b,i,h] = softmax_t(scale * q[b,i,h] . K[t, h/group]) V[t, h/group].
// The reference decodes one token per step (engine/runtime.js:447-467): a
// chain of n nodes computes what n of its steps would, a tree several such
// chains that share their beginnings, over one read of the cache.
//
// One warp per (sequence, node, head): the lanes hold 4 of the 128 dims each,
// a row's score is a warp sum, the softmax runs online in f32.
#include <cuda_fp16.h>

#include <cmath>

#include "nwd_common.h"
#include "tree.cuh"

namespace {

using nwd::TreeSeq;

constexpr uint32_t HD = 128;

struct TreeParams {
  const __half* q;
  const __half* k;
  const __half* v;
  __half* o;
  const int64_t* row_offset;
  const int32_t* seq_len;
  const int32_t* parents;
  const int32_t* tree_len;
  uint32_t* err;
  uint64_t pool_rows;
  uint32_t batch, n_nodes, n_heads, n_kv, group;
  float scale;
};

__device__ __forceinline__ float4 load4(const __half* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}

__global__ void tree_attn_kernel(const TreeParams p) {
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t hkv = blockIdx.x % p.n_kv, i = blockIdx.x / p.n_kv, b = blockIdx.y;
  const uint32_t h = hkv * p.group + warp;
  const TreeSeq s = nwd::tree_seq(p.row_offset, p.seq_len, p.tree_len, p.pool_rows, b, p.n_nodes,
                                  p.err);
  const uint64_t sees =
      i < s.nodes ? nwd::tree_mask(p.parents + (uint64_t)b * p.n_nodes, (int)i, p.err) : 0;
  const uint64_t at = (((uint64_t)b * p.n_nodes + i) * p.n_heads + h) * HD + lane * 4;
  const float4 q = load4(p.q + at);
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  const uint32_t rows = i < s.nodes ? s.ctx + i + 1 : 0;
  for (uint32_t t = 0; t < rows; t++) {
    if (t >= s.ctx && !((sees >> (t - s.ctx)) & 1)) continue;
    const uint64_t r = (((uint64_t)s.row0 + t) * p.n_kv + hkv) * HD + lane * 4;
    const float4 k = load4(p.k + r);
    float d = q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w;
#pragma unroll
    for (int x = 16; x; x >>= 1) d += __shfl_xor_sync(0xffffffffu, d, x);
    d *= p.scale;
    const float mn = fmaxf(m, d), alpha = m == -INFINITY ? 0.f : expf(m - mn), w = expf(d - mn);
    const float4 v = load4(p.v + r);
    l = l * alpha + w;
    acc.x = acc.x * alpha + w * v.x;
    acc.y = acc.y * alpha + w * v.y;
    acc.z = acc.z * alpha + w * v.z;
    acc.w = acc.w * alpha + w * v.w;
    m = mn;
  }
  const float inv = rows ? 1.f / l : 0.f;
  __half2* out = reinterpret_cast<__half2*>(p.o + at);
  out[0] = __floats2half2_rn(acc.x * inv, acc.y * inv);
  out[1] = __floats2half2_rn(acc.z * inv, acc.w * inv);
}

// The nodes' K / V rows [batch, n_nodes, n_kv, hd] into pool rows
// row_offset[b] + pos[b] + i, 16 bytes per thread (kv_append for a tree).
__global__ void tree_append_kernel(const uint4* __restrict__ k_new, const uint4* __restrict__ v_new,
                                   uint4* __restrict__ k_pool, uint4* __restrict__ v_pool,
                                   const int64_t* row_offset, const int32_t* pos,
                                   const int32_t* tree_len, uint64_t pool_rows, uint32_t n_nodes,
                                   uint32_t row_vec, uint32_t* err) {
  const uint32_t b = blockIdx.y;
  const TreeSeq s = nwd::tree_seq(row_offset, pos, tree_len, pool_rows, b, n_nodes, err);
  const uint64_t dst = ((uint64_t)s.row0 + s.ctx) * row_vec, src = (uint64_t)b * n_nodes * row_vec;
  for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < s.nodes * row_vec;
       i += gridDim.x * blockDim.x) {
    k_pool[dst + i] = __ldg(k_new + src + i);
    v_pool[dst + i] = __ldg(v_new + src + i);
  }
}

int check_tree(const char* who, const void* q, const void* k_pool, const void* v_pool,
               const void* row_offset, const void* seq_len, const void* parents, const void* o,
               uint64_t pool_rows, uint32_t batch, uint32_t n_nodes, uint32_t n_heads,
               uint32_t n_kv, uint32_t head_dim, float scale) {
  using namespace nwd;
  if (!q || !k_pool || !v_pool || !row_offset || !seq_len || !parents || !o)
    return fail(NWD_ERR_INVALID, "%s: null pointer", who);
  if (n_heads == 0 || n_kv == 0 || n_heads % n_kv)
    return fail(NWD_ERR_INVALID, "%s: n_heads must be a positive multiple of n_kv_heads", who);
  if (head_dim != HD || n_heads / n_kv > 8)
    return fail(NWD_ERR_UNSUPPORTED, "%s: head_dim %u, group %u (head_dim 128, group 1..8)", who,
                head_dim, n_heads / n_kv);
  if (n_nodes > TREE_MAX_NODES)
    return fail(NWD_ERR_UNSUPPORTED, "%s: %u nodes (at most %u)", who, n_nodes, TREE_MAX_NODES);
  if (batch > 4096) return fail(NWD_ERR_UNSUPPORTED, "%s: batch %u (at most 4096)", who, batch);
  if (!aligned16(q) || !aligned16(k_pool) || !aligned16(v_pool) || !aligned16(o))
    return fail(NWD_ERR_INVALID, "%s: tensors must be 16-byte aligned", who);
  if (!(scale >= 0.f) || std::isinf(scale))
    return fail(NWD_ERR_INVALID, "%s: scale must be finite and >= 0", who);
  if (pool_rows == 0 || pool_rows > (1ull << 31))
    return fail(NWD_ERR_INVALID, "%s: pool rows %llu outside [1, 2^31]", who,
                (unsigned long long)pool_rows);
  return NWD_OK;
}

}  // namespace

using namespace nwd;

extern "C" {

int nwd_attn_tree_workspace_size(uint32_t batch, uint32_t n_nodes, uint32_t n_heads,
                                 uint32_t n_kv_heads, uint32_t head_dim, size_t* bytes) {
  const char* who = "nwd_attn_tree_workspace_size";
  if (!bytes) return fail(NWD_ERR_INVALID, "%s: bytes is NULL", who);
  const void* p = reinterpret_cast<const void*>(16);
  int st = check_tree(who, p, p, p, p, p, p, p, 1, batch, n_nodes, n_heads, n_kv_heads, head_dim,
                      0.f);
  if (st) return st;
  *bytes = 256;
  return ok();
}

int nwd_attn_tree(const uint16_t* q, const uint16_t* k_pool, const uint16_t* v_pool,
                  uint64_t pool_rows, const int64_t* row_offset, const int32_t* seq_len,
                  const int32_t* parents, const int32_t* tree_len, uint16_t* o, uint32_t batch,
                  uint32_t n_nodes, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim,
                  float scale, void* workspace, size_t ws_bytes, uint32_t* err, void* stream) {
  const char* who = "nwd_attn_tree";
  int st = check_tree(who, q, k_pool, v_pool, row_offset, seq_len, parents, o, pool_rows, batch,
                      n_nodes, n_heads, n_kv_heads, head_dim, scale);
  if (st) return st;
  if (!workspace || ws_bytes < 256 || ((uintptr_t)workspace & 255u))
    return fail(NWD_ERR_WORKSPACE, "%s: needs a 256-byte aligned workspace of >= 256 bytes", who);
  if (batch == 0 || n_nodes == 0) return ok();
  TreeParams p{};
  p.q = reinterpret_cast<const __half*>(q);
  p.k = reinterpret_cast<const __half*>(k_pool);
  p.v = reinterpret_cast<const __half*>(v_pool);
  p.o = reinterpret_cast<__half*>(o);
  p.row_offset = row_offset;
  p.seq_len = seq_len;
  p.parents = parents;
  p.tree_len = tree_len;
  p.err = err;
  p.pool_rows = pool_rows;
  p.batch = batch;
  p.n_nodes = n_nodes;
  p.n_heads = n_heads;
  p.n_kv = n_kv_heads;
  p.group = n_heads / n_kv_heads;
  p.scale = scale != 0.f ? scale : 1.0f / sqrtf((float)head_dim);
  tree_attn_kernel<<<dim3(n_kv_heads * n_nodes, batch), 32 * p.group, 0, (cudaStream_t)stream>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, who);
  return ok();
}

int nwd_kv_append_attn_tree(const uint16_t* q, const uint16_t* k_new, const uint16_t* v_new,
                            uint16_t* k_pool, uint16_t* v_pool, uint64_t pool_rows,
                            const int64_t* row_offset, const int32_t* pos, const int32_t* parents,
                            const int32_t* tree_len, uint16_t* o, uint32_t batch, uint32_t n_nodes,
                            uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, float scale,
                            void* workspace, size_t ws_bytes, uint32_t* err, void* stream) {
  const char* who = "nwd_kv_append_attn_tree";
  int st = check_tree(who, q, k_pool, v_pool, row_offset, pos, parents, o, pool_rows, batch,
                      n_nodes, n_heads, n_kv_heads, head_dim, scale);
  if (st) return st;
  if (!k_new || !v_new) return fail(NWD_ERR_INVALID, "%s: null pointer", who);
  if (!aligned16(k_new) || !aligned16(v_new))
    return fail(NWD_ERR_INVALID, "%s: tensors must be 16-byte aligned", who);
  if (!workspace || ws_bytes < 256 || ((uintptr_t)workspace & 255u))
    return fail(NWD_ERR_WORKSPACE, "%s: needs a 256-byte aligned workspace of >= 256 bytes", who);
  if (batch == 0 || n_nodes == 0) return ok();
  const uint32_t row_vec = n_kv_heads * head_dim / 8;
  const uint32_t bx = (n_nodes * row_vec + 255) / 256;
  tree_append_kernel<<<dim3(bx, batch), 256, 0, (cudaStream_t)stream>>>(
      reinterpret_cast<const uint4*>(k_new), reinterpret_cast<const uint4*>(v_new),
      reinterpret_cast<uint4*>(k_pool), reinterpret_cast<uint4*>(v_pool), row_offset, pos,
      tree_len, pool_rows, n_nodes, row_vec, err);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, who);
  return nwd_attn_tree(q, k_pool, v_pool, pool_rows, row_offset, pos, parents, tree_len, o, batch,
                       n_nodes, n_heads, n_kv_heads, head_dim, scale, workspace, ws_bytes, err,
                       stream);
}

}  // extern "C"
