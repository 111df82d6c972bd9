// Attention for the tree of one short sequence (tree_attn.cu has the formula,
// the masks and the roundings), for instance a cache of the engine's 256 rows.
//
// There the general kernel's append, plan, pipeline fill and join are nearly
// all of its time.  Here a kv head is one CTA of 16 warps, or past 128 pool
// rows a thread-block cluster of up to 8, each with an equal part of the
// context and tree rows in shared memory, and one launch does it all:
//   S    a warp has 16 cache rows and all query rows (up to 64, as 16-row
//        tiles): mma.sync m16n8k16, Q and K through ldmatrix;
//   P    against the CTA's maximum per row, as fp16 head and fp16 remainder
//        into shared memory, its largest 2^15;
//   O    a warp has 16 output columns and every other row tile, so that P, which
//        all warps read, crosses shared memory half as often;
//   out  normalised, or joined over the cluster through distributed shared
//        memory, each CTA a share of the rows.
// With the append, tree rows come from k_new / v_new and are written to the
// pool by the CTA that has them.
//
// mma.sync: tcgen05 would need its tensor memory, descriptors and barriers set
// up for 40 rows x 158 keys of work.
//
// Bound by latency: launch, lengths, rows, then S, P and O with a barrier after
// each (about 1 us a stage at 40 query rows, most of it shared-memory reads).
// 40/8 heads, with the append, and the general kernel's time: 8 nodes over 150
// rows 7.5 us (11.7), over 1 000 9.8 (13.8), over 2 000 12.7 (14.7); 12 nodes
// over 2 000 14.3 (14.7); one node over 150 5.2 (11.7).
#include <cuda_fp16.h>

#include <algorithm>

#include "nwd_common.h"
#include "tree.cuh"

namespace {

constexpr uint32_t HD = 128;
constexpr uint32_t THREADS = 512, WARPS = THREADS / 32;
constexpr uint32_t MAX_ROWS = 64;      // query rows per kv head
constexpr uint32_t MAX_KEYS = 256;     // cache rows per CTA
constexpr uint32_t MAX_CLUSTER = 8;    // portable cluster size
// Up to ONE_KEYS pool rows are one CTA's, more are shared out by CLUSTER_KEYS.  A
// cluster's launch and barriers cost what 64 rows do: 8 nodes over 120 rows 7.2
// us in one CTA, 7.4 in a cluster; over 150 8.0 and 7.5; over 240 10.2 and 7.6, by
// 32 rows 7.9, by 128 9.4.
constexpr uint32_t ONE_KEYS = 128, CLUSTER_KEYS = 64;
constexpr float P_BIAS = 15.f;
static_assert(ONE_KEYS <= MAX_KEYS && MAX_KEYS == WARPS * 16 && HD == WARPS / 2 * 16 && MAX_ROWS * 8 == THREADS, "the warps' shares");

struct Params {
  const __half* q;
  const __half* k_new;  // nullptr: the rows are in the pools
  const __half* v_new;
  __half* k_pool;
  __half* v_pool;
  __half* o;
  const int64_t* row_offset;
  const int32_t* seq_len;
  const int32_t* parents;
  const int32_t* tree_len;
  const int32_t* capacity;
  uint32_t* err;
  uint64_t pool_rows;
  uint32_t n_nodes, n_heads, n_kv, group, cluster, keys;  // keys: a CTA's room, a multiple of 32
  float scale_log2;
};

__device__ __forceinline__ uint32_t s_u32(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// byte offset of 16-byte chunk c (0-15) of row r in a [rows][256 B] tile, the
// chunk index XOR-swizzled by the row
__device__ __forceinline__ uint32_t sw_off(uint32_t r, uint32_t c) {
  return r * 256u + ((c & 8u) | ((c ^ r) & 7u)) * 16u;
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
// the address that `local` has in CTA `rank` of the cluster
template <bool CLUSTER>
__device__ __forceinline__ uint32_t cluster_at(const void* local, uint32_t rank) {
  if (!CLUSTER) return s_u32(local);
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(s_u32(local)), "r"(rank));
  return at;
}

// Shared memory: K (later the CTA's O, f32), V, Q, P's heads and remainders, then what follows.
struct Tail {
  uint64_t sees[nwd::TREE_MAX_NODES];  // the rows of the tree that a node sees
  float2 ml[MAX_ROWS];
  float wmax[WARPS][MAX_ROWS];
  float wsum[WARPS][MAX_ROWS];
  unsigned int bad[2];  // rows of the tree with NaN or infinities in V
  uint8_t node[MAX_ROWS];  // of a query row
};
__host__ __device__ inline uint32_t k_bytes(uint32_t keys, uint32_t rows) {
  return keys * 256u > rows * HD * 4u ? keys * 256u : rows * HD * 4u;
}
__host__ __device__ inline uint32_t p_bytes(uint32_t keys, uint32_t rows) {
  return (keys + 127u) / 128u * rows * 256u;  // [128 keys][rows][256 B], of heads or remainders
}
inline uint32_t smem_bytes(uint32_t keys, uint32_t rows) {
  return k_bytes(keys, rows) + keys * 256u + rows * 256u + 2 * p_bytes(keys, rows) + (uint32_t)sizeof(Tail);
}

template <int MT, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, 1) tree_short_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) uint8_t sm[];
  constexpr uint32_t ROWS = MT * 16;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t g = lane >> 2, t = lane & 3;
  const uint32_t hkv = CLUSTER ? blockIdx.x / p.cluster : blockIdx.x;
  const uint32_t rank = CLUSTER ? blockIdx.x % p.cluster : 0u;
  uint8_t* ks = sm;
  uint8_t* vs = ks + k_bytes(p.keys, ROWS);
  uint8_t* qs = vs + p.keys * 256u;
  uint8_t* ps = qs + ROWS * 256u;
  const uint32_t rem = p_bytes(p.keys, ROWS);  // from a head to its remainder
  Tail& s = *reinterpret_cast<Tail*>(ps + 2 * rem);
  const uint32_t rows = p.n_nodes * p.group;  // of MT * 16

  nwd::pdl_trigger();
  nwd::pdl_wait();
  int2 par = make_int2(-1, -1);  // (asked for first, needed last)
  if (warp == WARPS - 1) {
    if (lane < p.n_nodes) par.x = p.parents[lane];
    if (lane + 32 < p.n_nodes) par.y = p.parents[lane + 32];
  }
  const nwd::TreeRaw raw = nwd::tree_raw(p.row_offset, p.seq_len, p.tree_len, p.capacity, 0,
                                         p.n_nodes);
  const uint32_t kb = s_u32(ks), vb = s_u32(vs), qb = s_u32(qs), pb = s_u32(ps);

  // ---- Q and K, then V, into shared memory ----
  for (uint32_t i = tid; i < ROWS * 16; i += THREADS) {
    const uint32_t r = i >> 4, c = i & 15, node = r / p.group;
    if (r < rows)
      cp16(qb + sw_off(r, c),
           p.q + ((size_t)node * p.n_heads + hkv * p.group + r - node * p.group) * HD + c * 8);
    else
      *reinterpret_cast<uint4*>(qs + sw_off(r, c)) = make_uint4(0u, 0u, 0u, 0u);
    if (c == 0) s.node[r] = (uint8_t)node;
  }
  const nwd::TreeSeq seq = nwd::tree_seq(raw, p.pool_rows, p.n_nodes,
                                         blockIdx.x == 0 && tid == 0 ? p.err : nullptr);
  // this CTA's rows of the sequence: [lo, lo + n); at most p.keys, as the
  // sequence fits the pool
  const uint32_t total = seq.nodes ? seq.ctx + seq.nodes : 0u;
  const uint32_t lo = CLUSTER ? total * rank / p.cluster : 0u;
  const uint32_t n = (CLUSTER ? total * (rank + 1) / p.cluster : total) - lo;
  const uint64_t first_row = ((uint64_t)seq.row0 + lo) * p.n_kv + hkv;  // of the pools
  auto copy = [&](uint32_t dst, const __half* pool, const __half* fresh) {
    for (uint32_t i = tid; i < n * 16; i += THREADS) {
      const uint32_t r = i >> 4, c = i & 15;
      const __half* src = pool + (first_row + (uint64_t)r * p.n_kv) * HD + c * 8;
      if (fresh && lo + r >= seq.ctx)
        src = fresh + ((size_t)(lo + r - seq.ctx) * p.n_kv + hkv) * HD + c * 8;
      cp16(dst + sw_off(r, c), src);
    }
  };
  copy(kb, p.k_pool, p.k_new);
  asm volatile("cp.async.commit_group;" ::: "memory");
  copy(vb, p.v_pool, p.v_new);
  asm volatile("cp.async.commit_group;" ::: "memory");
  // V rows behind the last one in its group of 16: P is 0 there, but 0 x NaN would not be
  for (uint32_t i = n * 16 + tid; i < (n + 15) / 16 * 256; i += THREADS)
    *reinterpret_cast<uint4*>(vs + sw_off(i >> 4, i & 15)) = make_uint4(0u, 0u, 0u, 0u);
  if (warp == WARPS - 1) {
    uint64_t seen[2];
    nwd::tree_closure(par, seq.nodes, blockIdx.x == 0 ? p.err : nullptr, seen);
    s.sees[lane] = lane < seq.nodes ? seen[0] : 0;
    s.sees[lane + 32] = lane + 32 < seq.nodes ? seen[1] : 0;
    if (lane < 2) s.bad[lane] = 0;
  }
  asm volatile("cp.async.wait_group 1;" ::: "memory");
  __syncthreads();
  // the first of the chunks that this thread copied in a row of the tree
  const uint32_t fresh0 = (seq.ctx > lo ? seq.ctx - lo : 0u) * 16;
  const uint32_t fresh_i = fresh0 + ((tid - fresh0) & (THREADS - 1));
  auto append = [&](__half* pool, uint32_t i, uint4 x) {
    *reinterpret_cast<uint4*>(pool + (first_row + (uint64_t)(i >> 4) * p.n_kv) * HD + (i & 15) * 8) = x;
  };

  // ---- S of this warp's 16 cache rows ----
  const uint32_t key0 = warp * 16, mi = lane >> 3, mr = lane & 7;
  float sc[MT][2][4];
#pragma unroll
  for (int m = 0; m < MT; m++)
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int e = 0; e < 4; e++) sc[m][h][e] = 0.f;
  if (key0 < n) {
#pragma unroll
    for (uint32_t k = 0; k < 8; k++) {
      uint32_t b[4];
      ldsm_x4(kb + sw_off(key0 + mr + (mi >> 1) * 8, 2 * k + (mi & 1)), b);
#pragma unroll
      for (uint32_t m = 0; m < (uint32_t)MT; m++) {
        uint32_t a[4];
        ldsm_x4(qb + sw_off(m * 16 + (lane & 15), 2 * k + (lane >> 4)), a);
        mma16816(sc[m][0], a, b[0], b[1]);
        mma16816(sc[m][1], a, b[2], b[3]);
      }
    }
    // bit k: this row attends key0 + k (context rows, then the tree's it sees)
    const uint32_t before = seq.ctx > lo + key0 ? min(seq.ctx - lo - key0, 16u) : 0u;
    const uint32_t have = n - key0 >= 16 ? 0xffffu : (1u << (n - key0)) - 1u;
    const uint32_t skip = lo + key0 + before - seq.ctx;  // tree rows before (if any is here)
    const bool tail = before < 16;
#pragma unroll
    for (uint32_t m = 0; m < (uint32_t)MT; m++) {
#pragma unroll
      for (uint32_t half = 0; half < 2; half++) {  // rows m * 16 + g, and 8 further
        const uint32_t row = m * 16 + g + half * 8;
        uint32_t vis = have;
        if (tail) vis &= (uint32_t)(s.sees[s.node[row]] >> skip) << before | ((1u << before) - 1u);
        float mx = -INFINITY;
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
          float& x = sc[m][i >> 1][half * 2 + (i & 1)];
          x = (vis >> ((i >> 1) * 8 + 2 * t + (i & 1))) & 1u ? x * p.scale_log2 : -INFINITY;
          mx = fmaxf(mx, x);
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        if (t == 0) s.wmax[warp][row] = mx;
      }
    }
  }
  __syncthreads();
  const uint32_t used = (n + 15) / 16;  // warps with cache rows
  // over the warps: eight threads per row
  if (tid < ROWS * 8) {
    float mx = -INFINITY;
    for (uint32_t w = tid & 7; w < used; w += 8) mx = fmaxf(mx, s.wmax[w][tid >> 3]);
#pragma unroll
    for (int i = 1; i < 8; i <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, i));
    if ((tid & 7) == 0) s.ml[tid >> 3].x = mx;
  }
  __syncthreads();

  // ---- P, and its sums ----
  if (key0 < n) {
#pragma unroll
    for (uint32_t m = 0; m < (uint32_t)MT; m++) {
#pragma unroll
      for (uint32_t half = 0; half < 2; half++) {
        const uint32_t row = m * 16 + g + half * 8;
        const float mx = s.ml[row].x, nb = mx == -INFINITY ? 0.f : P_BIAS - mx;
        float sum = 0.f;
#pragma unroll
        for (uint32_t h = 0; h < 2; h++) {
          const float e0 = ex2(sc[m][h][half * 2] + nb), e1 = ex2(sc[m][h][half * 2 + 1] + nb);
          sum += e0 + e1;
          const __half2 head = __floats2half2_rn(e0, e1);
          const float2 taken = __half22float2(head);
          const uint32_t key = key0 + h * 8;
          uint8_t* at = ps + (key >> 7) * (ROWS * 256u) + sw_off(row, (key & 127u) >> 3) + t * 4;
          *reinterpret_cast<__half2*>(at) = head;
          *reinterpret_cast<__half2*>(at + rem) = __floats2half2_rn(e0 - taken.x, e1 - taken.y);
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (t == 0) s.wsum[warp][row] = sum;
      }
    }
  }
  // ---- the tree's rows, each thread in what it copied: into the pools, then NaN and infinities
  // are taken out of V ----
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  for (uint32_t i = fresh_i; i < n * 16; i += THREADS) {
    const uint32_t r = i >> 4;
    uint4* at = reinterpret_cast<uint4*>(vs + sw_off(r, i & 15));
    uint4 x = *at;
    if (p.v_new) {
      append(p.v_pool, i, x);
      append(p.k_pool, i, *reinterpret_cast<const uint4*>(ks + sw_off(r, i & 15)));
    }
    uint32_t* w = &x.x;
    bool hit = false;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const bool a = (w[k] & 0x7c00u) == 0x7c00u, b = (w[k] & 0x7c000000u) == 0x7c000000u;
      hit |= a | b;
      if (a) w[k] &= 0xffff0000u;
      if (b) w[k] &= 0x0000ffffu;
    }
    if (hit) {
      *at = x;
      const uint32_t j = lo + r - seq.ctx;
      atomicOr(&s.bad[j >> 5], 1u << (j & 31));
    }
  }
  __syncthreads();
  if (tid < ROWS * 8) {
    float sum = 0.f;
    for (uint32_t w = tid & 7; w < used; w += 8) sum += s.wsum[w][tid >> 3];
#pragma unroll
    for (int i = 1; i < 8; i <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
    if ((tid & 7) == 0) s.ml[tid >> 3].y = sum;
  }

  // ---- O: 16 columns, every other row tile ----
  constexpr uint32_t OT = (MT + 1) / 2;
  const uint32_t col0 = warp / 2 * 16, tile0 = warp & 1;
  float acc[OT][2][4];
#pragma unroll
  for (uint32_t m = 0; m < OT; m++)
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int e = 0; e < 4; e++) acc[m][h][e] = 0.f;
  if (tile0 < (uint32_t)MT) {
#pragma unroll 2
    for (uint32_t k = 0; k < used; k++) {  // 16 cache rows
      const uint32_t key = k * 16;
      uint32_t b[4];
      ldsm_x4_t(vb + sw_off(key + (lane & 15), col0 / 8 + (lane >> 4)), b);
#pragma unroll
      for (uint32_t m = 0; m < OT; m++) {
        if (tile0 + 2 * m < (uint32_t)MT) {
          const uint32_t at =
              pb + (key >> 7) * (ROWS * 256u) +
              sw_off((tile0 + 2 * m) * 16 + (lane & 15), ((key & 127u) >> 3) + (lane >> 4));
          uint32_t a[4], a1[4];
          ldsm_x4(at, a);
          ldsm_x4(at + rem, a1);
          mma16816(acc[m][0], a, b[0], b[1]);
          mma16816(acc[m][1], a, b[2], b[3]);
          mma16816(acc[m][0], a1, b[0], b[1]);
          mma16816(acc[m][1], a1, b[2], b[3]);
        }
      }
    }
  }
  auto out = [&](uint32_t row, uint32_t node, uint32_t col) {
    return p.o + ((size_t)node * p.n_heads + hkv * p.group + row - node * p.group) * HD + col;
  };
  if (!CLUSTER) {
    __syncthreads();  // s.ml
    if (!(s.bad[0] | s.bad[1])) {  // nearly always
#pragma unroll
      for (uint32_t m = 0; m < OT; m++) {
#pragma unroll
        for (uint32_t half = 0; half < 2; half++) {
          const uint32_t row = (tile0 + 2 * m) * 16 + g + half * 8;
          if (row >= rows || tile0 + 2 * m >= (uint32_t)MT) continue;
          const uint32_t node = s.node[row];
          const float l = s.ml[row].y, inv = l != 0.f && node < seq.nodes ? 1.f / l : 0.f;
          __half* dst = out(row, node, col0 + 2 * t);
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const __half2 x = __floats2half2_rn(acc[m][h][half * 2] * inv, acc[m][h][half * 2 + 1] * inv);
            *reinterpret_cast<__half2*>(dst + h * 8) =
                node < seq.nodes ? x : __floats2half2_rn(0.f, 0.f);
          }
        }
      }
      return;
    }
  }
  // ---- into K's place (every warp is through with it), then out ----
  float* co = reinterpret_cast<float*>(ks);
#pragma unroll
  for (uint32_t m = 0; m < OT; m++) {
    if (tile0 + 2 * m < (uint32_t)MT) {
#pragma unroll
      for (uint32_t i = 0; i < 4; i++) {  // column half i & 1, rows g and g + 8
        const uint32_t row = (tile0 + 2 * m) * 16 + g + (i >> 1) * 8;
        *reinterpret_cast<float2*>(co + row * HD + col0 + (i & 1) * 8 + 2 * t) =
            make_float2(acc[m][i & 1][(i >> 1) * 2], acc[m][i & 1][(i >> 1) * 2 + 1]);
      }
    }
  }
  if (CLUSTER) cluster_sync();
  else __syncthreads();
  constexpr uint32_t MOST = CLUSTER ? MAX_CLUSTER : 1;
#pragma unroll 1
  for (uint32_t i = rank * THREADS + tid; i < rows * (HD / 4); i += (CLUSTER ? p.cluster : 1) * THREADS) {
    const uint32_t row = i / (HD / 4), col = i % (HD / 4) * 4, node = s.node[row];
    float2 ml[MOST];
    float4 x[MOST];
    uint64_t bad = 0;
    float mx = -INFINITY;
#pragma unroll
    for (uint32_t c = 0; c < MOST; c++) {
      ml[c] = make_float2(-INFINITY, 0.f);
      if (!CLUSTER || c < p.cluster) {
        uint32_t b0, b1;
        asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];"
                     : "=f"(ml[c].x), "=f"(ml[c].y)
                     : "r"(cluster_at<CLUSTER>(&s.ml[row], c))
                     : "memory");
        asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                     : "=f"(x[c].x), "=f"(x[c].y), "=f"(x[c].z), "=f"(x[c].w)
                     : "r"(cluster_at<CLUSTER>(co + row * HD + col, c))
                     : "memory");
        asm volatile("ld.shared::cluster.v2.u32 {%0,%1}, [%2];"
                     : "=r"(b0), "=r"(b1)
                     : "r"(cluster_at<CLUSTER>(s.bad, c))
                     : "memory");
        bad |= (uint64_t)b1 << 32 | b0;
        mx = fmaxf(mx, ml[c].x);
      }
    }
    float l = 0.f;
    float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t c = 0; c < MOST; c++) {
      if (ml[c].y != 0.f) {  // a part without weights counts for nothing (l may be NaN)
        const float e = ex2(ml[c].x - mx);
        l += ml[c].y * e;
        y[0] += x[c].x * e;
        y[1] += x[c].y * e;
        y[2] += x[c].z * e;
        y[3] += x[c].w * e;
      }
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int k = 0; k < 4; k++) y[k] *= inv;
    // what was taken out of V comes back for the rows that see it
    for (uint64_t from = bad & s.sees[node]; from; from &= from - 1) {
      const uint32_t j = (uint32_t)__ffsll((long long)from) - 1;
      const __half* src =
          (p.v_new ? p.v_new + ((size_t)j * p.n_kv + hkv) * HD
                   : p.v_pool + (((uint64_t)seq.row0 + seq.ctx + j) * p.n_kv + hkv) * HD) + col;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const float e = __half2float(src[k]);
        if (!isfinite(e)) y[k] += e;
      }
    }
    if (node >= seq.nodes) y[0] = y[1] = y[2] = y[3] = 0.f;
    const __half2 h[2] = {__floats2half2_rn(y[0], y[1]), __floats2half2_rn(y[2], y[3])};
    *reinterpret_cast<uint2*>(out(row, node, col)) = *reinterpret_cast<const uint2*>(h);
  }
  if (CLUSTER) {  // no CTA leaves while another may still read its shared memory
    __syncwarp();
    cluster_sync();
  }
}

template <int MT>
cudaError_t launch(const Params& p, uint32_t smem, int device, cudaStream_t stream) {
  const bool cl = p.cluster > 1;
  auto* kernel = cl ? tree_short_kernel<MT, true> : tree_short_kernel<MT, false>;
  static bool set[64][2] = {};
  if (device >= 64 || !set[device][cl]) {
    const cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)smem_bytes(MAX_KEYS, MT * 16));
    if (e != cudaSuccess) return e;
    if (device < 64) set[device][cl] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.n_kv * p.cluster);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cl ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace

namespace nwd {

bool tree_short_fits(uint64_t pool_rows, uint32_t batch, uint32_t rows) {
  return batch == 1 && rows <= MAX_ROWS && pool_rows <= TREE_SHORT_ROWS;
}

int launch_tree_short(const TreeShortArgs& a, const char* who) {
  static_assert(TREE_SHORT_ROWS <= MAX_KEYS * MAX_CLUSTER, "a CTA's room");
  DeviceInfo di;
  int st = current_device_info(&di);
  if (st) return st;
  const uint32_t group = a.n_heads / a.n_kv, rows = a.n_nodes * group;
  Params p{};
  p.q = reinterpret_cast<const __half*>(a.q);
  p.k_new = reinterpret_cast<const __half*>(a.k_new);
  p.v_new = reinterpret_cast<const __half*>(a.v_new);
  p.k_pool = reinterpret_cast<__half*>(a.k_pool);
  p.v_pool = reinterpret_cast<__half*>(a.v_pool);
  p.o = reinterpret_cast<__half*>(a.o);
  p.row_offset = a.row_offset;
  p.seq_len = a.seq_len;
  p.parents = a.parents;
  p.tree_len = a.tree_len;
  p.capacity = a.capacity;
  p.err = a.err;
  p.pool_rows = a.pool_rows;
  p.n_nodes = a.n_nodes;
  p.n_heads = a.n_heads;
  p.n_kv = a.n_kv;
  p.group = group;
  p.scale_log2 = a.scale_log2;
  const uint32_t most = (uint32_t)a.pool_rows;
  p.cluster = most <= ONE_KEYS ? 1 : std::min(MAX_CLUSTER, (most + CLUSTER_KEYS - 1) / CLUSTER_KEYS);
  p.keys = ((most + p.cluster - 1) / p.cluster + 31) / 32 * 32;
  const uint32_t mt = (rows + 15) / 16, smem = smem_bytes(p.keys, mt * 16);
  cudaStream_t s = (cudaStream_t)a.stream;
  const cudaError_t e = mt == 1   ? launch<1>(p, smem, di.device, s)
                        : mt == 2 ? launch<2>(p, smem, di.device, s)
                        : mt == 3 ? launch<3>(p, smem, di.device, s)
                                  : launch<4>(p, smem, di.device, s);
  if (e != cudaSuccess) return cuda_fail(e, who);
  return ok();
}

}  // namespace nwd
