// Verification of a tree of drafted tokens against the target's
// probabilities, from given uniform numbers (multi-round rejection sampling:
// the tokens that come out are distributed as the target alone would draw
// them).  The reference takes the likeliest token of one row per step
// (engine/runtime.js:395-398); this decides for several positions at once.
//
// The walk starts at node 0 (the pending token, already accepted) with
// r = p[0].  At node i its children c are tried in index order:
//   accepted if u_c * q_i(t_c) < r(t_c): the walk goes on at c with r = p[c];
//   else r = max(r - q_i, 0), renormalised to a sum of 1 (all zero: r = p[i]
//   again).  Without draft rows the drafted tokens count as certain: accepted
//   if u_c < r(t_c), else r(t_c) = 0, renormalised.
// Where no child is left the next token is the lowest x whose running sum of
// r exceeds w * sum(r).
//
// r is kept unnormalised: r~ = max(r~ - S q, 0) with S its previous sum (S = 1
// for p itself), so u_c q S < r~ is the same test without a division, and r~
// at any x is recomputed from p, q and the list of the S of this node's
// rejections.  Products, differences and sums are f64: with f32 sums the
// border between two tokens of a 10^5-token vocabulary would move by about one
// part in 10^7, enough to change a drawn token now and then with the order of
// summation; in f64 the borders hold to 10^-15.
//
// A sequence has a cluster of up to 16 CTAs, each with a contiguous part of the
// vocabulary, its warps with contiguous parts of that.  Every CTA walks the
// tree for itself, on the same numbers: the entries at the drafted tokens,
// fetched for all nodes at once, decide while nothing is rejected.  A rejection
// takes one pass over the row (p and q): each CTA's sum goes to all of them
// through distributed shared memory, one cluster barrier a pass, and is added
// in CTA order, so they agree to the bit.  The last pass at the last node also
// serves the draw.  Without draft rows a node's rejections share one pass: the
// sum over all tokens but its children's, to which the entries of those not
// rejected are added.
//
// Bound by the rows' bytes where there are many sequences: 256 chains of 5 nodes
// over 131 072 tokens read 248 MB in 51 us (4.9 TB/s; the pass itself runs at
// 7, gathers before it and the draw behind it read little).  Else by the
// longest walk, a pass of which is 3 to 5 us (fetching the row's part, its
// conversions to f64 on a pipe of 16 per clock, the differences on one of 64,
// two barriers): 32 trees of 26 nodes 43 us, with 3.1 passes on average and 7
// in one; one chain 8 us with its launch.
#include "nwd_common.h"
#include "tree.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int CTAS_PER_SM = 4;  // 64 registers per thread
constexpr uint32_t MAX_CLUSTER = 16;
constexpr uint32_t MIN_PART = 1024;  // tokens per CTA that make a larger cluster worth its barriers

struct VerifyParams {
  const int32_t* tokens;
  const int32_t* parents;
  const int32_t* tree_len;
  const float* target;
  const float* draft;
  const float* u;
  const float* w;
  int32_t* path;
  int32_t* n_accepted;
  int32_t* next_token;
  uint32_t* err;
  uint32_t n_nodes, vocab, cluster;
};

// A probability as it counts: what is not above zero (NaN too) is zero.
__device__ __forceinline__ double prob(float x) { return x > 0.f ? (double)x : 0.0; }

struct Walk {
  float u[nwd::TREE_MAX_NODES];
  float p[nwd::TREE_MAX_NODES];  // target and draft row of the parent at the token
  float q[nwd::TREE_MAX_NODES];
  int32_t token[nwd::TREE_MAX_NODES];   // -1: outside the vocabulary, never accepted
  double sum[nwd::TREE_MAX_NODES];      // S before each rejection at the current node
  double from[2][MAX_CLUSTER];          // the CTAs' sums of a pass, by its parity
  double part[WARPS];                   // the warps' sums of the last pass
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int i = 16; i; i >>= 1) v += __shfl_xor_sync(0xffffffffu, v, i);
  return v;
}
// Lane i holds part i of a sum: the part that takes it past `goal` (the last
// one with mass, should rounding leave the border behind; -1: none has any),
// and the sum before it.  The same in all lanes, and wherever the parts are.
__device__ __forceinline__ int find_part(double mine, double goal, double* before) {
  const uint32_t lane = threadIdx.x & 31;
  double upto = mine;
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    const double v = __shfl_up_sync(0xffffffffu, upto, i);
    if ((int)lane >= i) upto += v;
  }
  const double ahead = *before + upto;
  const uint32_t mass = __ballot_sync(0xffffffffu, mine > 0.0);
  const uint32_t over = __ballot_sync(0xffffffffu, mine > 0.0 && ahead > goal);
  if (!mass) return -1;
  const int at = over ? __ffs(over) - 1 : 31 - __clz(mass);
  const double up = __shfl_up_sync(0xffffffffu, upto, 1);
  *before += __shfl_sync(0xffffffffu, lane ? up : 0.0, at);
  return at;
}

// max(p - q, 0): r~ of an entry after one rejection (S was 1), with the
// comparison in f32, which is exact, so that the f64 pipe has one difference.
__device__ __forceinline__ double rest1(float p, float q) {
  p = fmaxf(p, 0.f);  // (NaN gives 0)
  q = fmaxf(q, 0.f);
  const bool in = p > q;
  return (double)(in ? p : 0.f) - (double)(in ? q : 0.f);
}
// max(t, 0) by the sign bit: a comparison in f64 would take the pipe that the
// differences need
__device__ __forceinline__ double positive(double t) {
  return __double2hiint(t) < 0 ? 0.0 : t;
}
// r~ of N entries after k rejections at the current node (with draft rows).
template <int N>
__device__ __forceinline__ void rest(const Walk& s, int k, const float* p, const float* q, double* r) {
  double qd[N];  // (two conversions per entry: they bound a pass)
#pragma unroll
  for (int e = 0; e < N; e++) {
    r[e] = prob(p[e]);
    qd[e] = prob(q[e]);
    const double t = r[e] - qd[e];
    if (k) r[e] = positive(t);
  }
#pragma unroll 1
  for (int i = 1; i < k; i++) {
    const double sum = s.sum[i];
#pragma unroll
    for (int e = 0; e < N; e++) {
      r[e] = positive(r[e] - sum * qd[e]);
    }
  }
}

// A row of the vocabulary in groups of four entries from a 16-byte boundary at
// or before its start; entries outside the row read as zero.
struct Row {
  const float* p;
  const float* q;      // nullptr without draft rows
  uint32_t lead, size;  // entries before the row in its first group; entries
  bool vec;            // p and q lie alike: whole groups are single loads
  __device__ __forceinline__ Row(const float* p_, const float* q_, uint32_t size_)
      : p(p_), q(q_), size(size_) {
    lead = (uint32_t)(reinterpret_cast<uintptr_t>(p) >> 2) & 3u;
    vec = !q || ((reinterpret_cast<uintptr_t>(q) >> 2) & 3u) == lead;
  }
  __device__ __forceinline__ uint32_t groups() const { return (size + lead + 3) / 4; }
  __device__ __forceinline__ uint32_t first(uint32_t g) const { return 4 * g - lead; }  // may wrap
  __device__ __forceinline__ float4 load(const float* row, uint32_t g) const {
    const uint32_t x = first(g);
    if (vec && x < size && size - x >= 4)
      return __ldg(reinterpret_cast<const float4*>(row + x));
    float4 v;
    v.x = x < size ? row[x] : 0.f;
    v.y = x + 1 < size ? row[x + 1] : 0.f;
    v.z = x + 2 < size ? row[x + 2] : 0.f;
    v.w = x + 3 < size ? row[x + 3] : 0.f;
    return v;
  }
};

// The tokens taken out of a row (without draft rows): lane l holds those of
// nodes l and l + 32, -1 where there is none.
struct Gone {
  int32_t a, b;
  // Zeroes the ones among the entries v, which are tokens x .. x + 3 of this
  // lane and x0 .. x0 + 127 of the warp (x0 may have wrapped below zero).
  __device__ __forceinline__ void clear(double (&v)[4], uint32_t x, uint32_t x0) const {
#pragma unroll
    for (int half = 0; half < 2; half++) {
      const int32_t mine = half ? b : a;
      uint32_t in = __ballot_sync(0xffffffffu, mine >= 0 && (uint32_t)mine - x0 < 128u);
      for (; in; in &= in - 1) {
        const uint32_t at = (uint32_t)__shfl_sync(0xffffffffu, mine, __ffs(in) - 1) - x;
#pragma unroll
        for (uint32_t i = 0; i < 4; i++)
          if (at == i) v[i] = 0.0;
      }
    }
  }
};

__device__ __forceinline__ void cluster_put(double* slot, uint32_t rank, double v) {
  uint32_t at = (uint32_t)__cvta_generic_to_shared(slot);
  asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(at) : "r"(rank));
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(v) : "memory");
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The warp's groups [lo, hi) of a row, in steps of 32.
struct Part {
  uint32_t lo, hi;
};
__device__ __forceinline__ Part piece(uint32_t groups, uint32_t i, uint32_t pieces) {
  return Part{(uint32_t)((uint64_t)groups * i / pieces),
              (uint32_t)((uint64_t)groups * (i + 1) / pieces)};
}
__device__ __forceinline__ Part warp_part(uint32_t groups, uint32_t rank, uint32_t cluster) {
  return piece(groups, rank * WARPS + (threadIdx.x >> 5), cluster * WARPS);
}

// What r~ is made of: the row alone, p - q once, or the node's rejections one
// after the other.
enum Rest { WHOLE, ONCE, CHAIN };

// The sum of r~ over the warp's groups [lo, hi) of a row, this lane's share;
// AHEAD groups per lane in flight, as many as 64 registers hold (CHAIN with 1: 32
// trees of 26 nodes 48 us, with 3 46, with 2 43).
template <bool DRAFT, int REST>
__device__ __forceinline__ double part_sum(const Walk& s, int k, const Gone& gone, const Row& row,
                                           Part w) {
  constexpr uint32_t AHEAD = REST == WHOLE ? 8 : REST == ONCE ? 4 : 2;
  const uint32_t lane = threadIdx.x & 31;
  double v = 0.0;
  for (uint32_t g0 = w.lo; g0 < w.hi; g0 += 32 * AHEAD) {
    float4 p[AHEAD], q[AHEAD];
#pragma unroll
    for (uint32_t i = 0; i < AHEAD; i++) {
      const uint32_t g = g0 + 32 * i + lane;
      p[i] = q[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (g < w.hi) {
        p[i] = row.load(row.p, g);
        if (REST != WHOLE) q[i] = row.load(row.q, g);
      }
    }
    const float* pe = &p[0].x;
    const float* qe = &q[0].x;
    if (REST == CHAIN) {
      double r[4 * AHEAD];
      rest<4 * AHEAD>(s, k, pe, qe, r);
#pragma unroll
      for (uint32_t i = 0; i < 4 * AHEAD; i++) v += r[i];
    } else {
#pragma unroll
      for (uint32_t i = 0; i < AHEAD; i++) {
        double e[4];
#pragma unroll
        for (uint32_t c = 0; c < 4; c++)
          e[c] = REST == ONCE ? rest1(pe[4 * i + c], qe[4 * i + c]) : prob(pe[4 * i + c]);
        if (!DRAFT) gone.clear(e, row.first(g0 + 32 * i + lane), row.first(g0 + 32 * i));
        v += (e[0] + e[1]) + (e[2] + e[3]);
      }
    }
  }
  return v;
}
template <bool DRAFT>
__device__ __forceinline__ double any_part_sum(const Walk& s, int k, const Gone& gone,
                                               const Row& row, Part w) {
  if (!DRAFT || k == 0) return part_sum<DRAFT, WHOLE>(s, k, gone, row, w);
  if (k == 1) return part_sum<DRAFT, ONCE>(s, k, gone, row, w);
  return part_sum<DRAFT, CHAIN>(s, k, gone, row, w);
}

// The warps' sums, in s.part, added up: the same in every thread of the CTA.
__device__ __forceinline__ double block_sum(Walk& s, double v) {
  const uint32_t lane = threadIdx.x & 31;
  v = warp_sum(v);
  __syncthreads();  // the last pass's s.part has been read
  if (lane == 0) s.part[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum(lane < WARPS ? s.part[lane] : 0.0);
}

// One pass: the sum of r~ over the vocabulary, the same in every thread of the
// cluster; s.part holds this CTA's warps' shares, s.from[parity] the CTAs'.
template <bool DRAFT>
__device__ double row_sum(Walk& s, int k, const Gone& gone, const Row& row, uint32_t rank,
                          uint32_t cluster, uint32_t parity) {
  const uint32_t lane = threadIdx.x & 31;
  const Part w = warp_part(row.groups(), rank, cluster);
  const double t = block_sum(s, any_part_sum<DRAFT>(s, k, gone, row, w));
  if (cluster == 1) return t;
  if (threadIdx.x < cluster) cluster_put(&s.from[parity][rank], threadIdx.x, t);
  cluster_arrive();
  cluster_wait();
  return warp_sum(lane < cluster ? s.from[parity][lane] : 0.0);
}

template <bool DRAFT>
__global__ void __launch_bounds__(THREADS, CTAS_PER_SM) verify_tree_kernel(const VerifyParams a) {
  __shared__ Walk s;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t b = blockIdx.x / a.cluster, rank = blockIdx.x % a.cluster;
  const uint32_t V = a.vocab, N = a.n_nodes;
  const uint64_t node0 = (uint64_t)b * N;
  nwd::pdl_trigger();
  cluster_arrive();  // this CTA has started: its shared memory may be written
  nwd::pdl_wait();
  const uint32_t n = nwd::tree_nodes(a.tree_len, b, N, a.err);
  // every warp has the nodes' parents and tokens, lane l those of l and l + 32
  int par[2] = {-1, -1}, tok[2] = {-1, -1};
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const uint32_t c = lane + 32 * i;
    if (c > 0 && c < n) {
      par[i] = nwd::tree_parent(a.parents + node0, (int)c, a.err);
      tok[i] = a.tokens[node0 + c];
      if (tok[i] < 0 || (uint32_t)tok[i] >= V) {
        if (a.err) atomicOr(a.err, NWD_DEVERR_TREE);
        tok[i] = -1;
      }
    }
  }
  if (warp < 2) {  // warp i: the entries at the tokens of nodes 32 i ..
    const uint32_t c = tid;
    if (c < N) {
      s.token[c] = tok[warp];
      s.u[c] = c < n ? a.u[node0 + c] : 0.f;
      s.p[c] = s.q[c] = 0.f;
      if (par[warp] >= 0 && tok[warp] >= 0) {
        const uint64_t at = (node0 + (uint32_t)par[warp]) * V + (uint32_t)tok[warp];
        s.p[c] = a.target[at];
        s.q[c] = DRAFT ? a.draft[at] : 1.f;
      }
      if (rank == 0) a.path[node0 + c] = -1;
    }
  }
  cluster_wait();  // every CTA of the cluster has
  __syncthreads();
  if (n == 0) {
    if (rank == 0 && tid == 0) {
      a.n_accepted[b] = 0;
      a.next_token[b] = -1;
    }
    return;  // the whole cluster
  }
  const bool scribe = rank == 0 && tid == 0;
  if (scribe) a.path[node0] = 0;
  uint32_t cur = 0, count = 1, parity = 0;
  double total = 1.0;   // S: 1 for p itself, else the sum of r~
  Gone gone{-1, -1};
  bool summed = false;  // the last pass was over r~ as it now is
  for (;;) {
    const Row row(a.target + (node0 + cur) * V, DRAFT ? a.draft + (node0 + cur) * V : nullptr, V);
    const uint64_t children = (uint64_t)__ballot_sync(0xffffffffu, par[1] == (int)cur) << 32 |
                              __ballot_sync(0xffffffffu, par[0] == (int)cur);
    int k = 0;  // rejections that r~ has taken in (since it was last the whole row)
    int next = -1;
    bool have_base = false, first[2] = {false, false};
    double base = 0.0;  // without draft rows: the sum but for the children's tokens
    total = 1.0;
    gone.a = gone.b = -1;
    summed = false;
    for (uint64_t left = children; left; left &= left - 1) {
      const int c = __ffsll((long long)left) - 1;
      const int t = s.token[c];
      if (t >= 0) {
        double r;
        if (DRAFT) rest<1>(s, k, &s.p[c], &s.q[c], &r);
        else r = __any_sync(0xffffffffu, gone.a == t || gone.b == t) ? 0.0 : prob(s.p[c]);
        if ((double)s.u[c] * prob(s.q[c]) * total < r) {
          next = c;
          break;
        }
      }
      if (DRAFT) {
        __syncthreads();
        if (tid == 0) s.sum[k] = total;
        __syncthreads();
        total = row_sum<true>(s, ++k, gone, row, rank, a.cluster, parity);
        parity ^= 1;
        summed = true;
      } else {
        const Gone mine{par[0] == (int)cur ? tok[0] : -1, par[1] == (int)cur ? tok[1] : -1};
        if (!have_base) {  // the children's tokens left out, all at once
          base = row_sum<false>(s, 0, mine, row, rank, a.cluster, parity);
          parity ^= 1;
          have_base = true;
          first[0] = mine.a >= 0;
          first[1] = mine.b >= 0;
          const uint32_t same = __match_any_sync(0xffffffffu, first[0] ? mine.a : -1 - (int)lane);
          if (same & ((1u << lane) - 1u)) first[0] = false;
          for (uint32_t left_b = __ballot_sync(0xffffffffu, first[1]); left_b; left_b &= left_b - 1) {
            const int l = __ffs(left_b) - 1, tb = __shfl_sync(0xffffffffu, mine.b, l);
            const uint32_t ahead = __ballot_sync(0xffffffffu, mine.a == tb);
            const uint32_t ahead_b = __ballot_sync(0xffffffffu, mine.b == tb) & ((1u << l) - 1u);
            if ((int)lane == l && (ahead | ahead_b)) first[1] = false;
          }
        }
        if (t >= 0) {
          if (mine.a == t) gone.a = t;
          if (mine.b == t) gone.b = t;
        }
        // the entries of the children's tokens that are still in, each token
        // once: at its first node
        const bool in[2] = {first[0] && gone.a < 0, first[1] && gone.b < 0};
        summed = !__any_sync(0xffffffffu, in[0] || in[1]);  // the pass left out just those: its
        double more = 0.0;                                   // parts serve the draw
        if (in[0]) more += prob(s.p[lane]);
        if (in[1]) more += prob(s.p[lane + 32]);
        total = base + (summed ? 0.0 : warp_sum(more));
      }
      if (!(total > 0.0)) {  // nothing left: the whole row again
        k = 0;
        total = 1.0;
        gone.a = gone.b = -1;
        summed = false;
      }
    }
    if (next < 0) {
      if (!summed) {
        total = row_sum<DRAFT>(s, k, gone, row, rank, a.cluster, parity);
        parity ^= 1;
      }
      // ---- the draw: the CTA whose part holds the border, then its warp
      const double goal = (double)a.w[b] * total;
      if (scribe) a.n_accepted[b] = (int32_t)count;
      double before = 0.0;
      if (a.cluster > 1) {
        const int cta = find_part(lane < a.cluster ? s.from[parity ^ 1][lane] : 0.0, goal, &before);
        if (cta < 0 && scribe) a.next_token[b] = -1;
        if (cta != (int)rank) return;
      }
      int owner = find_part(lane < WARPS ? s.part[lane] : 0.0, goal, &before);
      if (owner < 0) {  // (a cluster of one: no mass at all)
        if (tid == 0) a.next_token[b] = -1;
        return;
      }
      Part w = piece(row.groups(), rank * WARPS + owner, a.cluster * WARPS);
      while (w.hi - w.lo > 64) {  // all warps on the owner's part
        const uint32_t lo = w.lo, n_all = w.hi - w.lo;
        w = piece(n_all, warp, WARPS);
        w.lo += lo;
        w.hi += lo;
        block_sum(s, any_part_sum<DRAFT>(s, k, gone, row, w));
        owner = find_part(lane < WARPS ? s.part[lane] : 0.0, goal, &before);
        if (owner < 0) break;  // (cannot be: the part has mass)
        w = piece(n_all, (uint32_t)owner, WARPS);
        w.lo += lo;
        w.hi += lo;
      }
      if (warp != 0) return;
      int32_t last = -1;  // the last token with mass, should rounding leave the border behind
      for (uint32_t g0 = w.lo; g0 < w.hi; g0 += 32) {
        const uint32_t g = g0 + lane, x = row.first(g);
        float4 p = make_float4(0.f, 0.f, 0.f, 0.f), q = p;
        if (g < w.hi) {
          p = row.load(row.p, g);
          if (DRAFT) q = row.load(row.q, g);
        }
        double v[4];
        rest<4>(s, k, &p.x, &q.x, v);
        if (!DRAFT) gone.clear(v, x, row.first(g0));
        const double own = ((v[0] + v[1]) + v[2]) + v[3];
        double cum = own;
#pragma unroll
        for (int i = 1; i < 32; i <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, cum, i);
          if ((int)lane >= i) cum += y;
        }
        // within the lane: the first entry that takes the sum past the goal
        double at = before + cum - own;
        int32_t hit = -1, some = -1;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          at += v[i];
          if (v[i] > 0.0) {
            some = (int32_t)(x + i);
            if (hit < 0 && at > goal) hit = some;
          }
        }
        const uint32_t hits = __ballot_sync(0xffffffffu, hit >= 0);
        const uint32_t somes = __ballot_sync(0xffffffffu, some >= 0);
        if (somes) last = __shfl_sync(0xffffffffu, some, 31 - __clz(somes));
        if (hits) {
          last = __shfl_sync(0xffffffffu, hit, __ffs(hits) - 1);
          break;
        }
        before += __shfl_sync(0xffffffffu, cum, 31);
      }
      if (lane == 0) a.next_token[b] = last;
      return;
    }
    if (scribe) a.path[node0 + count] = next;
    count++;
    cur = (uint32_t)next;
  }
}

template <bool DRAFT>
cudaError_t launch_verify(const VerifyParams& a, uint32_t batch, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(batch * a.cluster);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = a.cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, verify_tree_kernel<DRAFT>, a);
}

}  // namespace

using namespace nwd;

extern "C" int nwd_verify_tree(const int32_t* tokens, const int32_t* parents,
                               const int32_t* tree_len, const float* target_probs,
                               const float* draft_probs, const float* u, const float* w,
                               int32_t* path, int32_t* n_accepted, int32_t* next_token,
                               uint32_t batch, uint32_t n_nodes, uint32_t vocab, uint32_t* err,
                               void* stream) {
  const char* who = "nwd_verify_tree";
  if (!tokens || !parents || !target_probs || !u || !w || !path || !n_accepted || !next_token)
    return fail(NWD_ERR_INVALID, "%s: null pointer", who);
  if (n_nodes == 0 || vocab == 0) return fail(NWD_ERR_INVALID, "%s: zero shape", who);
  if (n_nodes > TREE_MAX_NODES)
    return fail(NWD_ERR_UNSUPPORTED, "%s: %u nodes (at most %u)", who, n_nodes, TREE_MAX_NODES);
  if (vocab > 0x7fffffffu) return fail(NWD_ERR_UNSUPPORTED, "%s: vocabulary %u", who, vocab);
  if (batch > 65535u) return fail(NWD_ERR_UNSUPPORTED, "%s: batch > 65535", who);
  if (batch == 0) return ok();
  // The CTAs of a cluster walk the tree each for itself, on the same numbers: an
  // output written over an input that another CTA has yet to read would let them
  // part ways.
  const uint64_t each = (uint64_t)batch * 4, nodes = each * n_nodes;
  const Span span[] = {{"path", path, nodes},
                       {"n_accepted", n_accepted, each},
                       {"next_token", next_token, each},
                       {"tokens", tokens, nodes},
                       {"parents", parents, nodes},
                       {"tree_len", tree_len, each},
                       {"target_probs", target_probs, nodes * vocab},
                       {"draft_probs", draft_probs, nodes * vocab},
                       {"u", u, nodes},
                       {"w", w, each},
                       {"err", err, 4}};
  for (uint32_t i = 0; i < 3; i++)
    for (uint32_t j = i + 1; j < sizeof(span) / sizeof(span[0]); j++)
      if (overlap(span[i], span[j]))
        return fail(NWD_ERR_INVALID, "%s: %s and %s must not overlap", who, span[i].name,
                    span[j].name);
  DeviceInfo di;
  int st = current_device_info(&di);
  if (st) return st;
  static bool wide_set[64] = {};  // clusters of 16 allowed, per device
  if (!wide_set[di.device]) {
    cudaError_t e = cudaFuncSetAttribute(verify_tree_kernel<true>,
                                         cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(verify_tree_kernel<false>,
                               cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(verify_tree_kernel)");
    wide_set[di.device] = true;
  }
  // The largest cluster that leaves all CTAs resident at once and each a part
  // of the vocabulary worth a barrier.  Up to 16, 8, 4 and 1 CTAs: one chain
  // over 131 072 tokens 8.0, 10.0, 13.8 and 34 us, 32 trees 43, 65, 99 and 334;
  // 256 chains, which get two, 51 and with one 67.
  uint32_t cluster = 1;
  while (cluster < MAX_CLUSTER && (uint64_t)batch * cluster * 2 <= (uint64_t)di.sm_count * CTAS_PER_SM &&
         vocab / (cluster * 2) >= MIN_PART)
    cluster *= 2;
  const VerifyParams a{tokens, parents,    tree_len,   target_probs, draft_probs, u,       w,
                       path,   n_accepted, next_token, err,          n_nodes,     vocab,   cluster};
  cudaError_t e = draft_probs ? launch_verify<true>(a, batch, (cudaStream_t)stream)
                              : launch_verify<false>(a, batch, (cudaStream_t)stream);
  if (e != cudaSuccess) return cuda_fail(e, who);
  return ok();
}
