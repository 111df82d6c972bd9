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
// One CTA per sequence; a pass over a row gives each warp a contiguous part.
#include "nwd_common.h"
#include "tree.cuh"

namespace {

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;

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
  uint32_t n_nodes, vocab;
};

// A probability as it counts: what is not above zero (NaN too) is zero.
__device__ __forceinline__ double prob(float x) { return x > 0.f ? (double)x : 0.0; }

struct Walk {
  int32_t parent[nwd::TREE_MAX_NODES];
  int32_t token[nwd::TREE_MAX_NODES];  // -1: outside the vocabulary, never accepted
  float u[nwd::TREE_MAX_NODES];
  float p[nwd::TREE_MAX_NODES];  // target and draft row of the parent at the token
  float q[nwd::TREE_MAX_NODES];
  double sum[nwd::TREE_MAX_NODES];       // S before each rejection at the current node
  int32_t gone[nwd::TREE_MAX_NODES];     // tokens rejected at the current node
  double part[WARPS];
  int32_t found;
};

// r~ at token x after k rejections at the current node.
template <bool DRAFT>
__device__ __forceinline__ double rest_at(const Walk& s, int k, uint32_t x, float p, float q) {
  double r = prob(p);
  if (DRAFT) {
    const double qd = prob(q);
    for (int i = 0; i < k; i++) r = fmax(r - s.sum[i] * qd, 0.0);
  } else {
    for (int i = 0; i < k; i++)
      if (s.gone[i] == (int32_t)x) r = 0.0;
  }
  return r;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int i = 16; i; i >>= 1) v += __shfl_xor_sync(0xffffffffu, v, i);
  return v;
}

// The sum of r~ over the vocabulary; s.part holds the warps' shares of it.
template <bool DRAFT>
__device__ double row_sum(Walk& s, int k, const float* p, const float* q, uint32_t lo, uint32_t hi) {
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double v = 0.0;
  for (uint32_t x = lo + lane; x < hi; x += 32)
    v += rest_at<DRAFT>(s, k, x, p[x], DRAFT ? q[x] : 0.f);
  v = warp_sum(v);
  __syncthreads();
  if (lane == 0) s.part[warp] = v;
  __syncthreads();
  double t = 0.0;
  for (int i = 0; i < WARPS; i++) t += s.part[i];
  return t;
}

template <bool DRAFT>
__global__ void __launch_bounds__(THREADS) verify_tree_kernel(const VerifyParams a) {
  __shared__ Walk s;
  const uint32_t b = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t V = a.vocab, N = a.n_nodes;
  const uint64_t node0 = (uint64_t)b * N;
  const uint32_t n = nwd::tree_nodes(a.tree_len, b, N, a.err);
  if (tid < N) a.path[node0 + tid] = -1;
  if (n == 0) {
    if (tid == 0) {
      a.n_accepted[b] = 0;
      a.next_token[b] = -1;
    }
    return;
  }
  if (tid < n) {
    const int par = nwd::tree_parent(a.parents + node0, (int)tid, a.err);
    int tok = a.tokens[node0 + tid];
    if (tid > 0 && (tok < 0 || (uint32_t)tok >= V)) {
      if (a.err) atomicOr(a.err, NWD_DEVERR_TREE);
      tok = -1;
    }
    s.parent[tid] = par;
    s.token[tid] = tok;
    s.u[tid] = a.u[node0 + tid];
    if (par >= 0 && tok >= 0) {
      const uint64_t at = (node0 + (uint32_t)par) * V + (uint32_t)tok;
      s.p[tid] = a.target[at];
      s.q[tid] = DRAFT ? a.draft[at] : 1.f;
    }
  }
  __syncthreads();
  const uint32_t lo = (uint32_t)((uint64_t)V * warp / WARPS);
  const uint32_t hi = (uint32_t)((uint64_t)V * (warp + 1) / WARPS);
  uint32_t cur = 0, count = 1;
  int k = 0;          // rejections that r~ has taken in at `cur`
  double total = 1.0; // S: 1 for p itself, else the sum of r~
  if (tid == 0) a.path[node0] = 0;
  for (uint32_t c = 1; c < n; c++) {
    if (s.parent[c] != (int32_t)cur) continue;
    const float* p = a.target + (node0 + cur) * V;
    const float* q = DRAFT ? a.draft + (node0 + cur) * V : nullptr;
    const int tok = s.token[c];
    const double r = tok < 0 ? 0.0 : rest_at<DRAFT>(s, k, (uint32_t)tok, s.p[c], s.q[c]);
    if (tok >= 0 && (double)s.u[c] * prob(s.q[c]) * total < r) {
      if (tid == 0) a.path[node0 + count] = (int32_t)c;
      count++;
      cur = c;
      k = 0;
      total = 1.0;
      continue;
    }
    __syncthreads();
    if (tid == 0) {
      s.sum[k] = total;
      s.gone[k] = tok;
    }
    __syncthreads();
    total = row_sum<DRAFT>(s, ++k, p, q, lo, hi);
    if (!(total > 0.0)) {
      k = 0;
      total = 1.0;
    }
  }
  const float* p = a.target + (node0 + cur) * V;
  const float* q = DRAFT ? a.draft + (node0 + cur) * V : nullptr;
  total = row_sum<DRAFT>(s, k, p, q, lo, hi);
  // the warp whose part holds the border, then its rows of 32
  const double goal = (double)a.w[b] * total;
  double before = 0.0, mine = 0.0;
  int owner = -1;
  for (int i = 0; i < WARPS; i++) {
    const double v = s.part[i];
    if (v > 0.0) {
      owner = i;
      before = mine;
      if (mine + v > goal) break;
    }
    mine += v;
  }
  if (tid == 0) {
    a.n_accepted[b] = (int32_t)count;
    if (owner < 0) a.next_token[b] = -1;
  }
  if ((int)warp != owner) return;
  int32_t last = -1;  // the last token with a probability, should rounding leave the border behind
  for (uint32_t x0 = lo; x0 < hi; x0 += 32) {
    const uint32_t x = x0 + lane;
    const double v = x < hi ? rest_at<DRAFT>(s, k, x, p[x], DRAFT ? q[x] : 0.f) : 0.0;
    double cum = v;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, cum, i);
      if ((int)lane >= i) cum += y;
    }
    const uint32_t some = __ballot_sync(0xffffffffu, v > 0.0);
    const uint32_t over = __ballot_sync(0xffffffffu, v > 0.0 && before + cum > goal);
    if (some) last = (int32_t)(x0 + 31 - __clz(some));
    if (over) {
      last = (int32_t)(x0 + __ffs(over) - 1);
      break;
    }
    before += __shfl_sync(0xffffffffu, cum, 31);
  }
  if (lane == 0) a.next_token[b] = last;
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
  VerifyParams a{tokens, parents,    tree_len,   target_probs, draft_probs, u,     w, path,
                 n_accepted, next_token, err, n_nodes, vocab};
  if (draft_probs)
    verify_tree_kernel<true><<<batch, THREADS, 0, (cudaStream_t)stream>>>(a);
  else
    verify_tree_kernel<false><<<batch, THREADS, 0, (cudaStream_t)stream>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, who);
  return ok();
}
