// Attention for a tree of drafted tokens over the KV pool, on the
// 5th-generation tensor cores (tcgen05.mma, accumulators in tensor memory).
//
// Node i of sequence b sits at pool row row_offset[b] + seq_len[b] + i and
// attends the seq_len[b] context rows, its ancestors' rows and its own:
//   O[b,i,h] = softmax_t(scale * q[b,i,h] . K[t, h/group]) V[t, h/group].
// The reference decodes one token per step (engine/runtime.js:447-467): a
// chain of n nodes computes what n of its steps would, a tree several such
// chains that share their beginnings, over one read of the cache.
//
// Tiles.  The n_nodes * group query rows of a kv head (node-major) are cut
// into tiles of whole nodes, at most 128 rows: the M of an MMA.  A unit is a
// (sequence, kv head) with one or two of its tiles, a block 64 cache rows.
// Tiles past tree_len are no units: the planner writes their rows' zeros.
// The blocks of all units form one line that is cut into an equal range per
// persistent CTA (one per SM); a unit that a cut divides leaves one partial
// (m, l, O) per CTA in the workspace, which merge_kernel joins in order.
//
// A CTA's 20 warps:
//   warps 0, 1    TMA producers: K blocks into 5 stages; V blocks into 5 and
//                 each unit's Q tiles into 2 (as 64-column chunks, 128-byte
//                 swizzle: the K-major operand layout).  Warp 0 also owns the
//                 tensor memory.
//   warp 2        makes V blocks with rows of the tree, or behind it, fit to
//                 multiply (below).
//   warp 3        plans: finds this CTA's range and hands its pieces (blocks of
//                 one unit) to the other warps through a ring of descriptors.
//                 (Nine roles that each walked the sequences for themselves
//                 made the kernel larger than the instruction cache, and a
//                 unit's end cost 5 to 9 us.)
//   warps 4 - 7   MMA issuers: S of softmax group 0, of group 1, P V of group
//                 0, of group 1.  A turn is S = Q K^T of one (block, tile) and
//                 O += P V after its softmax; S runs two turns ahead into the
//                 other of the group's two score buffers, so the softmax of a
//                 turn does not wait for the P V of the one before it.
//   warps 8-11, 12-15  the softmax groups, a thread per query row, each with
//                 its own score buffers and output accumulator (all 512
//                 columns).  A unit of two tiles gives each group a tile and
//                 both use every K/V block; a unit of one tile gives the
//                 groups alternate blocks, which keeps both busy when there
//                 are few query rows.
//   warps 16-19   the epilogue: a unit's O out of tensor memory, joined over
//                 the two groups where they shared its tile, normalised and
//                 stored (or left as a partial), while the softmax groups are
//                 at the next unit.
//
// Softmax in the log2 domain with a lazily moved maximum (O is rescaled in
// tensor memory only when a row's maximum grows by more than 2^8).  P goes to
// P V as an fp16 head and an fp16 remainder, two MMAs over the same V, as in the
// decode and prefill kernels: one rounding to fp16, 2^-11 of a weight, puts
// outputs that average out to nearly nothing up to 7 % off, where the decode
// path keeps 1 %.  Its price, with the remainder's conversions: 64 nodes over
// 32 768 rows 78 us (one rounding 66), 64 trees of 16 nodes 256 (219), sixteen of
// up to 61 185 (138), 256 chains of 5 1 080 (900).  A row's largest P lies
// between 2^7 (P_BIAS) and 2^15, and an fp16 step below the normal range is
// 2^-24: a weight is off by 2^-22 of itself, or by 2^-32 of the largest where
// that is more.  Sums and accumulators are f32.
//
// Rows a node does not attend never reach its output: scores are selected to
// -inf before the maximum, V rows behind the tree are zeroed in shared memory
// (0 x NaN would be NaN), and NaN or infinities in the V rows of the tree are
// zeroed there too and added at the end to the nodes that see them.
//
// Bound by (figures here and below are replays of one call, inputs as L2 holds
// them, unless they say otherwise).  Few query rows: the cache's bytes and, in
// steady use, the 1 kW power cap: 256 chains of 5 nodes, group 4, 4.7 GB, take 995
// us after a pause and 1 150 at the 1.46 GHz of the cap (4.1 TB/s; the decode
// kernel reads the same bytes at 6.8).  An MMA has 128 rows of which these use
// 20, and the remainder doubles P V, so most of what the tensor pipe (active 53 %
// of the time) multiplies, and the cap pays for, is padding.  Two tiles: a turn's
// chain S -> softmax -> P V, 1.2 us per block and pair of tiles at 1.9 GHz.
// Sixteen trees of up to 61 nodes, group 5, 157 us after a pause, 182 at the cap's
// 1.59 GHz: tensor pipe active 50 %, issue slots 43 %, exponentials 36 %, DRAM
// 36 %.  S alone reads 6 KB of operands from shared memory per 32 clocks of
// multiplication (64 cache rows against 128 query rows), 48 clocks at 128 bytes a
// clock, so part of the pipe's time is waiting for operands.  Shared memory
// and tensor memory are full with two groups; a third turn in flight would need
// smaller blocks, fewer operand bytes per turn larger ones.  Built and measured
// before the remainder, and not kept (64 nodes over 32 768 rows, then 66 us):
// scores in registers at once with the weights in buffers of their own 69.5; one
// arrival per warp on the barriers 68.4; a quarter of the exponentials by
// polynomial 66.4; one issuer per group instead of two cost the 256 chains a
// third.
//
// All waits are bounded: the planner gives the CTA up after 2 s without
// progress, records NWD_DEVERR_PIPE_TIMEOUT, and every role lets its copies and
// MMAs land and returns; the tensor memory is freed.
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "nwd_common.h"
#include "ptx.cuh"
#include "tc.cuh"
#include "tree.cuh"

namespace {

using namespace nwd::ptx;
using namespace nwd::tc;
using nwd::TreeSeq;

constexpr uint32_t HD = 128;
constexpr uint32_t BM = 128;            // query rows per tile
constexpr uint32_t BN = 64;             // cache rows per block
constexpr int THREADS = 640;
constexpr int LAUNCH_REGS = 96;         // what __launch_bounds__ gives 640 threads
constexpr uint32_t Q_CHUNK = BM * 128;  // rows x 64 fp16
constexpr uint32_t Q_TILE = 2 * Q_CHUNK;
constexpr uint32_t CHUNK = BN * 128;
constexpr uint32_t TILE = 2 * CHUNK;    // a K or V block: 16 KiB
constexpr uint32_t NQ = 2, NK = 5, NV = 5;  // stages
constexpr uint32_t NP = 4;              // piece descriptors
constexpr uint32_t PIECE_USERS = 19;    // warps that read them: all but the planner
// What a block costs in a unit of one tile, of two (in the same unit of time):
// 64 nodes over 32 768 rows, three tiles, 78.4 us; as 3 to 5 78.3, 3 to 4 81.5.
constexpr uint32_t COST1 = 1, COST2 = 2;
// How many blocks' time a unit's beginning and end take: 64 trees of 16 nodes
// over 512 to 8 192 rows 256 us; with none 263, with twelve 259.
constexpr uint32_t UNIT_BLOCKS = 6;
// Least part of a unit, of a single sequence: more parts are more partials to
// join.  26 nodes over 4 070 rows 19.4 us; with 1 block 20.4, with 8 23.1; 8
// nodes over 3 000 rows 16.7, 16.7 and 18.0.
constexpr uint32_t MIN_BLOCKS = 4;

constexpr uint32_t O_Q = 0;
constexpr uint32_t O_K = O_Q + NQ * Q_TILE;
constexpr uint32_t O_V = O_K + NK * TILE;
constexpr uint32_t O_ML = O_V + NV * TILE;        // [2 groups][128] (m, l)
constexpr uint32_t O_BAR = O_ML + 2 * BM * 8;
constexpr int B_QFULL = 0, B_QEMPTY = B_QFULL + NQ, B_KFULL = B_QEMPTY + NQ,
              B_KEMPTY = B_KFULL + NK, B_VFULL = B_KEMPTY + NK, B_VEMPTY = B_VFULL + NV,
              B_VTMA = B_VEMPTY + NV,
              // by 2 * softmax group + score buffer
    B_SFULL = B_VTMA + NV, B_PFULL = B_SFULL + 4, B_PVDONE = B_PFULL + 4,
              // by softmax group
    B_OEMPTY = B_PVDONE + 4, B_ML = B_OEMPTY + 2, B_DRAIN = B_ML + 2,
              B_PCFULL = B_DRAIN + 1, B_PCEMPTY = B_PCFULL + NP, B_DONE = B_PCEMPTY + NP,
              NBAR = B_DONE + 1;
constexpr uint32_t O_PIECE = (O_BAR + NBAR * 8 + 15) / 16 * 16;  // [NP] Piece
constexpr uint32_t O_VBAD = O_PIECE + NP * 64;    // [NV] u64: tree rows with NaN or inf in V
constexpr uint32_t O_GBAD = O_VBAD + NV * 8;      // [2] u64: the same, gathered per group
constexpr uint32_t O_MISC = O_GBAD + 16;          // tensor memory base, abort flag
constexpr uint32_t O_DONE = O_MISC + 8;           // [2] u32: K blocks issued, pieces finished
constexpr uint32_t SMEM_USED = O_MISC + 16;
// dynamic shared memory starts 1024-byte aligned (there is no static shared
// memory in this kernel); the kernel checks it
constexpr uint32_t SMEM_BYTES = SMEM_USED;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory");

constexpr uint32_t TMEM_COLS = 512;  // 2 groups x 2 score buffers of 64, then O0 O1 of 128
constexpr uint32_t TMEM_O = 256;
constexpr float RESCALE_LOG2 = 8.f;
constexpr float P_BIAS = 7.f;  // P = 2^(s - m + 7) <= 2^15, m within 2^8 of the maximum
constexpr uint32_t IDESC_S = idesc_f16(BM, BN, false);
constexpr uint32_t IDESC_O = idesc_f16(BM, HD, true);

struct TParams {
  const __half* v;
  __half* o;
  const int64_t* row_offset;
  const int32_t* seq_len;
  const int32_t* parents;
  const int32_t* tree_len;
  const int32_t* capacity;  // rows of the sequences' regions, or nullptr
  uint32_t* err;      // the caller's error word, or the workspace's
  uint8_t* ws;
  uint64_t pool_rows;
  uint32_t batch, n_nodes, n_heads, n_kv, group;
  uint32_t tile_nodes, n_tiles, unit_tiles;  // of a sequence with all its nodes
  uint32_t head_ctas;                        // one sequence: CTAs per kv head; 0: a batch
  float scale_log2;
};

// Blocks [blk, blk + nb) of a unit: what the roles do with it.
struct __align__(16) Piece {
  uint32_t row0, ctx, nodes, b;  // the sequence: first pool row, context rows, nodes
  uint32_t blk, nb, hkv, tile0;
  uint32_t tiles;                // 1 or 2; 0: no more pieces
  uint32_t whole;                // the unit is this piece: its outputs are final
  uint32_t x0, n0, q0;           // turns, blocks and Q tiles of this CTA before it
  uint32_t pad[3];
};
static_assert(sizeof(Piece) == 64, "piece");

// ---- workspace: [0, 256) an error word nobody reads (when the caller gives
// none), MergeDesc per CTA, then per CTA two slots (the piece its range begins
// with, the piece it ends with) of unit_tiles tiles: (m, l) [tile][128], then
// O [tile][32 column quads][128 rows][4] f32.
struct MergeDesc {
  uint32_t valid, b, u, first;  // 1 + the sequence's nodes; the unit's pieces are CTAs first .. this one
};
constexpr uint32_t MAX_CTAS = 240;
constexpr size_t WS_DESC = 256;
constexpr size_t WS_ML = WS_DESC + MAX_CTAS * sizeof(MergeDesc);
__host__ __device__ inline size_t ws_o(uint32_t ctas, uint32_t unit_tiles) {
  return WS_ML + (size_t)ctas * 2 * unit_tiles * BM * 8;
}
__host__ __device__ inline size_t ws_total(uint32_t ctas, uint32_t unit_tiles) {
  return ws_o(ctas, unit_tiles) + (size_t)ctas * 2 * unit_tiles * BM * HD * 4;
}
static_assert(WS_ML % 256 == 0, "alignment");

__device__ __forceinline__ TreeSeq load_seq(const TParams& p, uint32_t b, uint32_t* err) {
  return nwd::tree_seq(p.row_offset, p.seq_len, p.tree_len, p.capacity, p.pool_rows, b, p.n_nodes,
                       err);
}
// A unit has at least one block, so that its output rows are written; without
// nodes there is nothing to read.
__device__ __forceinline__ uint32_t seq_blocks(const TreeSeq& s) {
  return s.nodes ? (s.ctx + s.nodes + BN - 1) / BN : 1u;
}
// The tiles that hold a sequence's present nodes (one at least): the others
// are no work but their rows' zeros.
__device__ __forceinline__ uint32_t seq_tiles(const TParams& p, uint32_t nodes) {
  return max(1u, (nodes + p.tile_nodes - 1) / p.tile_nodes);
}
// What a block costs in all units of a kv head with so many tiles.
__device__ __forceinline__ uint32_t head_cost(uint32_t tiles) {
  return tiles / 2 * COST2 + (tiles & 1) * COST1;
}
__device__ __forceinline__ uint64_t warp_sum64(uint32_t v) {
  return ((uint64_t)__reduce_add_sync(0xffffffffu, v >> 16) << 16) +
         __reduce_add_sync(0xffffffffu, v & 0xffffu);
}

// A value that is the same in all lanes of a warp, in a way that the compiler
// sees: it then stays in uniform registers, which the MMA instructions take
// their operands from.
__device__ __forceinline__ uint32_t uniform(uint32_t x) {
  return __reduce_max_sync(0xffffffffu, x);
}
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
  return is != 0;
}

// A unit's kv head, first tile and number of tiles, in a sequence of n_tiles.
struct Unit {
  uint32_t hkv, tile0, tiles;
};
__device__ __forceinline__ Unit unit_of(uint32_t n_tiles, uint32_t u) {
  const uint32_t per_head = (n_tiles + 1) / 2;
  Unit r;
  r.hkv = u / per_head;
  r.tile0 = (u % per_head) * 2;
  r.tiles = min(2u, n_tiles - r.tile0);
  return r;
}

// Position in a ring of N stages.
template <uint32_t N>
struct Ring {
  uint32_t i = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++i == N) {
      i = 0;
      phase ^= 1u;
    }
  }
  __device__ __forceinline__ void add(uint32_t n) {
    i += n;
    phase ^= (i / N) & 1u;
    i %= N;
  }
};

// What every warp of a CTA knows.
struct Ctx {
  uint8_t* smem;
  uint32_t sb, bar;  // shared memory, its barriers
  volatile int32_t* abort_flag;
  uint32_t* err;
  // Waits, the whole warp, until the phase is complete or the CTA gives up:
  // the planner watches over the others' progress (watch), so that the many
  // waits are a few instructions each.
  __device__ __forceinline__ bool wait(int b, uint32_t parity) const {
    while (!__all_sync(0xffffffffu, mbar_try_wait(bar + 8 * b, parity)))
      if (*abort_flag) return false;
    return true;
  }
  __device__ __forceinline__ void arrive(int b) const { mbar_arrive(bar + 8 * b); }
};

// A warp's way through the piece descriptors.
struct PieceIn {
  Ring<NP> r;
  // the next piece; false: there is none (or the CTA is aborting, then !ok)
  __device__ __forceinline__ bool get(const Ctx& c, Piece& d, bool& ok) {
    if (!c.wait(B_PCFULL + (int)r.i, r.phase)) {
      ok = false;
      return false;
    }
    d = reinterpret_cast<const Piece*>(c.smem + O_PIECE)[r.i];
    __syncwarp();
    if ((threadIdx.x & 31) == 0) c.arrive(B_PCEMPTY + (int)r.i);
    r.next();
    return d.tiles != 0;
  }
};

// An issuer's way through the stages of a ring.  Both groups' issuers wait for
// every copy, in order, and release it, the ones that only the other group
// uses too: a parity wait cannot tell a phase from the one two before or after
// it, so nobody may fall, or run, two uses of a stage behind the others.
template <uint32_t N>
struct Walker {
  Ring<N> r;
  uint32_t n = 0;
  __device__ __forceinline__ void next() {
    n++;
    r.next();
  }
  // waits for copy `to`; the ones before it are released as they land
  __device__ __forceinline__ bool reach(const Ctx& c, uint32_t to, int full, int empty) {
    for (;;) {
      if (!c.wait(full + (int)r.i, r.phase)) return false;
      if (n == to) return true;
      if (elect_one()) c.arrive(empty + (int)r.i);
      next();
    }
  }
};

// a / b, by the 32-bit division where both fit it (nearly always), else bit by
// bit: the compiler's 64-bit division is some hundred instructions wherever it
// stands, and this kernel's code has to fit the instruction cache.
__device__ __forceinline__ uint64_t div_small(uint64_t a, uint64_t b) {
  if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
  uint64_t q = 0, r = 0;
#pragma unroll 1
  for (int i = 63; i >= 0; i--) {
    r = r << 1 | ((a >> i) & 1);
    q <<= 1;
    if (r >= b) {
      r -= b;
      q |= 1;
    }
  }
  return q;
}

// The planner's wait: gives the CTA up, with NWD_DEVERR_PIPE_TIMEOUT, after
// WAIT_LIMIT_NS without a K block issued or a piece finished.
__device__ __forceinline__ bool watch(const Ctx& c, int b, uint32_t parity) {
  const volatile uint32_t* done = reinterpret_cast<const uint32_t*>(c.smem + O_DONE);
  uint32_t last = 0;
  uint64_t since = 0;
  while (!__all_sync(0xffffffffu, mbar_try_wait(c.bar + 8 * b, parity))) {
    if (*c.abort_flag) return false;
    const uint32_t now = done[0] + done[1];
    const uint64_t t = globaltimer();
    if (since == 0 || now != last) {
      last = now;
      since = t;
    }
    if (__any_sync(0xffffffffu, t - since > WAIT_LIMIT_NS)) {
      if ((threadIdx.x & 31) == 0) {
        *c.abort_flag = 1;
        atomicOr(c.err, NWD_DEVERR_PIPE_TIMEOUT);
      }
      return false;
    }
  }
  return true;
}

// The planner (one warp): this CTA's range, its join, and its pieces; then the
// zeros of the tiles without present nodes.
//
// One sequence: its units get CTAs in proportion to their costs, each a part of
// one unit's blocks, so that no CTA has two units' beginnings and ends to wait
// for (8 nodes over 3 000 rows 16.7 us, 26 over 4 070 19.4, 64 over 32 768 78.4;
// cut as a batch 17.6, 21.3, 79.0).
//
// A batch: the units make a line, each as long as its blocks' costs and
// UNIT_BLOCKS more for its beginning and end, which is cut into equal ranges.
// A cut inside a block gives the block to the CTA before the cut.
__device__ __forceinline__ void plan(const TParams& p, const Ctx& c) {
  const uint32_t lane = threadIdx.x & 31;
  auto cost_of = [](uint32_t tiles) { return tiles == 2 ? COST2 : COST1; };
  MergeDesc join{0, 0, 0, 0};
  int64_t left = 0;
  uint32_t b = 0, u = 0, blk = 0, nblk = 0, nt = 1;
  TreeSeq s{};
  if (p.head_ctas) {
    s = load_seq(p, 0, p.err);
    nblk = seq_blocks(s);
    nt = seq_tiles(p, s.nodes);
    const uint32_t head = blockIdx.x / p.head_ctas, i = blockIdx.x % p.head_ctas;
    const uint32_t pairs = nt / 2;
    uint32_t singles = nt & 1 ? max(1u, p.head_ctas * COST1 / head_cost(nt)) : 0;
    uint32_t k = pairs ? (p.head_ctas - singles) / pairs : 0;
    singles = p.head_ctas - pairs * k;
    uint32_t unit = pairs ? i / k : 0, at = pairs ? i % k : i;
    if (unit >= pairs) {
      unit = pairs;
      at = i - pairs * k;
      k = singles;
    }
    if (head < p.n_kv && unit < (nt + 1) / 2) {
      k = max(1u, min(k, nblk / MIN_BLOCKS));  // parts of at least MIN_BLOCKS
      u = head * ((nt + 1) / 2) + unit;
      if (at < k) {
        // nblk * at / k, in 32 bits
        const uint32_t each = nblk / k, rest = nblk - each * k;
        blk = each * at + rest * at / k;
        const uint32_t end = each * (at + 1) + rest * (at + 1) / k;
        left = (int64_t)(end - blk) * cost_of(unit < pairs ? 2 : 1);
        if (at > 0 && at + 1 == k) join = MergeDesc{1 + s.nodes, 0, u, blockIdx.x - at};
      }
    }
  } else {
    const uint32_t groups = (p.batch + 31) / 32;
    // a sequence's length on the line, per kv head
    auto length = [&](const TreeSeq& q) {
      return (seq_blocks(q) + UNIT_BLOCKS) * head_cost(seq_tiles(p, q.nodes));
    };
    // of 32 sequences at a time; lane l keeps group l's, s is group `loaded`'s
    uint32_t loaded = 0;
    auto group_length = [&](uint32_t g, uint32_t* err) -> uint64_t {
      const uint32_t i = g * 32 + lane;
      loaded = g;
      if (i < p.batch) s = load_seq(p, i, err);
      return warp_sum64(i < p.batch ? length(s) : 0u);
    };
    uint64_t kept = 0, total = 0;
#pragma unroll 1
    for (uint32_t g = 0; g < groups; g++) {
      const uint64_t sum = group_length(g, p.err);
      if (lane == g) kept = sum;
      total += sum;
    }
    total *= p.n_kv;
    const uint64_t per = max(div_small(total + gridDim.x - 1, gridDim.x), (uint64_t)COST2);
    const uint64_t x0 = min(total, (uint64_t)blockIdx.x * per), x1 = min(total, x0 + per);
    if (x1 > x0) {
      // the sequence that x0 falls into: its group, then its lane
      const uint64_t y = div_small(x0, p.n_kv);  // per kv head
      uint64_t base = 0, upto = kept;
#pragma unroll
      for (int i = 1; i < 32; i <<= 1) {
        const uint64_t v = __shfl_up_sync(0xffffffffu, upto, i);
        if ((int)lane >= i) upto += v;
      }
      uint32_t group;
      const uint32_t hit = __ballot_sync(0xffffffffu, y < upto);
      if (hit) {
        group = (uint32_t)__ffs(hit) - 1;
        base = __shfl_sync(0xffffffffu, upto - kept, (int)group);
      } else {  // past the first 1024 sequences
        base = __shfl_sync(0xffffffffu, upto, 31);
        for (group = 32;; group++) {
          const uint64_t sum = group_length(group, nullptr);
          if (y < base + sum) break;
          base += sum;
        }
      }
      b = group * 32 + lane;
      if (b < p.batch && loaded != group) s = load_seq(p, b, nullptr);
      const uint64_t len = b < p.batch ? length(s) : 0u;
      upto = len;
#pragma unroll
      for (int i = 1; i < 32; i <<= 1) {
        const uint64_t v = __shfl_up_sync(0xffffffffu, upto, i);
        if ((int)lane >= i) upto += v;
      }
      const int at = __ffs(__ballot_sync(0xffffffffu, y < base + upto)) - 1;
      base += __shfl_sync(0xffffffffu, upto - len, at);
      b = group * 32 + (uint32_t)at;
      s.row0 = __shfl_sync(0xffffffffu, s.row0, at);
      s.ctx = __shfl_sync(0xffffffffu, s.ctx, at);
      s.nodes = __shfl_sync(0xffffffffu, s.nodes, at);
      nblk = seq_blocks(s);
      nt = seq_tiles(p, s.nodes);
      // the unit of this sequence that x0 falls into, and where it starts
      const uint64_t of_head = (uint64_t)(nblk + UNIT_BLOCKS) * head_cost(nt);
      const uint64_t of_pair = (uint64_t)(nblk + UNIT_BLOCKS) * COST2;
      uint64_t r = x0 - base * p.n_kv;
      const uint32_t head = (uint32_t)div_small(r, of_head);
      r -= head * of_head;
      const uint32_t k = min((uint32_t)div_small(r, of_pair), (nt + 1) / 2 - 1);
      r -= k * of_pair;
      const uint64_t start = x0 - r;  // of the unit, on the line
      u = head * ((nt + 1) / 2) + k;
      const uint32_t cost = cost_of(unit_of(nt, u).tiles);
      blk = (uint32_t)div_small(r + cost - 1, cost);
      if (blk < nblk) {
        left = (int64_t)(x1 - start) - (int64_t)((uint64_t)blk * cost);
        if (blk > 0 && left > 0 && blk + div_small(left + cost - 1, cost) >= nblk)
          join = MergeDesc{1 + s.nodes, b, u, (uint32_t)div_small(start, per)};
      } else {  // the unit's last block is the CTA's before
        left = (int64_t)(x1 - start) - (int64_t)((uint64_t)(nblk + UNIT_BLOCKS) * cost);
        blk = nblk;
      }
    }
  }
  if (lane == 0) reinterpret_cast<MergeDesc*>(p.ws + WS_DESC)[blockIdx.x] = join;

  Ring<NP> r;
  uint32_t turns = 0, blocks = 0, tiles = 0;
  nwd::TreeRaw ahead{};
  if (left > 0 && b + 1 < p.batch)
    ahead = nwd::tree_raw(p.row_offset, p.seq_len, p.tree_len, p.capacity, b + 1, p.n_nodes);
  for (;;) {
    Piece d{};
    if (left > 0 && blk == nblk) {  // on to the next unit
      blk = 0;
      if (++u == p.n_kv * ((nt + 1) / 2)) {
        u = 0;
        b++;
        s = nwd::tree_seq(ahead, p.pool_rows, p.n_nodes, nullptr);
        nblk = seq_blocks(s);
        nt = seq_tiles(p, s.nodes);
        if (b + 1 < p.batch)
          ahead = nwd::tree_raw(p.row_offset, p.seq_len, p.tree_len, p.capacity, b + 1, p.n_nodes);
      }
    }
    if (left > 0) {
      const Unit un = unit_of(nt, u);
      const uint32_t cost = cost_of(un.tiles);
      const uint64_t most = (uint64_t)(nblk - blk) * cost;
      d.nb = (uint64_t)left >= most ? nblk - blk : ((uint32_t)left + cost - 1) / cost;
      d.row0 = (uint32_t)s.row0;
      d.ctx = s.ctx;
      d.nodes = s.nodes;
      d.b = b;
      d.blk = blk;
      d.hkv = un.hkv;
      d.tile0 = un.tile0;
      d.tiles = un.tiles;
      d.whole = d.nb == nblk;
      d.x0 = turns;
      d.n0 = blocks;
      d.q0 = tiles;
      turns += d.nb * un.tiles;
      blocks += d.nb;
      tiles += un.tiles;
      blk += d.nb;
      left -= (int64_t)(d.nb + (blk == nblk ? UNIT_BLOCKS : 0)) * cost;
    }
    if (!watch(c, B_PCEMPTY + (int)r.i, r.phase ^ 1u)) break;
    if (lane == 0) {
      reinterpret_cast<Piece*>(c.smem + O_PIECE)[r.i] = d;
      c.arrive(B_PCFULL + (int)r.i);
    }
    __syncwarp();
    r.next();
    if (d.tiles == 0) break;
  }
  if (p.n_tiles > 1) {
    // all sequences' rows of zeros, dealt out to the CTAs one after the other
    // (without tree_len those of sequences that leave the pool)
    const uint32_t row_vec = p.n_heads * (HD / 8);
    uint32_t turn = 0;  // the CTA whose row comes next
#pragma unroll 1
    for (uint32_t b0 = 0; b0 < p.batch; b0 += 32) {
      uint32_t first = p.n_nodes;
      if (b0 + lane < p.batch)
        first = min(first, seq_tiles(p, load_seq(p, b0 + lane, nullptr).nodes) * p.tile_nodes);
#pragma unroll 1
      for (uint32_t some = __ballot_sync(0xffffffffu, first < p.n_nodes); some; some &= some - 1) {
        const uint32_t at = (uint32_t)__ffs(some) - 1;
        uint32_t node = __shfl_sync(0xffffffffu, first, at);
        const uint32_t rows = p.n_nodes - node;
        node += blockIdx.x - turn + (blockIdx.x < turn ? gridDim.x : 0);
        for (; node < p.n_nodes; node += gridDim.x) {
          uint4* o = reinterpret_cast<uint4*>(p.o) + ((size_t)(b0 + at) * p.n_nodes + node) * row_vec;
          for (uint32_t k = lane; k < row_vec; k += 32) o[k] = make_uint4(0u, 0u, 0u, 0u);
        }
        turn = (turn + rows) % gridDim.x;
      }
    }
  }
  watch(c, B_DONE, 0);
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mov.b64 z, {%6, %7};\n\tfma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
// The rows of the tree that `node` sees (its ancestors and itself), from the
// parents of its n nodes: lane i has those of nodes i and i + 32.
__device__ uint64_t tree_masks(int2 par, uint32_t n, uint32_t node, uint32_t* err) {
  uint64_t seen[2];
  nwd::tree_closure(par, n, err, seen);
  const uint64_t lo = __shfl_sync(0xffffffffu, seen[0], (int)(node & 31));
  const uint64_t hi = __shfl_sync(0xffffffffu, seen[1], (int)(node & 31));
  return node < 32 ? lo : hi;
}

// 32 bytes, a whole sector, at a 32-byte aligned address.
__device__ __forceinline__ void store32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// Before a CTA that gives up can exit: waits, within the limit, for a phase, and
// for the last of `issued` copies into each stage of a ring.
__device__ __forceinline__ void land_one(const Ctx& c, int b, uint32_t parity) {
  const uint64_t t0 = globaltimer();
  while (!mbar_try_wait(c.bar + 8 * b, parity) && globaltimer() - t0 < WAIT_LIMIT_NS) {
  }
}
template <uint32_t N>
__device__ __forceinline__ void land(const Ctx& c, int full, uint32_t issued) {
#pragma unroll 1
  for (uint32_t i = 0; i < N; i++) {
    const uint32_t uses = (issued + N - 1 - i) / N;
    if (uses) land_one(c, full + (int)i, (uses - 1) & 1);
  }
}

__global__ void __launch_bounds__(THREADS, 1)
    tree_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                const __grid_constant__ CUtensorMap tmv, const __grid_constant__ TParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + O_MISC);
  volatile uint64_t* vbad = reinterpret_cast<uint64_t*>(smem + O_VBAD);
  volatile uint64_t* gbad = reinterpret_cast<uint64_t*>(smem + O_GBAD);
  volatile uint32_t* done = reinterpret_cast<uint32_t*>(smem + O_DONE);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Ctx c{smem, smem_u32(smem), smem_u32(smem) + O_BAR,
              reinterpret_cast<int32_t*>(smem + O_MISC + 4), p.err};

  nwd::pdl_trigger();
  if (warp == 1) {
    if (lane == 0) {
      *c.abort_flag = 0;
      reinterpret_cast<uint2*>(smem + O_DONE)[0] = make_uint2(0u, 0u);
    }
    for (int i = lane; i < NBAR; i += 32) {
      uint32_t count = 1;
      // a stage is released by both groups' issuers
      if ((i >= B_QEMPTY && i < B_KFULL) || (i >= B_KEMPTY && i < B_VFULL) ||
          (i >= B_VEMPTY && i < B_VTMA))
        count = 2;
      if ((i >= B_PFULL && i < B_PVDONE) || (i >= B_OEMPTY && i < B_DRAIN)) count = BM;
      if (i == B_DRAIN) count = 4;
      if (i >= B_PCEMPTY) count = PIECE_USERS;  // and B_DONE: the same warps
      mbar_init(c.bar + 8 * i, count);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 64) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmq)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmk)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmv)) : "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  nwd::pdl_wait();
  if (c.sb & 1023u) {  // the swizzled tiles would not line up: no work
    *c.abort_flag = 1;
    if (tid == 0) atomicOr(p.err, NWD_DEVERR_PIPE_TIMEOUT);
  }
  const uint32_t tmem = *tmem_slot;
  PieceIn in;
  Piece d;
  bool ok = true;

  // Registers per thread: 48 for the first two warpgroups, 152 for the softmax
  // groups, 80 for the epilogue: 128 * (2 * 48 + 2 * 152 + 80) = 61440, the
  // 640 * 96 of the launch.
  if (warp < 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;" ::: "memory");
    // K and V are read once, unless a head's query rows are several units
    const uint64_t policy = p.n_tiles <= 2 ? evict_first_policy() : evict_last_policy();
    if (warp == 0) {
      // ======================= K =======================
      Ring<NK> r;
      uint32_t issued = 0;
      while (ok && in.get(c, d, ok)) {
        int row = (int)(d.row0 + d.blk * BN);
#pragma unroll 1
        for (uint32_t j = 0; j < d.nb; j++, row += BN) {
          ok = c.wait(B_KEMPTY + (int)r.i, r.phase ^ 1u);
          if (!ok) break;
          if (lane == 0) {
            const uint32_t fb = c.bar + 8 * (B_KFULL + r.i), dst = c.sb + O_K + r.i * TILE;
            mbar_arrive_tx(fb, TILE);
            tma_load_4d(dst, &tmk, fb, 0, 0, (int)d.hkv, row, policy);
            tma_load_4d(dst + CHUNK, &tmk, fb, 0, 1, (int)d.hkv, row, policy);
          }
          __syncwarp();
          r.next();
          issued++;
          if (lane == 0) done[0] = issued;
        }
      }
      if (!ok) land<NK>(c, B_KFULL, issued);
    } else if (warp == 1) {
      // ======================= V and Q =======================
      // The next piece's Q goes out as soon as its buffers are free, looked
      // for with every V block; with the piece's last one it is waited for.
      const uint64_t q_policy = evict_first_policy();
      const uint32_t q_bytes = 2 * p.tile_nodes * p.group * 128;
      Ring<NV> r;
      Ring<NQ> rq;
      uint32_t issued = 0, q_issued = 0, tails = 0, q_tile = 0;
      auto load_q = [&](const Piece& e, bool block) -> bool {
        while (q_tile < e.tiles) {
          const int empty = B_QEMPTY + (int)rq.i;
          if (!__all_sync(0xffffffffu, mbar_test_wait(c.bar + 8 * empty, rq.phase ^ 1u))) {
            if (!block) return true;
            if (!c.wait(empty, rq.phase ^ 1u)) return false;
          }
          if (lane == 0) {
            const uint32_t fb = c.bar + 8 * (B_QFULL + rq.i), dst = c.sb + O_Q + rq.i * Q_TILE;
            const int node = (int)(e.b * p.n_nodes + (e.tile0 + q_tile) * p.tile_nodes);
            mbar_arrive_tx(fb, q_bytes);
            tma_load_5d(dst, &tmq, fb, 0, 0, 0, (int)e.hkv, node, q_policy);
            tma_load_5d(dst + Q_CHUNK, &tmq, fb, 0, 1, 0, (int)e.hkv, node, q_policy);
          }
          __syncwarp();
          rq.next();
          q_issued++;
          q_tile++;
        }
        return true;
      };
      Piece e;  // the piece after d
      bool more = in.get(c, e, ok);
      d.nb = 0;
      while (ok) {
        // d's blocks, with e's Q (at first only e's Q)
        int row = (int)(d.row0 + d.blk * BN);
        uint32_t j = 0;
#pragma unroll 1
        do {
          if (j < d.nb) {
            ok = c.wait(B_VEMPTY + (int)r.i, r.phase ^ 1u);
            if (!ok) break;
            // a block with rows of the tree, or behind it, completes on VTMA:
            // warp 2 releases it to its users
            const bool tail = (d.blk + j + 1) * BN > d.ctx;
            if (lane == 0) {
              const uint32_t fb = c.bar + 8 * ((tail ? B_VTMA : B_VFULL) + (int)r.i);
              const uint32_t dst = c.sb + O_V + r.i * TILE;
              mbar_arrive_tx(fb, TILE);
              tma_load_4d(dst, &tmv, fb, 0, 0, (int)d.hkv, row, policy);
              tma_load_4d(dst + CHUNK, &tmv, fb, 0, 1, (int)d.hkv, row, policy);
            }
            __syncwarp();
            if (tail) tails ^= 1u << r.i;
            r.next();
            issued++;
            row += BN;
          }
          j++;
          if (more) ok = load_q(e, j >= d.nb);
        } while (ok && j < d.nb);
        if (!ok || !more) break;
        d = e;
        more = in.get(c, e, ok);
        q_tile = 0;
      }
      if (!ok) {
        // (a block's last completion on VFULL may be warp 2's, of a tail)
        land<NV>(c, B_VFULL, issued);
        land<NQ>(c, B_QFULL, q_issued);
        for (uint32_t i = 0; i < NV; i++) land_one(c, B_VTMA + (int)i, ((tails >> i) & 1u) ^ 1u);
      }
    } else if (warp == 2) {
      // ======================= V blocks with rows of the tree =======================
      // Rows behind the tree become zeros (0 x NaN would be NaN), NaN and
      // infinities in the tree's rows too; which rows had some is noted.
      uint32_t phases = 0;  // of VTMA, bit i: stage i
      Ring<NV> r;
      while (ok && in.get(c, d, ok)) {
        // the blocks before the tree's first row are not this warp's
        const uint32_t from = d.ctx / BN, skip = from > d.blk ? min(from - d.blk, d.nb) : 0;
        r.add(skip);
#pragma unroll 1
        for (uint32_t j = skip; j < d.nb; j++, r.next()) {
          ok = c.wait(B_VTMA + (int)r.i, (phases >> r.i) & 1u);
          if (!ok) break;
          phases ^= 1u << r.i;
          const uint32_t key0 = (d.blk + j) * BN, rows = d.ctx + d.nodes;
          const uint32_t t0 = d.ctx > key0 ? d.ctx - key0 : 0;
          const uint32_t t1 = max(rows > key0 ? min(rows - key0, BN) : 0u, t0);
          // 8 uint4 of a row per chunk (a swizzled row stays within its 128
          // bytes): lane l has those of rows l / 8, l / 8 + 4, ..
          uint4* st = reinterpret_cast<uint4*>(smem + O_V + r.i * TILE) + lane;
          uint64_t bad = 0;
#pragma unroll 1
          for (uint32_t i = t0 / 4; i < BN / 4; i++) {
            const uint32_t row = i * 4 + (uint32_t)lane / 8;
            uint4 x[2] = {st[i * 32], st[CHUNK / 16 + i * 32]};
            if (row < t0) continue;
#pragma unroll
            for (int h = 0; h < 2; h++) {
              uint32_t* w = &x[h].x;
              bool hit = row >= t1;
#pragma unroll
              for (int k = 0; k < 4; k++) {
                const bool lo = (w[k] & 0x7c00u) == 0x7c00u || row >= t1;
                const bool hi = (w[k] & 0x7c000000u) == 0x7c000000u || row >= t1;
                hit |= lo | hi;
                if (lo) w[k] &= 0xffff0000u;
                if (hi) w[k] &= 0x0000ffffu;
              }
              if (hit) {
                st[h * (CHUNK / 16) + i * 32] = x[h];
                if (row < t1) bad |= 1ull << (key0 + row - d.ctx);
              }
            }
          }
          const uint32_t blo = __reduce_or_sync(0xffffffffu, (uint32_t)bad);
          const uint32_t bhi = __reduce_or_sync(0xffffffffu, (uint32_t)(bad >> 32));
          if (lane == 0) vbad[r.i] = (uint64_t)bhi << 32 | blo;
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) c.arrive(B_VFULL + (int)r.i);
        }
      }
    } else if (warp == 3) {
      plan(p, c);
    } else {
      // ======================= MMA issuers =======================
      // The whole warp walks its group's turns x, one lane issues.
      const uint32_t role = uniform((uint32_t)warp - 4);
      const uint32_t g = role & 1;
      const bool leader = elect_one();
      const uint32_t tm = uniform(tmem);
      const uint32_t tmem_s = tm + g * 2 * BN;
      uint32_t buf = 0, phase = 0;  // of the group's score buffers
      if (role < 2) {
        // ---- S(x), once P V(x - 2) has read the P in its buffer
        Walker<NQ> q;
        Walker<NK> k;
        while (ok && in.get(c, d, ok)) {
          const bool two = uniform(d.tiles) == 2;
          const uint32_t mine = uniform((g - d.x0) & 1);  // two tiles: the tile; one: the first block
          const uint32_t step = two ? 1 : 2, nb = uniform(d.nb);
          uint32_t j = two ? 0 : mine;
          if (j >= nb) continue;
          ok = q.reach(c, uniform(d.q0) + (two ? mine : 0), B_QFULL, B_QEMPTY);
          if (!ok) break;
          const uint32_t da = (c.sb + O_Q + q.r.i * Q_TILE) >> 4;
          const uint32_t n0 = uniform(d.n0);
#pragma unroll 1
          for (; j < nb; j += step) {
            ok = k.reach(c, n0 + j, B_KFULL, B_KEMPTY) &&
                 c.wait(B_PVDONE + (int)(2 * g + buf), phase ^ 1u);
            if (!ok) break;
            tc_fence_after();
            const uint32_t db = (c.sb + O_K + k.r.i * TILE) >> 4;
            constexpr uint64_t top = sdesc(0, 16, 1024);
            if (leader) {
#pragma unroll
              for (uint32_t kk = 0; kk < 8; kk++)
                umma(tmem_s + buf * BN, top | (da + (((kk >> 2) * Q_CHUNK + (kk & 3) * 32) >> 4)),
                     top | (db + (((kk >> 2) * CHUNK + (kk & 3) * 32) >> 4)), IDESC_S, kk > 0);
              umma_commit(c.bar + 8 * (B_SFULL + 2 * g + buf));
              umma_commit(c.bar + 8 * (B_KEMPTY + k.r.i));
            }
            __syncwarp();
            k.next();
            phase ^= buf;
            buf ^= 1u;
          }
          if (leader) umma_commit(c.bar + 8 * (B_QEMPTY + q.r.i));
          __syncwarp();
          q.next();
        }
      } else {
        // ---- P V(x)
        const uint32_t tmem_o = tm + TMEM_O + g * HD;
        Walker<NV> v;
        uint32_t o_phase = 1;
        while (ok && in.get(c, d, ok)) {
          const bool two = uniform(d.tiles) == 2;
          const uint32_t mine = uniform((g - d.x0) & 1);
          const uint32_t step = two ? 1 : 2, nb = uniform(d.nb), n0 = uniform(d.n0);
          uint32_t j = two ? 0 : mine;
          if (j >= nb) continue;
          ok = c.wait(B_OEMPTY + (int)g, o_phase);
          o_phase ^= 1u;
          uint32_t add = 0;
#pragma unroll 1
          for (; ok && j < nb; j += step) {
            ok = v.reach(c, n0 + j, B_VFULL, B_VEMPTY) && c.wait(B_PFULL + (int)(2 * g + buf), phase);
            if (!ok) break;
            tc_fence_after();
            // P: key pairs, the heads in the buffer's first 32 columns, the
            // remainders in the other 32; V MN-major (head_dim contiguous),
            // its 64-column chunks 8 KiB apart, 16 keys 2 KiB
            const uint32_t dv = (c.sb + O_V + v.r.i * TILE) >> 4;
            constexpr uint64_t top = sdesc(0, CHUNK, 1024);
            if (leader) {
              umma_ts(tmem_o, tmem_s + buf * BN, top | dv, IDESC_O, add);
#pragma unroll
              for (uint32_t kk = 1; kk < 2 * BN / 16; kk++)
                umma_ts(tmem_o, tmem_s + buf * BN + kk * 8u,
                        top | (dv + ((kk % (BN / 16) * 16 * 128) >> 4)), IDESC_O, 1u);
              umma_commit(c.bar + 8 * (B_PVDONE + 2 * g + buf));
              umma_commit(c.bar + 8 * (B_VEMPTY + v.r.i));
            }
            __syncwarp();
            add = 1;
            v.next();
            phase ^= buf;
            buf ^= 1u;
          }
        }
      }
      // every MMA this warp issued has completed before the tensor memory is
      // released
      if (leader) umma_commit(c.bar + 8 * B_DRAIN);
      __syncwarp();
      land_one(c, B_DRAIN, 0);
    }
  } else if (warp < 16) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 152;" ::: "memory");
    // ======================= softmax groups =======================
    const uint32_t g = (uint32_t)(warp - 8) >> 2;
    const uint32_t quad = (uint32_t)warp & 3u;
    const uint32_t r = quad * 32u + (uint32_t)lane;  // row of the tile = tensor memory lane
    const uint32_t lanes = quad * 32u << 16;
    const uint32_t tmem_o = tmem + TMEM_O + g * HD + lanes;
    const uint32_t q_node = r / p.group;
    uint32_t turn = 0, units = 0;
    while (ok && in.get(c, d, ok)) {
      const bool two = d.tiles == 2;
      const uint32_t mine = (g - d.x0) & 1;  // two tiles: my tile; one: my first block
      const uint32_t tile = d.tile0 + (two ? mine : 0);
      const uint32_t tile_nodes = min(p.tile_nodes, p.n_nodes - tile * p.tile_nodes);
      const uint32_t node = tile * p.tile_nodes + q_node;
      const bool row_used = q_node < tile_nodes;
      const bool warp_used = quad * 32u < tile_nodes * p.group;
      // which rows of the tree this row sees (none if its node is absent):
      // found at the first block that has some, from parents fetched now
      int2 par = make_int2(-1, -1);
      if ((d.blk + d.nb) * BN > d.ctx) {
        const int32_t* src = p.parents + (size_t)d.b * p.n_nodes;
        if ((uint32_t)lane < p.n_nodes) par.x = src[lane];
        if ((uint32_t)lane + 32 < p.n_nodes) par.y = src[lane + 32];
      }
      bool have_mask = false;
      uint64_t sees = 0;
      float m = -INFINITY, l = 0.f;
      uint64_t bad = 0;
      const uint32_t step = two ? 1 : 2;
      const uint32_t first_turn = turn;
#pragma unroll 1
      for (uint32_t j = two ? 0 : mine; j < d.nb; j += step, turn++) {
        const uint32_t buf = turn & 1;
        const uint32_t tmem_s = tmem + (2 * g + buf) * BN + lanes;
        const uint32_t key0 = (d.blk + j) * BN;
        const bool tail = key0 + BN > d.ctx;
        ok = c.wait(B_SFULL + (int)(2 * g + buf), (turn >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        if (warp_used) {
          if (tail && !have_mask) {
            have_mask = true;
            const uint64_t all = tree_masks(par, d.nodes, node, c.err);
            sees = row_used && node < d.nodes ? all : 0;
          }
          // The exponentials are taken against the maximum so far, beside the
          // search for this block's: only where that lies 2^8 above it is O
          // rescaled and are they taken again, from the scores, which are
          // still in the buffer.
          float s[BN];
          float2 sum, sum1;
          bool again;
          do {
            tmem_ld32(tmem_s, s);
            tmem_ld32(tmem_s + 32, s + 32);
            tmem_ld_wait();
            if (tail) {
              // bit k of word i: this row attends cache row key0 + 32 i + k
#pragma unroll
              for (int i = 0; i < 2; i++) {
                const int64_t at = (int64_t)key0 + 32 * i - (int64_t)d.ctx;  // in the tree
                uint32_t ok32;
                if (at <= -32) ok32 = 0xffffffffu;
                else if (at < 0) ok32 = (uint32_t)(sees << -at) | ((1u << -at) - 1u);
                else ok32 = at < 64 ? (uint32_t)(sees >> at) : 0u;
#pragma unroll
                for (int k = 0; k < 32; k++)
                  if (!((ok32 >> k) & 1u)) s[32 * i + k] = -INFINITY;
              }
            }
            if (turn == first_turn) {
              float mv[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
              for (int k = 4; k < (int)BN; k++) mv[k & 3] = fmaxf(mv[k & 3], s[k]);
              m = fmaxf(fmaxf(mv[0], mv[1]), fmaxf(mv[2], mv[3])) * p.scale_log2;
            }
            const float nb = m == -INFINITY ? 0.f : P_BIAS - m;
            const float2 sc = make_float2(p.scale_log2, p.scale_log2), nb2 = make_float2(nb, nb);
            sum = sum1 = make_float2(0.f, 0.f);
            float mv[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int k = 0; k < 32; k++) {
              const float2 x = fma2(make_float2(s[2 * k], s[2 * k + 1]), sc, nb2);
              const float2 e = make_float2(ex2f(x.x), ex2f(x.y));
              mv[k & 3] = fmaxf(mv[k & 3], fmaxf(s[2 * k], s[2 * k + 1]));
              if (k & 1) sum1 = add2(sum1, e);
              else sum = add2(sum, e);
              s[2 * k] = e.x;
              s[2 * k + 1] = e.y;
            }
            const float mx = fmaxf(fmaxf(mv[0], mv[1]), fmaxf(mv[2], mv[3])) * p.scale_log2;
            const bool up = mx > m + RESCALE_LOG2;
            again = __any_sync(0xffffffffu, up);
            if (again) {
              const float alpha = up ? ex2f(m - mx) : 1.f;  // 0 while m is -inf
              if (turn != first_turn) {
                // O is rescaled once the P V of the group's last turn is in it
                const uint32_t last = turn - 1;
                if (!c.wait(B_PVDONE + (int)(2 * g + (last & 1)), (last >> 1) & 1)) {
                  ok = false;
                  break;
                }
                tc_fence_after();
#pragma unroll 1
                for (int k = 0; k < 8; k++) {
                  float ov[16];
                  tmem_ld16(tmem_o + k * 16, ov);
                  tmem_ld_wait();
#pragma unroll
                  for (int i = 0; i < 16; i++) ov[i] *= alpha;
                  tmem_st16(tmem_o + k * 16, ov);
                }
              }
              l *= alpha;
              if (up) m = mx;
            }
          } while (again);
          if (!ok) break;
#pragma unroll
          for (int h = 0; h < 2; h++) {
            float head[16], rem[16];
#pragma unroll
            for (int k = 0; k < 16; k++) {
              const float e0 = s[32 * h + 2 * k], e1 = s[32 * h + 2 * k + 1];
              const __half2 hh = __floats2half2_rn(e0, e1);
              const float2 taken = __half22float2(hh);
              const __half2 rr = __floats2half2_rn(e0 - taken.x, e1 - taken.y);
              head[k] = __uint_as_float(*reinterpret_cast<const uint32_t*>(&hh));
              rem[k] = __uint_as_float(*reinterpret_cast<const uint32_t*>(&rr));
            }
            tmem_st16(tmem_s + 16 * h, head);
            tmem_st16(tmem_s + 32 + 16 * h, rem);
          }
          l += (sum.x + sum.y) + (sum1.x + sum1.y);
          tmem_st_wait();
        }
        if (tail && quad == 0) {  // V rows with NaN or infinities, noted by warp 2
          const uint32_t n = d.n0 + j;
          ok = c.wait(B_VFULL + (int)(n % NV), (n / NV) & 1);
          if (!ok) break;
          bad |= vbad[n % NV];
        }
        tc_fence_before();
        c.arrive(B_PFULL + (int)(2 * g + buf));
      }
      if (!ok) break;
      if (turn != first_turn) {
        // (m, l) to the epilogue, once it has read the last ones
        ok = c.wait(B_OEMPTY + (int)g, (units & 1) ^ 1);
        if (!ok) break;
        units++;
        reinterpret_cast<float2*>(smem + O_ML)[g * BM + r] = make_float2(m, l);
        if (r == 0) gbad[g] = bad;
        c.arrive(B_ML + (int)g);
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;" ::: "memory");
    // ======================= epilogue =======================
    const uint32_t quad = (uint32_t)warp & 3u;
    const uint32_t r = quad * 32u + (uint32_t)lane;
    const uint32_t tmem_o = tmem + TMEM_O + (quad * 32u << 16);
    const float2* ml = reinterpret_cast<const float2*>(smem + O_ML);
    const uint32_t q_node = r / p.group, q_head = r % p.group;
    const bool wide = (reinterpret_cast<uintptr_t>(p.o) & 31u) == 0;  // whole sectors per store
    uint32_t turns = 0, turns1 = 0, units = 0, units1 = 0;  // of group 0, of group 1
    // group i's part of the piece is complete: its (m, l), and its last P V
    auto complete = [&](uint32_t i) -> bool {
      const uint32_t last = (i ? turns1 : turns) - 1;
      return c.wait(B_ML + (int)i, (i ? units1 : units) & 1) &&
             c.wait(B_PVDONE + (int)(2 * i + (last & 1)), (last >> 1) & 1);
    };
    while (ok && in.get(c, d, ok)) {
      const bool two = d.tiles == 2;
      const uint32_t lead = d.x0 & 1;  // one tile: the group of the first block
      const uint32_t of_lead = two ? d.nb : (d.nb + 1) / 2, of_other = two ? d.nb : d.nb / 2;
      turns += lead ? of_other : of_lead;
      turns1 += lead ? of_lead : of_other;
      // two tiles: group 0's, then group 1's; one: both groups' halves of it
#pragma unroll 1
      for (uint32_t part = 0; part < d.tiles; part++) {
        const uint32_t g0 = two ? part : lead;
        const bool both = !two && d.nb > 1;
        ok = complete(g0) && (!both || complete(g0 ^ 1));
        if (!ok) break;
        tc_fence_after();
        const float2 a = ml[g0 * BM + r];
        const float2 b = both ? ml[(g0 ^ 1) * BM + r] : make_float2(-INFINITY, 0.f);
        // a group without weights counts for nothing (l may be NaN)
        const float M = fmaxf(a.x, b.x);
        const float wa = a.y != 0.f ? ex2f(a.x - M) : 0.f, wb = b.y != 0.f ? ex2f(b.x - M) : 0.f;
        const float L = (a.y != 0.f ? a.y * wa : 0.f) + (b.y != 0.f ? b.y * wb : 0.f);
        const uint32_t t = two ? (g0 - d.x0) & 1 : 0;
        const uint32_t tile = d.tile0 + t, node = tile * p.tile_nodes + q_node;
        const bool row_used = q_node < min(p.tile_nodes, p.n_nodes - tile * p.tile_nodes);
        const bool absent = node >= d.nodes;
        const float inv = L != 0.f && !absent ? 1.f / L : 0.f;
        // what was taken out of the V rows that this row sees
        uint64_t lost = gbad[g0] | (both ? gbad[g0 ^ 1] : 0);
        if (lost)
          lost &= absent || !row_used ? 0
                                      : nwd::tree_mask(p.parents + (size_t)d.b * p.n_nodes,
                                                       (int)node, nullptr);
        const size_t slot = (size_t)((blockIdx.x * 2 + (d.blk > 0 ? 0 : 1)) * p.unit_tiles + t) * BM;
        __half* dst = p.o + (((size_t)d.b * p.n_nodes + node) * p.n_heads + d.hkv * p.group +
                             q_head) * HD;
        float* part_o =
            reinterpret_cast<float*>(p.ws + ws_o(gridDim.x, p.unit_tiles)) + slot * HD + r * 4;
#pragma unroll 1
        for (uint32_t col = 0; col < HD; col += 32) {
          float ov[32];
          tmem_ld32(tmem_o + g0 * HD + col, ov);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; i++) ov[i] = a.y != 0.f ? ov[i] * wa : 0.f;
          if (both) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
              float o1[16];
              tmem_ld16(tmem_o + (g0 ^ 1) * HD + col + 16 * h, o1);
              tmem_ld_wait();
              if (b.y != 0.f) {
#pragma unroll
                for (int i = 0; i < 16; i++) ov[16 * h + i] += o1[i] * wb;
              }
            }
          }
          if (row_used && (d.whole || !absent)) {  // (absent nodes have no partials)
            for (uint64_t x = lost; x; x &= x - 1) {
              const size_t row = (size_t)d.row0 + d.ctx + (uint32_t)__ffsll((long long)x) - 1;
              const __half* src = p.v + (row * p.n_kv + d.hkv) * HD + col;
#pragma unroll
              for (int i = 0; i < 32; i++) {
                const float e = __half2float(src[i]);
                if (!isfinite(e)) ov[i] += e;
              }
            }
            if (d.whole) {
              uint32_t h[16];
#pragma unroll
              for (int k = 0; k < 16; k++) {
                const __half2 x = __floats2half2_rn(ov[2 * k] * inv, ov[2 * k + 1] * inv);
                h[k] = absent ? 0u : *reinterpret_cast<const uint32_t*>(&x);
              }
              if (wide) {
                store32(dst + col, h);
                store32(dst + col + 16, h + 8);
              } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                  reinterpret_cast<uint4*>(dst + col)[i] =
                      make_uint4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                *reinterpret_cast<float4*>(part_o + (size_t)(col + i) * BM) =
                    make_float4(ov[i], ov[i + 1], ov[i + 2], ov[i + 3]);
            }
          }
        }
        if (!d.whole && row_used && !absent)
          reinterpret_cast<float2*>(p.ws + WS_ML)[slot + r] = make_float2(M, L);
        tc_fence_before();
        // the groups' accumulators, and their (m, l), have been read
        c.arrive(B_OEMPTY + (int)g0);
        if (both) c.arrive(B_OEMPTY + (int)(g0 ^ 1));
        units += both || g0 == 0;
        units1 += both || g0 == 1;
        if (tid == 512) done[1] = units + units1;
      }
    }
  }
  if (warp != 3 && lane == 0) c.arrive(B_DONE);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(TMEM_COLS)
                 : "memory");
}

// Joins the partials of the units that cuts divided, each unit's in CTA order
// (deterministic): M = max m, O = sum O_c 2^(m_c - M) / sum l_c 2^(m_c - M).
//
// A work item is 8 rows of a tile of such a unit.  Every block finds the units
// (all CTAs' descriptors in one round of loads), works out where each one's rows
// are, once, and takes its share of the items; a thread has one row's column
// quad, and fetches 8 pieces' (m, l) and O terms at a time, all in flight
// together, with no word to the other threads.  26 nodes over 4 070 rows, 8.5 MB
// of partials: 3 us after its launch; sixteen trees of up to 61 nodes, some 22
// MB: 9 to 17 us.  (Divisions for every item cost the first 1 us; a form with a
// block per item and piece, the weights in shared memory, took 5 and 24.)
constexpr uint32_t MERGE_ROWS = 8;
constexpr uint32_t MERGE_THREADS = 256;
constexpr uint32_t MERGE_AHEAD = 8;
constexpr uint32_t MERGE_PER_SM = 2;  // resident blocks (98 registers): one wave
struct Join {
  uint32_t first, n;    // its pieces: CTAs first .. first + n - 1
  uint32_t rows[2];     // per tile: query rows
  uint32_t present[2];  // ... of present nodes
  size_t out;           // its first row in o
};
__global__ void __launch_bounds__(MERGE_THREADS)
    tree_merge_kernel(const __grid_constant__ TParams p, uint32_t ctas) {
  __shared__ Join joins[MAX_CTAS];
  __shared__ uint32_t counts[MERGE_THREADS / 32];
  static_assert(MAX_CTAS <= MERGE_THREADS, "one descriptor per thread");
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  nwd::pdl_trigger();
  nwd::pdl_wait();
  MergeDesc d{0, 0, 0, 0};
  if (tid < ctas) d = reinterpret_cast<const MergeDesc*>(p.ws + WS_DESC)[tid];
  const uint32_t some = __ballot_sync(0xffffffffu, d.valid != 0);
  if (lane == 0) counts[warp] = (uint32_t)__popc(some);
  __syncthreads();
  uint32_t n_joins = 0, before = 0;
#pragma unroll
  for (uint32_t i = 0; i < MERGE_THREADS / 32; i++) {
    if (i < warp) before += counts[i];
    n_joins += counts[i];
  }
  if (d.valid) {  // what the items need of it, found once
    const uint32_t nodes = d.valid - 1;
    const Unit un = unit_of(seq_tiles(p, nodes), d.u);
    Join j;
    j.first = d.first;
    j.n = tid - d.first + 1;
#pragma unroll
    for (uint32_t t = 0; t < 2; t++) {
      const uint32_t node0 = (un.tile0 + t) * p.tile_nodes;
      j.rows[t] = t < un.tiles ? min(p.tile_nodes, p.n_nodes - node0) * p.group : 0;
      j.present[t] = nodes > node0 ? min((nodes - node0) * p.group, j.rows[t]) : 0;
    }
    j.out = (((size_t)d.b * p.n_nodes + un.tile0 * p.tile_nodes) * p.n_heads + un.hkv * p.group) * HD;
    joins[before + (uint32_t)__popc(some & ((1u << lane) - 1u))] = j;
  }
  __syncthreads();
  const float2* ml = reinterpret_cast<const float2*>(p.ws + WS_ML);
  const float4* po = reinterpret_cast<const float4*>(p.ws + ws_o(ctas, p.unit_tiles));
  const uint32_t r = tid & 7, quad = tid >> 3;
  const uint32_t per_group = (65536u + p.group - 1) / p.group;  // row / group, as a product
  constexpr uint32_t CHUNKS = BM / MERGE_ROWS;
#pragma unroll 1
  for (uint32_t item = blockIdx.x; item < n_joins * p.unit_tiles * CHUNKS; item += gridDim.x) {
    const uint32_t row = item % CHUNKS * MERGE_ROWS + r;
    const uint32_t t = p.unit_tiles == 2 ? item / CHUNKS & 1 : 0;
    const Join& join = joins[p.unit_tiles == 2 ? item / (2 * CHUNKS) : item / CHUNKS];
    if (row >= join.rows[t]) continue;
    const uint32_t first = join.first, n = row < join.present[t] ? join.n : 0;  // none: zeros
    float M = -INFINITY, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (uint32_t i0 = 0; i0 < n; i0 += MERGE_AHEAD) {
      float4 x[MERGE_AHEAD];
      float2 a[MERGE_AHEAD];
#pragma unroll
      for (uint32_t k = 0; k < MERGE_AHEAD; k++) {
        // the unit's first piece is the one its CTA ended with, the others begin theirs
        const uint32_t i = i0 + k;
        const uint32_t slot = (((first + i) * 2 + (i == 0 ? 1 : 0)) * p.unit_tiles + t) * BM;
        a[k] = make_float2(-INFINITY, 0.f);
        if (i < n) {
          a[k] = __ldcg(ml + slot + row);
          x[k] = __ldcg(po + (size_t)slot * (HD / 4) + quad * BM + row);
        }
      }
      float top = M;
#pragma unroll
      for (uint32_t k = 0; k < MERGE_AHEAD; k++) top = fmaxf(top, a[k].x);
      const float alpha = L != 0.f ? ex2f(M - top) : 0.f;
      L = L != 0.f ? L * alpha : 0.f;
      o.x *= alpha;
      o.y *= alpha;
      o.z *= alpha;
      o.w *= alpha;
      M = top;
#pragma unroll
      for (uint32_t k = 0; k < MERGE_AHEAD; k++) {
        if (a[k].y != 0.f) {  // a piece without weights counts for nothing (l may be NaN)
          const float e = ex2f(a[k].x - top);
          L += a[k].y * e;
          o.x += x[k].x * e;
          o.y += x[k].y * e;
          o.z += x[k].z * e;
          o.w += x[k].w * e;
        }
      }
    }
    const float inv = L != 0.f ? 1.f / L : 0.f;
    const __half2 h[2] = {__floats2half2_rn(o.x * inv, o.y * inv),
                          __floats2half2_rn(o.z * inv, o.w * inv)};
    const uint32_t node = row * per_group >> 16;  // within the tile
    *reinterpret_cast<uint2*>(p.o + join.out +
                              ((size_t)(t * p.tile_nodes + node) * p.n_heads + row - node * p.group) * HD +
                              quad * 4) = *reinterpret_cast<const uint2*>(h);
  }
}

// The nodes' K / V rows [batch, n_nodes, n_kv, hd] into pool rows
// row_offset[b] + pos[b] + i, 16 bytes per thread (kv_append for a tree).  A
// launch of its own, because any CTA of the attention may meet any tree's rows;
// its time (2 to 3 us) lies mostly under the attention kernel's own start.
__global__ void tree_append_kernel(const uint4* __restrict__ k_new, const uint4* __restrict__ v_new,
                                   uint4* __restrict__ k_pool, uint4* __restrict__ v_pool,
                                   const int64_t* row_offset, const int32_t* pos,
                                   const int32_t* tree_len, const int32_t* capacity,
                                   uint64_t pool_rows, uint32_t n_nodes, uint32_t row_vec,
                                   uint32_t* err) {
  nwd::pdl_trigger();
  nwd::pdl_wait();
  const uint32_t b = blockIdx.y;
  const TreeSeq s = nwd::tree_seq(row_offset, pos, tree_len, capacity, pool_rows, b, n_nodes, err);
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
  if (n_heads > 16384) return fail(NWD_ERR_UNSUPPORTED, "%s: %u heads (at most 16384)", who, n_heads);
  if (batch > 4096) return fail(NWD_ERR_UNSUPPORTED, "%s: batch %u (at most 4096)", who, batch);
  if (!aligned16(q) || !aligned16(k_pool) || !aligned16(v_pool) || !aligned16(o))
    return fail(NWD_ERR_INVALID, "%s: tensors must be 16-byte aligned", who);
  if (!(scale >= 0.f) || std::isinf(scale))
    return fail(NWD_ERR_INVALID, "%s: scale must be finite and >= 0", who);
  if (batch && n_nodes && q == o) return fail(NWD_ERR_INVALID, "%s: q and o must not overlap", who);
  if (pool_rows == 0 || pool_rows > (1ull << 31))
    return fail(NWD_ERR_INVALID, "%s: pool rows %llu outside [1, 2^31]", who,
                (unsigned long long)pool_rows);
  return NWD_OK;
}

// How a shape's query rows are tiled: as many whole nodes per tile as fit, so that
// the tiles are few and short trees, where lengths differ, need few of them.
// Group 5, shared out evenly instead: 16 trees of up to 61 nodes 156 us (160), of
// up to 26 86 (105), of 26 each 138 (152); 64 nodes over 32 768 rows 82 (86).
struct Tiling {
  uint32_t tile_nodes, n_tiles, unit_tiles;
};
Tiling tiling(uint32_t n_nodes, uint32_t group) {
  Tiling t;
  t.tile_nodes = std::min(n_nodes, BM / group);
  t.n_tiles = (n_nodes + t.tile_nodes - 1) / t.tile_nodes;
  t.unit_tiles = t.n_tiles > 1 ? 2 : 1;
  return t;
}

// What a call reads and writes, as it may not overlap: o, and the workspace, with
// nothing else.  The planners read lengths and offsets while other CTAs write o
// and partials; a length that changed under them could leave a search for a
// sequence without an end, a join descriptor that did would send its rows
// anywhere.
struct Spans {
  enum { O, V_POOL, K_POOL, COUNT = 11 };
  nwd::Span at[COUNT];
};
int refuse_overlap(const char* who, const nwd::Span& a, const nwd::Span& b) {
  if (!nwd::overlap(a, b)) return NWD_OK;
  return nwd::fail(NWD_ERR_INVALID, "%s: %s and %s must not overlap", who, a.name, b.name);
}

// Checks the workspace, then launches the append (when there are new rows),
// the attention and the join of its partials.
int run_tree(const char* who, const uint16_t* q, const uint16_t* k_pool, const uint16_t* v_pool,
             uint64_t pool_rows, const int64_t* row_offset, const int32_t* seq_len,
             const int32_t* parents, const int32_t* tree_len, uint16_t* o, uint32_t batch,
             uint32_t n_nodes, uint32_t n_heads, uint32_t n_kv, uint32_t head_dim, float scale,
             void* workspace, size_t ws_bytes, uint32_t* err, void* stream,
             const uint16_t* k_new = nullptr, const uint16_t* v_new = nullptr,
             const int32_t* capacity = nullptr) {
  using namespace nwd;
  const uint32_t group = n_heads / n_kv;
  const Tiling t = tiling(n_nodes, group);
  if (!workspace || ((uintptr_t)workspace & 255u))
    return fail(NWD_ERR_WORKSPACE, "%s: the workspace is NULL or not 256-byte aligned", who);
  if (ws_bytes < ws_total(1, t.unit_tiles))
    return fail(NWD_ERR_WORKSPACE, "%s: a workspace of %zu bytes is too small", who, ws_bytes);
  const uint64_t nodes = (uint64_t)batch * n_nodes, row = (uint64_t)n_kv * head_dim * 2;
  const Spans spans = {{{"o", o, nodes * n_heads * head_dim * 2},
                        {"v_pool", v_pool, pool_rows * row},
                        {"k_pool", k_pool, pool_rows * row},
                        {"q", q, nodes * n_heads * head_dim * 2},
                        {"k_new", k_new, nodes * row},
                        {"v_new", v_new, nodes * row},
                        {"row_offset", row_offset, (uint64_t)batch * 8},
                        {"lengths", seq_len, (uint64_t)batch * 4},
                        {"parents", parents, nodes * 4},
                        {"tree_len", tree_len, (uint64_t)batch * 4},
                        {"capacity", capacity, (uint64_t)batch * 4}}};
  int st = NWD_OK;
  for (uint32_t i = 1; i < Spans::COUNT && !st; i++)
    st = refuse_overlap(who, spans.at[Spans::O], spans.at[i]);
  if (!st) st = refuse_overlap(who, spans.at[Spans::O], {"err", err, 4});
  if (!st && k_new) st = refuse_overlap(who, spans.at[Spans::K_POOL], spans.at[Spans::V_POOL]);
  if (st) return st;
  DeviceInfo di;
  st = current_device_info(&di);
  if (st) return st;
  if (di.sm_count > (int)MAX_CTAS)
    return fail(NWD_ERR_UNSUPPORTED, "%s: %d SMs (at most %u)", who, di.sm_count, MAX_CTAS);
  const size_t need = ws_total((uint32_t)di.sm_count, t.unit_tiles);
  if (ws_bytes < need)
    return fail(NWD_ERR_WORKSPACE, "%s: needs a workspace of >= %zu bytes, got %zu", who, need,
                ws_bytes);
  for (uint32_t i = 0; i < Spans::COUNT && !st; i++)
    st = refuse_overlap(who, {"the workspace", workspace, need}, spans.at[i]);
  if (st) return st;
  const float scale_log2 =
      (scale != 0.f ? scale : 1.0f / sqrtf((float)head_dim)) * 1.4426950408889634f;
  if (tree_short_fits(pool_rows, batch, n_nodes * group))  // one launch, no partials
    return launch_tree_short({q, k_new, v_new, const_cast<uint16_t*>(k_pool),
                              const_cast<uint16_t*>(v_pool), o, pool_rows, row_offset, seq_len,
                              parents, tree_len, capacity, n_nodes, n_heads, n_kv, scale_log2,
                              err ? err : reinterpret_cast<uint32_t*>(workspace), stream},
                             who);
  static bool smem_set[64] = {};
  if (!smem_set[di.device]) {
    cudaError_t e = cudaFuncSetAttribute(tree_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)SMEM_BYTES);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(tree_kernel)");
    // setmaxnreg's shares add up to the registers of the launch: fewer would
    // leave the softmax groups waiting for theirs
    cudaFuncAttributes at;
    e = cudaFuncGetAttributes(&at, tree_kernel);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncGetAttributes(tree_kernel)");
    if (at.numRegs < LAUNCH_REGS)
      return fail(NWD_ERR_UNSUPPORTED, "%s: built with %d registers per thread, not %d", who,
                  at.numRegs, LAUNCH_REGS);
    smem_set[di.device] = true;
  }
  CUtensorMap tq, tk, tv;
  if ((st = tree_q_tensor_map(&tq, q, (uint64_t)batch * n_nodes, n_kv, group, t.tile_nodes)) ||
      (st = kv_tensor_map(&tk, k_pool, pool_rows, n_kv, head_dim, BN, 1)) ||
      (st = kv_tensor_map(&tv, v_pool, pool_rows, n_kv, head_dim, BN, 1)))
    return st;
  TParams p{};
  p.v = reinterpret_cast<const __half*>(v_pool);
  p.o = reinterpret_cast<__half*>(o);
  p.row_offset = row_offset;
  p.seq_len = seq_len;
  p.parents = parents;
  p.tree_len = tree_len;
  p.capacity = capacity;
  p.ws = reinterpret_cast<uint8_t*>(workspace);
  p.err = err ? err : reinterpret_cast<uint32_t*>(workspace);
  p.pool_rows = pool_rows;
  p.batch = batch;
  p.n_nodes = n_nodes;
  p.n_heads = n_heads;
  p.n_kv = n_kv;
  p.group = group;
  p.tile_nodes = t.tile_nodes;
  p.n_tiles = t.n_tiles;
  p.unit_tiles = t.unit_tiles;
  const uint32_t of_head = (uint32_t)di.sm_count / n_kv;
  p.head_ctas = batch == 1 && of_head >= (t.n_tiles + 1) / 2 ? of_head : 0;
  p.scale_log2 = scale_log2;
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e = cudaSuccess;
  if (k_new) {
    const uint32_t row_vec = n_kv * head_dim / 8;
    e = launch_pdl(tree_append_kernel, dim3((n_nodes * row_vec + 255) / 256, batch), dim3(256), 0, s,
                   reinterpret_cast<const uint4*>(k_new), reinterpret_cast<const uint4*>(v_new),
                   reinterpret_cast<uint4*>(const_cast<uint16_t*>(k_pool)),
                   reinterpret_cast<uint4*>(const_cast<uint16_t*>(v_pool)), row_offset, seq_len,
                   tree_len, capacity, pool_rows, n_nodes, row_vec, p.err);
    if (e != cudaSuccess) return cuda_fail(e, who);
  }
  const uint32_t ctas = (uint32_t)di.sm_count;
  e = launch_pdl(tree_kernel, dim3(ctas), dim3(THREADS), SMEM_BYTES, s, tq, tk, tv, p);
  if (e == cudaSuccess)
    e = launch_pdl(tree_merge_kernel, dim3(ctas * MERGE_PER_SM), dim3(MERGE_THREADS), 0, s, p, ctas);
  if (e != cudaSuccess) return cuda_fail(e, who);
  return ok();
}

}  // namespace

using namespace nwd;

extern "C" {

int nwd_attn_tree_workspace_size(uint32_t batch, uint32_t n_nodes, uint32_t n_heads,
                                 uint32_t n_kv_heads, uint32_t head_dim, size_t* bytes) {
  const char* who = "nwd_attn_tree_workspace_size";
  if (!bytes) return fail(NWD_ERR_INVALID, "%s: bytes is NULL", who);
  const void *p = reinterpret_cast<const void*>(16), *o = reinterpret_cast<const void*>(32);
  int st = check_tree(who, p, p, p, p, p, p, o, 1, batch, n_nodes, n_heads, n_kv_heads, head_dim,
                      0.f);
  if (st) return st;
  DeviceInfo di;
  st = current_device_info(&di);
  if (st) return st;
  const Tiling t = tiling(n_nodes ? n_nodes : 1, n_heads / n_kv_heads);
  *bytes = ws_total((uint32_t)di.sm_count, t.unit_tiles);
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
  if (batch == 0 || n_nodes == 0) return ok();
  return run_tree(who, q, k_pool, v_pool, pool_rows, row_offset, seq_len, parents, tree_len, o,
                  batch, n_nodes, n_heads, n_kv_heads, head_dim, scale, workspace, ws_bytes, err,
                  stream);
}

int nwd_kv_append_attn_tree(const uint16_t* q, const uint16_t* k_new, const uint16_t* v_new,
                            uint16_t* k_pool, uint16_t* v_pool, uint64_t pool_rows,
                            const int64_t* row_offset, const int32_t* pos, const int32_t* parents,
                            const int32_t* tree_len, uint16_t* o, uint32_t batch, uint32_t n_nodes,
                            uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, float scale,
                            void* workspace, size_t ws_bytes, uint32_t* err, void* stream) {
  return nwd_kv_append_attn_tree_bounded(q, k_new, v_new, k_pool, v_pool, pool_rows, row_offset,
                                         pos, nullptr, parents, tree_len, o, batch, n_nodes,
                                         n_heads, n_kv_heads, head_dim, scale, workspace, ws_bytes,
                                         err, stream);
}

int nwd_kv_append_attn_tree_bounded(const uint16_t* q, const uint16_t* k_new, const uint16_t* v_new,
                                    uint16_t* k_pool, uint16_t* v_pool, uint64_t pool_rows,
                                    const int64_t* row_offset, const int32_t* pos,
                                    const int32_t* capacity, const int32_t* parents,
                                    const int32_t* tree_len, uint16_t* o, uint32_t batch,
                                    uint32_t n_nodes, uint32_t n_heads, uint32_t n_kv_heads,
                                    uint32_t head_dim, float scale, void* workspace,
                                    size_t ws_bytes, uint32_t* err, void* stream) {
  const char* who = "nwd_kv_append_attn_tree";
  int st = check_tree(who, q, k_pool, v_pool, row_offset, pos, parents, o, pool_rows, batch,
                      n_nodes, n_heads, n_kv_heads, head_dim, scale);
  if (st) return st;
  if (!k_new || !v_new) return fail(NWD_ERR_INVALID, "%s: null pointer", who);
  if (!aligned16(k_new) || !aligned16(v_new))
    return fail(NWD_ERR_INVALID, "%s: tensors must be 16-byte aligned", who);
  if (batch == 0 || n_nodes == 0) return ok();
  if (k_pool == v_pool)
    return fail(NWD_ERR_INVALID, "%s: k_pool and v_pool must not overlap", who);
  return run_tree(who, q, k_pool, v_pool, pool_rows, row_offset, pos, parents, tree_len, o, batch,
                  n_nodes, n_heads, n_kv_heads, head_dim, scale, workspace, ws_bytes, err, stream,
                  k_new, v_new, capacity);
}

}  // extern "C"
