// Flash-attention forward kernel for sm_100a: dense batches (attn_fwd.cu) and packed sequences with
// grouped heads (attn_varlen.cu).
//
// Computes what the reference's _attn_fwd / _attn_fwd_inner compute
// (python/tutorials/06-fused-attention.py:25-187): O = softmax(Q K^T * sm_scale [causal]) V with
// an online softmax in base 2 (scores scaled by sm_scale * log2 e, :160-161), fp32 statistics,
// P rounded to the storage type before the second product (:66-69), O = acc / l rounded once,
// and M = m + log2(l) per row (:183-187).  Masked scores contribute exactly 0.
//
// One CTA owns 256 query rows of one (batch, head): two 128-row tiles that ping-pong so that the
// tensor pipe works on one tile while the other tile's softmax runs (one 128-row tile at head dim
// 256, where a tile's accumulator alone takes half of TMEM).  Sixteen warps:
//   warps 0-3 / 4-7   softmax of tile 0 / 1, one thread per query row (no cross-thread reduction):
//                     tcgen05.ld S, running max and sum, exp2, P packed to 16 bit and written back over S in TMEM
//                     (tcgen05.st) as the A operand of the second MMA.  The accumulator O is
//                     rescaled lazily: only when the running max grew by more than kRescaleThreshold does the
//                     warp multiply its O rows in TMEM (the reference rescales every step; the
//                     result is the same up to fp32 rounding since P and l carry the same factor).
//                     At the end: O / l -> storage type -> global, M -> global.
//   warp 8            MMA issuer (one elected lane): S_i = Q_i K_j^T (operands in shared memory) and
//                     O_i += P_i V_j (P from TMEM, V from shared memory, N-major).  MMAs of one
//                     thread execute in issue order, which is what lets P alias S.
//   warp 9            TMA producer: Q tiles once, then K_0, V_0, K_1, V_1 ... through a ring.
//   warps 10-15       lend their registers: the CTA's 64K registers are re-divided at run time
//                     (setmaxnreg) so that a softmax thread can hold a whole 128-column score row
//                     without spilling (216 registers; with ten warps the limit was 168 and the
//                     row spilled to local memory, an L2 round trip per value).
// The kernel is persistent: one CTA per SM takes work items (256 query rows of one head) from an
// atomic counter, head-major and heavy-first, so a head's K/V stay in L2, causal work balances, and
// the epilogue of one item overlaps the loads and first MMAs of the next.
// Packed sequences (PACKED): q and o are [T, Hq, D], k and v [T, Hkv, D], sequence b the rows cu[b] ..
// cu[b + 1].  The tensor maps cover all T rows, a tile starts at the sequence's first row plus a multiple
// of 128, and what it reads of the next sequence is masked by the length as the ragged end of a dense
// batch is; the rows of V behind the end are cleared in shared memory before the MMA (they are another
// sequence's: 0 * inf would reach this one).  The scheduling warp finds the item of a ticket from cu
// (PackedWalk) and publishes it, so the lengths are never needed on the host.  With several heads per
// k/v head a tile can also be 128 / fold positions of all `fold` of them, row = position * fold + head: the
// tensor map of q brings such a tile as one box, and the mask goes by the row's position.
// TMEM columns: S0 [0,128) S1 [128,256) O0 [256,256+D) O1 [384,384+D); P_i = first 64 columns of S_i
// at head dim 128, and columns [320,384) / [448,512) at head dim 64 (16-bit), where S_i of the next
// block is then issued before P_i V of this one.  Head dim 256: S [0,128), O [256,512).
#pragma once
#include <cfloat>
#include <cmath>
#include <cstdlib>
#include <type_traits>

#define B200_INLINE_WAIT_SLOW  // this kernel re-divides registers between its warpgroups
#include "common.cuh"
#include "host.h"

namespace tb {

namespace {

constexpr int BLK = 128;           // rows of a Q tile and of a K/V block
constexpr int FWD_THREADS = 512;   // 8 softmax warps, MMA warp, TMA warp, 6 warps that only lend their registers
// registers per thread after the re-division; one warp of each warpgroup shares a scheduler's 16K
// registers: (2 * 216 + 56 + 24) * 32 lanes = 16384
constexpr int REGS_SOFTMAX = 216, REGS_MMA_TMA = 56, REGS_IDLE = 24;
// Lazy rescale: the accumulator and the row sum keep their reference point m_ref until the running
// maximum has grown past it by more than this many log2 units, so P may reach 2^threshold: 15 for an
// fp16 P (largest finite value 65504), 60 for bf16 (fp32 range; the row sum of 2^14 such values and the
// accumulator stay far below the fp32 limit).  The rounding of P is relative, so its bits do not
// depend on the reference point as long as it stays in range.
template <bool BF16> constexpr float kRescaleThreshold = BF16 ? 60.0f : 15.0f;

// Column pairs out of every 8 whose exp2 is computed by a cubic on the FMA pipe (0: all on the
// special-function unit).
#ifndef B200_FWD_POLY
#define B200_FWD_POLY 2
#endif
constexpr int kPolyStride = 3;  // spreads the chosen pairs over a group of 8 (3 is coprime to 8)

struct FwdParams {
  void* o;
  float* m;  // [Z*H, N] base-2 log-sum-exp of the scaled scores
  float* row_max;  // optional [Z*H, N]: base-2 row maximum of the scaled scores (the old-style kernels' M / ln 2)
  long long o_sz, o_sh, o_sn;  // element strides of O
  int Z, H, N;
  int causal;
  float scale_log2;  // sm_scale * log2(e)
  int num_qb;        // query blocks (one work item each: 256 rows, 128 at head dim 256) per head
  int total_items;   // num_qb * Z * H
  int* sched_counter;  // work counter of this launch: zero at launch, put back to zero by the last CTA (packed: or nullptr)
  int o_tma;           // O is written through shared-memory staging and TMA stores
  unsigned* status;
};

struct PackedFwdParams : FwdParams {
  const int* cu;    // [batch + 1] offsets into the T rows (N = T, Z = 1, H = Hq)
  int batch, group;  // group: query heads per k/v head
  int by_level;      // order of the items, see PackedWalk
  int fold;          // heads of a tile: 1, or all of a group
  int tile_pos;      // positions of a tile: 128 / fold
  int item_pos, item_shift;    // positions of an item, and their log2 (-1: no power of two)
  int block_items, kv_items;   // items per block of item_pos positions, and of those per k/v head
  int lane_most;     // (2^26 - 1) / block_items, see PackedWalk::init
  int rest;          // rows that belong to no sequence: bit 0 set to zero in o, bit 1 set to -inf in m
};

// FP8: Q, K, V, P and O are 8-bit (e5m2, the reference's fp8 forward, 06-fused-attention.py:38-40,
// 66-69, 127): both products use kind::f8f6f4 MMAs with K = 32 per instruction; V is read with its
// key dimension contiguous (the layout the reference gives an fp8 V), i.e. as a K-major operand.
template <int D, bool FP8 = false>
struct FwdCfg {
  static constexpr int TILE_BYTES = BLK * D * (FP8 ? 1 : 2);   // one Q tile or one K / V block
  static constexpr int TILES = (D == 256) ? 1 : 2;             // 128-row query tiles per work item
  static constexpr int KV_STAGES = (D == 256) ? 2 : ((D == 128 && !FP8) ? 4 : 8);
  // tiles + barriers + TMEM slot + scheduler slots + alignment slack
  static constexpr int STG_BYTES = 32 * 128;  // epilogue staging of one softmax warp: 32 rows x 64 columns
  static constexpr size_t SMEM = (size_t)TILES * TILE_BYTES + (size_t)KV_STAGES * TILE_BYTES + 4 * TILES * STG_BYTES + (2 * KV_STAGES + 22) * 8 + 32 + 1024;
};

// one Q tile or K / V block of 128 rows: boxes of 128 bytes x 128 rows.  `along_rows`: the 8-bit V,
// whose map is [D rows][N keys]: the block is 128 keys wide and starts at key row0.
template <int D, bool FP8>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int row0, int h, int z,
                                          bool along_rows = false) {
  if constexpr (FP8) {
    if (along_rows) tma_load_4d(dst, map, bar, row0, 0, h, z);
    else tma_load_4d(dst, map, bar, 0, row0, h, z);
  } else {
#pragma unroll
    for (int b = 0; b < D / 64; ++b) tma_load_4d(dst + b * (BLK * 128), map, bar, b * 64, row0, h, z);
  }
}

// One work item = TILES * 128 query rows of one (batch, head).  Items are numbered head-major, heavy
// (late, long) query blocks first inside a head, and handed out through an atomic counter.
struct Item {
  int qb, zh, z, h, n0, n1, nmax;  // n_i: K/V blocks tile i visits; nmax: blocks the item streams
  int row0, kh, N;                 // first row of the sequence in the tensors, k/v head, length
};
// tile_pos: query positions of a tile
template <int TILES>
__device__ __forceinline__ void count_blocks(Item& it, bool causal, int tile_pos = BLK) {
  const int nkv_all = (it.N + BLK - 1) / BLK, end0 = (TILES * it.qb + 1) * tile_pos, end1 = end0 + tile_pos;
  // K/V blocks per tile: up to and including the block that holds the tile's last diagonal when causal
  it.n0 = causal ? min((end0 + BLK - 1) / BLK, nkv_all) : nkv_all;
  it.n1 = (TILES == 2) ? (causal ? min((end1 + BLK - 1) / BLK, nkv_all) : nkv_all) : 0;  // n0 <= n1 <= n0 + 1 with two tiles
  it.nmax = (TILES == 2) ? it.n1 : it.n0;
}
template <int TILES>
__device__ __forceinline__ Item decode_item(const FwdParams& p, int w) {
  Item it;
  it.zh = w / p.num_qb;
  it.qb = p.num_qb - 1 - (w % p.num_qb);
  it.z = it.zh / p.H;
  it.h = it.zh % p.H;
  it.row0 = 0;
  it.kh = it.h;
  it.N = p.N;
  count_blocks<TILES>(it, p.causal);
  return it;
}

// The items of a pack, in the order of their tickets; tickets only grow, so a walk keeps its place between
// draws.  Two orders, each made of classes of sequences that the walk counts as it comes to them:
//   by level   for every query block from the highest down, the sequences that have it, every head of each:
//              the longest items of the whole pack first, which evens out the end of the launch;
//   by length  for every number of query blocks from the highest down, the sequences of that length, their
//              k/v heads in turn, each with its blocks from the last to the first and the heads of its group:
//              the items that read the same K and V follow one another, which is what counts when the pack's
//              K and V do not stay in L2.
// Warp-collective.  Offsets outside [0, T] and negative lengths are cut, so none can lead out of the tensors.
struct PackedWalk {
  int blocks, base, count, total;  // the class: query blocks, its first ticket, sequences in it
  int at, before;                  // where the last draw's search ended: 32 sequences from `at`, `before` of the class before them
  int start0, len0, blocks0;       // of sequence `lane`: most batches need no more than this one load
  bool by_level;

  static __device__ __forceinline__ void extent(const PackedFwdParams& p, int b, int& start, int& len) {
    start = min(max(__ldg(p.cu + b), 0), p.N);
    len = max(min(__ldg(p.cu + b + 1), p.N) - start, 0);
  }
  __device__ __forceinline__ int seq_blocks(const PackedFwdParams& p, int b) const {  // b = lane + 32 i
    if (b < 32) return blocks0;
    int start, len;
    extent(p, b, start, len);
    return blocks_of(p, len);
  }
  static __device__ __forceinline__ int blocks_of(const PackedFwdParams& p, int len) {
    return p.item_shift >= 0 ? (len + p.item_pos - 1) >> p.item_shift : (len + p.item_pos - 1) / p.item_pos;
  }
  __device__ __forceinline__ bool in_class(int n) const { return by_level ? n >= blocks : n == blocks; }
  __device__ __forceinline__ int tickets(const PackedFwdParams& p) const { return count * p.block_items * (by_level ? 1 : blocks); }
  // the class of the most blocks below `below`
  __device__ __forceinline__ void enter(const PackedFwdParams& p, int below) {
    const int lane = threadIdx.x & 31;
    int most = 0, c = 0;
    for (int b = lane; b < p.batch; b += 32) {
      const int n = seq_blocks(p, b);
      most = max(most, by_level ? min(n, below - 1) : n < below ? n : 0);
    }
    blocks = (int)__reduce_max_sync(0xffffffffu, (unsigned)most);
    for (int b = lane; b < p.batch; b += 32) c += in_class(seq_blocks(p, b));
    count = blocks > 0 ? (int)__reduce_add_sync(0xffffffffu, (unsigned)c) : 0;
    at = before = 0;
  }
  __device__ __forceinline__ void init(const PackedFwdParams& p) {
    by_level = p.by_level;
    start0 = len0 = 0;
    if ((int)(threadIdx.x & 31) < p.batch) extent(p, threadIdx.x & 31, start0, len0);
    blocks0 = blocks_of(p, len0);
    // Decreasing offsets can name the same rows over and over, up to more tickets than an int counts: of such a pack
    // nothing is computed.  (32 lanes of lane_most are still below 2^31; a pack that takes its rows once has fewer in
    // one lane, or its o were a terabyte.)
    int sum = 0;
    for (int b = threadIdx.x & 31; b < p.batch; b += 32) sum = min(sum + seq_blocks(p, b), 1 << 30);
    total = (int)__reduce_add_sync(0xffffffffu, (unsigned)sum) * p.block_items;
    if (__any_sync(0xffffffffu, sum > p.lane_most)) total = 0;
    base = 0;
    enter(p, 0x7fffffff);
  }
  __device__ __forceinline__ Item find(const PackedFwdParams& p, int w) {  // w < total
    while (blocks > 0 && w - base >= tickets(p)) {
      base += tickets(p);
      enter(p, blocks);
    }
    const int lane = threadIdx.x & 31, per_seq = p.block_items * (by_level ? 1 : blocks);
    const int nth = count == 1 ? 0 : (w - base) / per_seq;
    int r = (w - base) - nth * per_seq;
    Item it;
    if (by_level) {
      it.kh = r / p.kv_items;
      it.qb = blocks - 1;
      r -= it.kh * p.kv_items;
    } else {
      it.kh = r / (p.kv_items * blocks);
      r -= it.kh * p.kv_items * blocks;
      it.qb = blocks - 1 - r / p.kv_items;
      r %= p.kv_items;
    }
    it.h = it.kh * p.group + r;  // (folded: one item per k/v head, the first of its heads)
    it.z = it.zh = 0;
    it.row0 = it.N = 0;
    for (; at < p.batch; at += 32) {
      const int b = at + lane;
      const unsigned in = __ballot_sync(0xffffffffu, b < p.batch && in_class(seq_blocks(p, b)));
      const int here = __popc(in);
      if (nth < before + here) {
        const bool me = ((in >> lane) & 1u) && __popc(in & ((1u << lane) - 1u)) == nth - before;
        const int src = __ffs(__ballot_sync(0xffffffffu, me)) - 1;
        it.row0 = __shfl_sync(0xffffffffu, start0, src);
        it.N = __shfl_sync(0xffffffffu, len0, src);
        if (at > 0) extent(p, at + src, it.row0, it.N);
        break;
      }
      before += here;
    }
    return it;
  }
};

template <int D, bool BF16, bool FP8, bool PACKED = false>
__global__ void __launch_bounds__(FWD_THREADS, 1)
attn_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o_map,
                const std::conditional_t<PACKED, PackedFwdParams, FwdParams> p) {
  using Cfg = FwdCfg<D, FP8>;
  constexpr int TILE = Cfg::TILE_BYTES, NST = Cfg::KV_STAGES, TILES = Cfg::TILES;
  constexpr int ITEM_ROWS = TILES * BLK;
  constexpr int MMA_WARP = 8, TMA_WARP = 9;
  constexpr bool WAIT_PAUSE = (D != 64);  // see mbar_wait_slow
  // The running maximum is NaN once a score was, where some weights come from the cubic.  (Head dim 64 and the 8-bit
  // forward have them all from ex2, which passes a NaN on; at head dim 64 the 1 to 2 % that this costs buy nothing.)
  constexpr bool KEEP_NAN = !FP8 && D != 64;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
  uint8_t* smem = smem_raw + pad;
  uint8_t* sq = smem;                    // Q tiles
  uint8_t* skv = smem + TILES * TILE;    // ring
  uint8_t* sstage = skv + NST * TILE;  // one 4 KiB buffer per softmax warp, 128-byte swizzled
  uint64_t* bars = reinterpret_cast<uint64_t*>(sstage + 4 * TILES * Cfg::STG_BYTES);
  uint64_t* q_full = bars;             // [2]
  uint64_t* kv_full = bars + 2;        // [NST]
  uint64_t* kv_empty = kv_full + NST;  // [NST]
  uint64_t* s_full = kv_empty + NST;   // [2] S_i(j) is in TMEM
  uint64_t* p_full = s_full + 2;       // [2 tiles][2 halves] columns [64h, 64h+64) of P_i(j) are in TMEM (and O_i rescaled if it had to be)
  uint64_t* o_full = p_full + 4;       // [2] last P V of tile i done
  uint64_t* q_empty = o_full + 2;      // [1] every S MMA of the item has read the Q tiles
  uint64_t* sched_full = q_empty + 1;  // [2] an item id was published
  uint64_t* sched_empty = sched_full + 2;  // [2] all 9 readers have taken it
  uint64_t* s_free = sched_empty + 2;      // [2] (head dim 64) the softmax warps of tile i hold S_i(j) in registers
  uint64_t* pv_done = s_free + 2;          // [2] (head dim 64) P_i(j) V_j is complete: O_i and the P buffer may be touched
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pv_done + 2);
  // [2] ticket; packed: [2][8] ticket (-1: none left), query block, head, first row, length
  volatile int* sched_item = reinterpret_cast<volatile int*>(tmem_slot + 2);
  constexpr int SLOT = PACKED ? 8 : 1;
  // first position of tile i in its sequence
  auto tile_row0 = [&](const Item& it, int i) {
    if constexpr (PACKED) return (it.qb * TILES + i) * p.tile_pos;
    else return it.qb * ITEM_ROWS + i * BLK;
  };
  // the item that a published slot names, for the warps that read it; false: no item is left
  auto take_item = [&](int slot, int w, Item& it) {
    if constexpr (PACKED) {
      it.qb = sched_item[8 * slot + 1];
      it.h = sched_item[8 * slot + 2];
      it.row0 = sched_item[8 * slot + 3];
      it.N = sched_item[8 * slot + 4];
      it.z = it.zh = 0;
      it.kh = it.h / p.group;
      count_blocks<TILES>(it, p.causal, p.tile_pos);
      return w >= 0;
    } else {
      if (w >= p.total_items) return false;
      it = decode_item<TILES>(p, w);
      return true;
    }
  };

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  B200_TRACE_DECL;  // trace builds: regions 0 / 1 = first softmax warp of tile 0 / 1, region 2 = MMA warp

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 128);
      mbar_init(&p_full[2 * i + 1], 128);
      mbar_init(&o_full[i], 1);
      mbar_init(&s_free[i], 4);  // one arrival per softmax warp of the tile
      mbar_init(&pv_done[i], 1);
      mbar_init(&sched_full[i], 1);
      mbar_init(&sched_empty[i], 1 + 4 * TILES);  // MMA warp + one lane of each softmax warp
    }
    mbar_init(q_empty, 1);
    for (int s = 0; s < NST; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    fence_barrier_init();
    cta_wait_flag_clear();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    tma_prefetch_desc(&tm_o_map);
  }
  if (warp == MMA_WARP) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  const uint32_t tm_s[2] = {tmem_base, tmem_base + 128};
  const uint32_t tm_o[2] = {tmem_base + 256, tmem_base + 384};
  // At head dim 64 the O accumulators leave 2 x 64 columns free, which hold P: with P out of the
  // S buffer, S_i(j+1) is issued as soon as the softmax warps have S_i(j) in registers instead of
  // after P_i(j) V_j, so the scores of the next block are ready when a tile's softmax comes back
  // for them.  (At head dim 128 TMEM is full and P overwrites S.)
  constexpr bool SEP_P = (D == 64) && !FP8;
  auto tm_p = [&](int i) { return SEP_P ? tmem_base + (i ? 448u : 320u) : tm_s[i]; };

  // Every role ends with its own copy of the teardown and returns: no code is shared after the
  // register budgets have diverged (values live across a join would have to sit in registers that
  // every budget has).
  auto teardown = [&](bool owner) {
    // after a recorded failure give copies in flight time to land before the CTA exits
    cta_linger_after_failure();
    tc_fence_before();
    __syncthreads();
    if (owner) {
      tc_fence_after();
      tmem_dealloc(tmem_base, 512);
    }
  };
  if (warp >= 12 || (TILES == 1 && warp >= 4 && warp < 8)) {
    // nothing else: these warps only lend registers and take part in the barriers at both ends
    // (at head dim 256 the second tile's softmax warpgroup has no tile)
    if constexpr (PACKED) {
      if (p.rest && warp >= 12) {
        const int first = min(max(p.cu[0], 0), p.N), end = max(min(p.cu[p.batch], p.N), first);
        const long long per_row = (long long)p.H * (D / 8);
        for (long long at = (long long)blockIdx.x * 128 + (threadIdx.x - 384); at < (first + p.N - end) * per_row;
             at += (long long)gridDim.x * 128) {
          const long long r = at / per_row, row = r < first ? r : r - first + end;
          const int h = (int)(at % per_row) / (D / 8), d = (int)(at % (D / 8)) * 8;
          if (p.rest & 1) *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.o) + row * p.o_sn + h * p.o_sh + d) = make_uint4(0u, 0u, 0u, 0u);
          if (d == 0 && (p.rest & 2)) p.m[(long long)h * p.N + row] = -INFINITY;
        }
      }
    }
    reg_dec<REGS_IDLE>();
    teardown(false);
    return;
  } else if (warp >= 10) {
    reg_dec<REGS_MMA_TMA>();
    teardown(false);
    return;
  } else if (warp == TMA_WARP) {
    reg_dec<REGS_MMA_TMA>();
    // ------------------------------------------------------------------ scheduler + TMA producer
    uint32_t s = 0, ph = 0;  // K/V ring position, runs on across items
    // the loads of the n-th item; one lane
    auto load_item = [&](const Item& it, uint32_t n) {
      mbar_wait<WAIT_PAUSE>(q_empty, (n & 1u) ^ 1u, p.status, SITE_FWD_Q);  // previous item's S MMAs are done with Q
      for (int i = 0; i < TILES; ++i) {
        if constexpr (PACKED) {  // the map's dimensions are {d, head, row}: boxes of 64 columns x fold heads x tile_pos rows
          mbar_expect_tx(&q_full[i], D * 2 * p.fold * p.tile_pos);
#pragma unroll
          for (int b = 0; b < D / 64; ++b)
            tma_load_4d(sq + i * TILE + b * (BLK * 128), &tm_q, &q_full[i], b * 64, it.h, it.row0 + tile_row0(it, i), 0);
        } else {
          mbar_expect_tx(&q_full[i], TILE);
          load_tile<D, FP8>(sq + i * TILE, &tm_q, &q_full[i], tile_row0(it, i), it.h, it.z);
        }
      }
      for (int j = 0; j < it.nmax; ++j) {
        for (int kv = 0; kv < 2; ++kv) {  // K_j then V_j
          mbar_wait<WAIT_PAUSE>(&kv_empty[s], ph ^ 1u, p.status, SITE_FWD_KV_EMPTY);
          mbar_expect_tx(&kv_full[s], TILE);
          load_tile<D, FP8>(skv + s * TILE, kv == 0 ? &tm_k : &tm_v, &kv_full[s], it.row0 + j * BLK, it.kh, it.z, kv == 1);
          if (++s == NST) { s = 0; ph ^= 1u; }
        }
      }
    };
    if constexpr (PACKED) {
      PackedWalk walk;
      walk.init(p);
      // the first ticket is the CTA's number, without a draw; the counter hands out those behind the grid's
      const int grid = (int)gridDim.x;
      int w = blockIdx.x;
      for (uint32_t n = 0;; ++n) {
        const bool more = w < walk.total;
        Item it{};
        if (more) it = walk.find(p, w);
        count_blocks<TILES>(it, p.causal, p.tile_pos);
        if (lane == 0) {
          const uint32_t slot = n & 1u, sph = (n >> 1) & 1u;
          mbar_wait<WAIT_PAUSE>(&sched_empty[slot], sph ^ 1u, p.status, SITE_FWD_SCHED);
          sched_item[8 * slot] = more ? w : -1;
          sched_item[8 * slot + 1] = it.qb;
          sched_item[8 * slot + 2] = it.h;
          sched_item[8 * slot + 3] = it.row0;
          sched_item[8 * slot + 4] = it.N;
          mbar_arrive(&sched_full[slot]);
          if (more) {
            load_item(it, n);
            if (p.sched_counter) {
              const int drawn = atomicAdd(p.sched_counter, 1);
              // every CTA that had a first item draws until its ticket is past the end: the last of those draws puts
              // the zero back for the next launch that is handed this counter
              if (drawn == max(walk.total - grid, 0) + min(grid, walk.total) - 1) atomicExch(p.sched_counter, 0);
              w = grid + drawn;
            } else {  // captured while graphs hold all counters: every grid-th ticket (4 x 4096 rows at 32/8 heads 580 against 487 us)
              w += grid;
            }
          }
        }
        __syncwarp();
        if (!more) break;
        w = __shfl_sync(0xffffffffu, w, 0);
      }
    } else if (lane == 0) {
      for (uint32_t n = 0;; ++n) {
        const int w = atomicAdd(p.sched_counter, 1);
        const uint32_t slot = n & 1u, sph = (n >> 1) & 1u;
        mbar_wait<WAIT_PAUSE>(&sched_empty[slot], sph ^ 1u, p.status, SITE_FWD_SCHED);
        sched_item[slot] = w;
        mbar_arrive(&sched_full[slot]);
        // every CTA draws exactly one ticket past the end: the last of them puts the zero back for the
        // next launch that is handed this counter
        if (w == p.total_items + (int)gridDim.x - 1) atomicExch(p.sched_counter, 0);
        if (w >= p.total_items) break;
        load_item(decode_item<TILES>(p, w), n);
      }
    }
    __syncwarp();
    teardown(false);
    return;
  } else if (warp == MMA_WARP) {
    reg_dec<REGS_MMA_TMA>();
    // ------------------------------------------------------------------ MMA issuer
    // The warp stays converged and an elected lane issues, for both tiles.  (Two issuing threads,
    // one per tile, were measured 20 % slower: MMAs of different threads interleave in the pipe
    // at a cost.)
    {
      constexpr int FMT = (BF16 || FP8) ? 1 : 0;  // kind::f16: bf16 = 1; kind::f8f6f4: e5m2 = 1
      constexpr uint32_t IDESC_S = make_idesc(FMT, FMT, 0, 0, 128, BLK);  // Q (K-major) x K (K-major)
      constexpr uint32_t IDESC_O = make_idesc(FMT, FMT, 0, FP8 ? 0 : 1, 128, D);  // P (TMEM) x V (N-major; K-major when 8-bit)
      // Q and K: rows of 128 bytes (64 16-bit or 128 8-bit elements per box), 128-byte swizzle; the
      // 8-bit forward at head dim 64 has rows of 64 bytes, 64-byte swizzle (8-row groups 512 B apart)
      constexpr bool ROW64 = FP8 && D == 64;
      const uint64_t dq0 = ROW64 ? smem_desc_sw64(smem_u32(sq), 0, 512) : smem_desc_sw128(smem_u32(sq), 0, 1024);
      const uint64_t dk0 = ROW64 ? smem_desc_sw64(smem_u32(skv), 0, 512) : smem_desc_sw128(smem_u32(skv), 0, 1024);
      const uint64_t dv0 = smem_desc_sw128(smem_u32(skv), FP8 ? 0 : BLK * 128, 1024);  // LBO: next 64-column box
      uint32_t s = 0, ph = 0;        // ring position of the next unconsumed K / V block
      uint32_t pcnt[2] = {0, 0};     // blocks of tile i whose P has been consumed (parity of p_full)
      [[maybe_unused]] uint32_t fcnt[2] = {0, 0};  // (head dim 64) blocks of tile i so far, across items (parity of s_free)

      auto issue_s = [&](int i, uint32_t stage) {  // S_i = Q_i K^T, D/16 MMAs
        const uint64_t dq = dq0 + i * (TILE >> 4), dk = dk0 + stage * (TILE >> 4);
        if constexpr (FP8) {
#pragma unroll
          for (int kk = 0; kk < D / 32; ++kk)  // one 128-byte box: 32 B (32 elements) per step
            umma_ss_elect<true>(tm_s[i], dq + kk * 2, dk + kk * 2, IDESC_S, kk != 0);
        } else {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = (kk >> 2) * ((BLK * 128) >> 4) + (kk & 3) * 2;  // 64-col box, 32 B per step
            umma_ss_elect<false>(tm_s[i], dq + off, dk + off, IDESC_S, kk != 0);
          }
        }
        tc_commit_elect(&s_full[i]);
        if (lane == 0) B200_TRACE_EVENT(p.status, 2, 0x40 | i);
      };
      // O_i (+)= P_i V: 8 MMAs of 16 kv rows; the second four wait for the second half of P
      auto issue_pv = [&](int i, uint32_t stage, uint32_t accum, uint32_t parity) {
        const uint64_t dv = dv0 + stage * (TILE >> 4);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (lane == 0) B200_TRACE_EVENT(p.status, 2, 0x10 | (i << 1) | h);
          mbar_wait<WAIT_PAUSE>(&p_full[2 * i + h], parity, p.status, SITE_FWD_P_FULL);
          if (lane == 0) B200_TRACE_EVENT(p.status, 2, 0x20 | (i << 1) | h);
          tc_fence_after();
          if constexpr (FP8) {
#pragma unroll
            for (int kk = 2 * h; kk < 2 * h + 2; ++kk)  // 32 keys per MMA: 8 TMEM columns of P, 32 B of the V rows
              umma_ts_f8_elect(tm_o[i], tm_p(i) + kk * 8, dv + kk * 2, IDESC_O, (accum | kk) != 0);
          } else {
#pragma unroll
            for (int kk = 4 * h; kk < 4 * h + 4; ++kk)
              umma_ts_f16_elect(tm_o[i], tm_p(i) + kk * 8, dv + kk * ((16 * 128) >> 4), IDESC_O, (accum | kk) != 0);
          }
        }
      };
      auto advance = [&]() { if (++s == NST) { s = 0; ph ^= 1u; } };
      // packed: the rows of V behind the sequence's end are another sequence's (or nobody's); P is zero
      // there, but 0 * inf and 0 * NaN are not.  The softmax of the item's last scores runs meanwhile.
      auto clear_tail = [&](const Item& it, int j, uint32_t stage) {
        if constexpr (PACKED) {
          const int rows = it.N - j * BLK;
          if (rows < BLK) {
            uint8_t* v = skv + stage * TILE;
#pragma unroll
            for (int bx = 0; bx < D / 64; ++bx)
              for (int off = rows * 128 + lane * 16; off < BLK * 128; off += 512)
                *reinterpret_cast<uint4*>(v + bx * (BLK * 128) + off) = make_uint4(0u, 0u, 0u, 0u);
            fence_proxy_async_smem();
            __syncwarp();
          }
        }
      };

      for (uint32_t n = 0;; ++n) {
        const uint32_t slot = n & 1u, sph = (n >> 1) & 1u;
        mbar_wait<WAIT_PAUSE>(&sched_full[slot], sph, p.status, SITE_FWD_SCHED);
        Item it;
        const bool some = take_item(slot, sched_item[SLOT * slot], it);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sched_empty[slot]);
        if (!some) break;
        const int n0 = it.n0, n1 = it.n1, nmax = it.nmax;

        // prologue: S_0(0), S_1(0) on K_0
        mbar_wait<WAIT_PAUSE>(&kv_full[s], ph, p.status, SITE_FWD_KV_FULL);
        mbar_wait<WAIT_PAUSE>(&q_full[0], n & 1u, p.status, SITE_FWD_Q);
        issue_s(0, s);
        if constexpr (TILES == 2) {
          mbar_wait<WAIT_PAUSE>(&q_full[1], n & 1u, p.status, SITE_FWD_Q);
          issue_s(1, s);
        }
        tc_commit_elect(&kv_empty[s]);
        if (nmax == 1) tc_commit_elect(q_empty);
        advance();
        for (int j = 0; j < nmax; ++j) {
          const uint32_t vs = s, vph = ph;  // V_j
          advance();
          const uint32_t ks = s, kph = ph;  // K_{j+1} (if any)
          const bool more1 = (TILES == 2) && (j + 1 < n1), more0 = (j + 1 < n0);
          if constexpr (SEP_P) {
            // the next scores first: S_i(j+1) only needs the S buffer, which is free once the
            // softmax warps have loaded S_i(j)
            if (more0) {
              mbar_wait<WAIT_PAUSE>(&s_free[0], fcnt[0]++ & 1u, p.status, SITE_FWD_S_EMPTY);
              tc_fence_after();
              mbar_wait<WAIT_PAUSE>(&kv_full[ks], kph, p.status, SITE_FWD_KV_FULL);
              issue_s(0, ks);
            } else if (j < n0) {
              ++fcnt[0];  // the tile's last block: its arrival is not waited for, the count goes on
            }
            if (more1) {
              mbar_wait<WAIT_PAUSE>(&s_free[1], fcnt[1]++ & 1u, p.status, SITE_FWD_S_EMPTY);
              tc_fence_after();
              mbar_wait<WAIT_PAUSE>(&kv_full[ks], kph, p.status, SITE_FWD_KV_FULL);
              issue_s(1, ks);
              tc_commit_elect(&kv_empty[ks]);
              if (j + 2 == n1) tc_commit_elect(q_empty);  // that was the item's last S: the Q tiles may be replaced
            } else {
              ++fcnt[1];
            }
            if (lane == 0) B200_TRACE_EVENT(p.status, 2, 0x50);
            mbar_wait<WAIT_PAUSE>(&kv_full[vs], vph, p.status, SITE_FWD_KV_FULL);
            if (lane == 0) B200_TRACE_EVENT(p.status, 2, 0x60);
            clear_tail(it, j, vs);
            if (j < n0) {
              issue_pv(0, vs, j > 0, pcnt[0]++ & 1u);
              tc_commit_elect(&pv_done[0]);
              if (j == n0 - 1) tc_commit_elect(&o_full[0]);
            }
            issue_pv(1, vs, j > 0, pcnt[1]++ & 1u);
            tc_commit_elect(&kv_empty[vs]);
            tc_commit_elect(&pv_done[1]);
            if (j == n1 - 1) tc_commit_elect(&o_full[1]);
            if (more1) advance();
          } else {
            if (lane == 0) B200_TRACE_EVENT(p.status, 2, 0x50);
            mbar_wait<WAIT_PAUSE>(&kv_full[vs], vph, p.status, SITE_FWD_KV_FULL);
            if (lane == 0) B200_TRACE_EVENT(p.status, 2, 0x60);
            clear_tail(it, j, vs);
            if (j < n0) {
              issue_pv(0, vs, j > 0, pcnt[0]++ & 1u);
              if (TILES == 1) tc_commit_elect(&kv_empty[vs]);
              if (j == n0 - 1) tc_commit_elect(&o_full[0]);
              if (more0) {
                mbar_wait<WAIT_PAUSE>(&kv_full[ks], kph, p.status, SITE_FWD_KV_FULL);
                issue_s(0, ks);
                if (TILES == 1) {
                  tc_commit_elect(&kv_empty[ks]);
                  if (j + 2 == n0) tc_commit_elect(q_empty);
                  advance();
                }
              }
            }
            if constexpr (TILES == 2) {
              issue_pv(1, vs, j > 0, pcnt[1]++ & 1u);
              tc_commit_elect(&kv_empty[vs]);
              if (j == n1 - 1) tc_commit_elect(&o_full[1]);
              if (more1) {
                mbar_wait<WAIT_PAUSE>(&kv_full[ks], kph, p.status, SITE_FWD_KV_FULL);
                issue_s(1, ks);
                tc_commit_elect(&kv_empty[ks]);
                if (j + 2 == n1) tc_commit_elect(q_empty);  // that was the item's last S: the Q tiles may be replaced
                advance();
              }
            }
          }
        }
      }
    }
    __syncwarp();
    teardown(true);
    return;
  } else {
    reg_inc<REGS_SOFTMAX>();
    // ------------------------------------------------------------------ softmax + epilogue
    // 4 warps per tile, one thread per query row.
    const int i = warp >> 2;                 // tile
    const uint32_t quarter = warp & 3u;      // TMEM lanes [32*quarter, +32)
    const int row_in_tile = quarter * 32 + lane;
    // packed: the row's position in the tile and its head; rows past tile_pos * fold are nobody's
    int pos_in_tile = row_in_tile, head_in_tile = 0;
    if constexpr (PACKED) {
      pos_in_tile = row_in_tile / p.fold;
      head_in_tile = row_in_tile - pos_in_tile * p.fold;
    }
    const uint32_t lane_addr = (quarter * 32u) << 16;
    const float scale = p.scale_log2;
    const bool vec_ok = ((reinterpret_cast<uintptr_t>(p.o) & 15) == 0) && ((p.o_sn & 7) == 0) && ((p.o_sh & 7) == 0) &&
                        ((p.o_sz & 7) == 0);
    uint32_t scnt = 0;  // blocks of this tile seen so far, across items (parity of s_full)

    for (uint32_t n = 0;; ++n) {
      const uint32_t slot = n & 1u, sph = (n >> 1) & 1u;
      Item it;
      if constexpr (PACKED) {
        mbar_wait<WAIT_PAUSE>(&sched_full[slot], sph, p.status, SITE_FWD_SCHED);
        const bool some = take_item(slot, sched_item[SLOT * slot], it);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sched_empty[slot]);
        if (!some) break;
      } else {
        int w = 0;
        if (lane == 0) {
          mbar_wait<WAIT_PAUSE>(&sched_full[slot], sph, p.status, SITE_FWD_SCHED);
          w = sched_item[slot];
          mbar_arrive(&sched_empty[slot]);
        }
        w = __shfl_sync(0xffffffffu, w, 0);
        if (!take_item(slot, w, it)) break;
      }
      const int row0 = tile_row0(it, i), head = it.h + head_in_tile;
      const int N = PACKED ? it.N : p.N;
      const int row = row0 + pos_in_tile;  // query index
      bool valid = row < N;
      if constexpr (PACKED) valid = valid && pos_in_tile < p.tile_pos;
      const int nb = i ? it.n1 : it.n0;
      float m_ref = -INFINITY, l = 0.f;
      float m_true = -INFINITY;  // the exact running maximum (m_ref lags it by up to the rescale threshold)
      const bool traced = quarter == 0 && lane == 0;  // used by trace builds only
      if (traced) B200_TRACE_EVENT(p.status, i, 0x100 | nb);

      for (int j = 0; j < nb; ++j, ++scnt) {
        mbar_wait<WAIT_PAUSE>(&s_full[i], scnt & 1u, p.status, SITE_FWD_S_FULL);
        if (traced) B200_TRACE_EVENT(p.status, i, 1);
        tc_fence_after();
        const int col0 = j * BLK;
        const bool need_mask = (p.causal && col0 + BLK - 1 > row0) || (col0 + BLK > N);
        // load 32 columns at a time; the row maximum of a chunk is taken while the next chunk loads
        uint32_t r[BLK];
        float mx4[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) mx4[u] = -INFINITY;
        tmem_ld32(tm_s[i] + lane_addr, r);
        tmem_ld_wait32(r);
#pragma unroll
        for (int c = 0; c < BLK; c += 32) {
          if (c + 32 < BLK) tmem_ld32(tm_s[i] + lane_addr + c + 32, r + c + 32);
          if (need_mask) {
            // columns of this chunk that the row may see: below N and, when causal, up to the row itself
            const int lim = min(N, p.causal ? row + 1 : N) - (col0 + c);
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (k >= lim) r[c + k] = __float_as_uint(-INFINITY);
          }
#pragma unroll
          for (int u = 0; u < 16; ++u)  // three-input maximum: one instruction per column pair
            mx4[u] = max3<KEEP_NAN>(mx4[u], __uint_as_float(r[c + 2 * u]), __uint_as_float(r[c + 2 * u + 1]));
          if (c + 32 < BLK) tmem_ld_wait32(r + c + 32);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) mx4[u] = max2<KEEP_NAN>(max3<KEEP_NAN>(mx4[u], mx4[u + 4], mx4[u + 8]), mx4[u + 12]);
        const float mx = max2<KEEP_NAN>(max2<KEEP_NAN>(mx4[0], mx4[1]), max2<KEEP_NAN>(mx4[2], mx4[3]));
        if constexpr (SEP_P) {
          // S_i(j) is in registers: the S buffer may take S_i(j+1)
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_free[i]);
        }
        // (head dim 64) before O_i or the P buffer is touched, P_i(j-1) V must be complete; on an
        // item's first block the epilogue's wait for the last P V of the previous item has seen to that
        auto wait_pv = [&]() {
          if (SEP_P && j > 0) {
            mbar_wait<WAIT_PAUSE>(&pv_done[i], (scnt - 1u) & 1u, p.status, SITE_FWD_O_READY);
            tc_fence_after();
          }
        };
        if (traced) B200_TRACE_EVENT(p.status, i, 2);
        // (mx = -inf: all scores of the block are, or a folded tile's first positions see none of a later block; weights 0)
        const float m_new = fmaxf(m_ref, mx * scale);
        m_true = max2<KEEP_NAN>(m_true, mx * scale);
        // lazy rescale of the accumulator (the ld/st below are warp collectives, so the warp
        // rescales if any of its rows has to)
        // true on the first block (m_ref = -inf), also if all its scores are -inf and the difference is NaN.  The 8-bit forward follows the exact running maximum,
        // as the reference does: the 2-bit mantissa of P makes its rounding depend on the scale
        // (packed: the rows behind the sequence's end hold another's values; they have no vote, or that
        // sequence's values would decide when this one's weights are rounded against which reference)
        const bool grow = (!PACKED || valid) && (FP8 ? (m_new > m_ref) : !((m_new - m_ref) <= kRescaleThreshold<BF16>));
        if (__any_sync(0xffffffffu, grow)) {
          // every row of the warp moves its reference point to its exact running maximum (this block
          // included): the pass over O is paid for by the row that had to move, and the others start
          // their next window from zero lag.  (Leaving 6 log2 units of headroom above the maximum as
          // well bought another 2-3 % on sharply peaked scores; not taken: it costs P 6 bits of range.)
          // (finite where the scores so far are all -inf: against it they have weight 0 and not NaN)
          if (!FP8) m_true = max2<KEEP_NAN>(m_true, -FLT_MAX);
          const float m_to = FP8 ? m_new : m_true;
          const float alpha = (FP8 && !grow) ? 1.f : ex2(m_ref - m_to);  // 0 on the first block
          if (!FP8 || grow) { m_ref = m_to; l *= alpha; }
          if (j > 0) {
            wait_pv();
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              tmem_ld32(tm_o[i] + lane_addr + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
              tmem_st32(tm_o[i] + lane_addr + c, o);
            }
          }
        }
        if (traced) B200_TRACE_EVENT(p.status, i, 3);
        wait_pv();  // (head dim 64) before the exponential loop, not inside it: a wait in the unrolled loop keeps the compiler from interleaving its chunks
        // a row that has seen a NaN or +inf: NaN, which makes all its weights NaN (without it the cubic below, which
        // knows neither, would give such a key a finite weight at some positions)
        const float neg_m = KEEP_NAN ? fmaf(m_true, 0.f, -m_ref) : -m_ref;
        float sum4[4] = {0.f, 0.f, 0.f, 0.f};
        [[maybe_unused]] uint64_t sum2[2] = {pk2(0.f, 0.f), pk2(0.f, 0.f)};
        [[maybe_unused]] const uint64_t scale2 = pk2(scale, scale), neg_m2 = pk2(neg_m, neg_m);
#pragma unroll
        for (int c = 0; c < BLK; c += 32) {
          uint32_t wv[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float p0, p1;
            if constexpr (SEP_P) {
              // head dim 64 is bound by instruction issue: packed fp32 arithmetic for the scaling
              // and the row sum (one issue slot per column pair)
              float x0, x1;
              upk2(fma2(pk2(__uint_as_float(r[c + 2 * k]), __uint_as_float(r[c + 2 * k + 1])), scale2, neg_m2), x0, x1);
              p0 = ex2(x0);
              p1 = ex2(x1);
              sum2[k & 1] = add2(sum2[k & 1], pk2(p0, p1));
            } else if (!FP8 && ((k * kPolyStride) & 7) < B200_FWD_POLY) {
              // some of the exponentials on the FMA pipe: the special-function unit is the
              // busiest unit of this loop
              float x0, x1;
              upk2(fma2(pk2(__uint_as_float(r[c + 2 * k]), __uint_as_float(r[c + 2 * k + 1])), scale2, neg_m2), x0, x1);
              ex2_cubic2(x0, x1, p0, p1);
              sum4[k & 3] += p0 + p1;
            } else {
              p0 = ex2(fmaf(__uint_as_float(r[c + 2 * k]), scale, neg_m));
              p1 = ex2(fmaf(__uint_as_float(r[c + 2 * k + 1]), scale, neg_m));
              sum4[k & 3] += p0 + p1;
            }
            if constexpr (FP8) {  // keep the values; four are packed into one column below
              r[c + 2 * k] = __float_as_uint(p0);
              r[c + 2 * k + 1] = __float_as_uint(p1);
            } else {
              wv[k] = pack2<BF16>(p0, p1);
            }
          }
          if constexpr (FP8) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              wv[k] = pack4_e5m2(__uint_as_float(r[c + 4 * k]), __uint_as_float(r[c + 4 * k + 1]),
                                 __uint_as_float(r[c + 4 * k + 2]), __uint_as_float(r[c + 4 * k + 3]));
            tmem_st8(tm_s[i] + lane_addr + (c >> 2), wv);
          } else {
            tmem_st16(tm_p(i) + lane_addr + (c >> 1), wv);
          }
          if (c == 32 || c == 96) {  // a half of P is complete: its four P V MMAs may start
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(&p_full[2 * i + (c >> 6)]);
          }
        }
        if constexpr (SEP_P) {
          float a0, a1, b0, b1;
          upk2(sum2[0], a0, a1);
          upk2(sum2[1], b0, b1);
          l += (a0 + a1) + (b0 + b1);
        } else {
          l += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
        }
        if (traced) B200_TRACE_EVENT(p.status, i, 4);
      }

      // epilogue: O / l and M.  It overlaps the next item's Q / K loads and first S MMAs; the next
      // item's first P V (which overwrites O) needs this tile's next P, i.e. comes after these
      // reads in program order.
      mbar_wait<WAIT_PAUSE>(&o_full[i], n & 1u, p.status, SITE_FWD_O_FULL);
      if (traced) B200_TRACE_EVENT(p.status, i, 8);
      tc_fence_after();
      const float inv_l = 1.f / l;
      uint16_t* orow = reinterpret_cast<uint16_t*>(p.o) + (long long)it.z * p.o_sz + (long long)head * p.o_sh +
                       (long long)(it.row0 + row) * p.o_sn;
      // packed: a box that reaches past the sequence's end would overwrite the next one (the lanes' positions rise)
      bool boxed = p.o_tma;
      [[maybe_unused]] unsigned rows_valid = 0;
      if constexpr (PACKED) {
        rows_valid = __ballot_sync(0xffffffffu, valid);
        boxed = boxed && rows_valid == 0xffffffffu;
      }
      if (PACKED ? rows_valid != 0 : boxed) {
        // 64 columns at a time: scaled, packed, written to this warp's swizzled staging buffer and
        // stored by TMA (full 128-byte lines; rows past N are clipped by the hardware).  A warp-wide
        // store of one row per lane touches 32 lines per instruction and made this epilogue cost
        // 5200 clk per item at D = 128.
        uint8_t* stg = sstage + warp * Cfg::STG_BYTES;
        const int warp_row0 = row0 + quarter * 32;
        if constexpr (FP8) {
          // 8-bit O: the D columns of a row are one line of the staging buffer
          if (lane == 0) tma_store_wait_read<0>();
          __syncwarp();
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld32(tm_o[i] + lane_addr + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
              uint32_t wv[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                wv[k] = pack4_e5m2(__uint_as_float(o[16 * ch + 4 * k]) * inv_l, __uint_as_float(o[16 * ch + 4 * k + 1]) * inv_l,
                                   __uint_as_float(o[16 * ch + 4 * k + 2]) * inv_l, __uint_as_float(o[16 * ch + 4 * k + 3]) * inv_l);
              // one line of the staging buffer per row: 128 bytes (128-byte swizzle) or, at head dim 64, 64 bytes
              const uint32_t off = (D == 64) ? sw64_offset(lane, (c >> 4) + ch) : sw128_offset(lane, (c >> 4) + ch);
              *reinterpret_cast<uint4*>(stg + off) = make_uint4(wv[0], wv[1], wv[2], wv[3]);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && warp_row0 < N) {
            tma_store_4d(&tm_o_map, stg, 0, warp_row0, it.h, it.z);
            tma_store_commit();
          }
        } else
#pragma unroll 1
        for (int c = 0; c < D; c += 64) {
          uint32_t o[64];
          tmem_ld32(tm_o[i] + lane_addr + c, o);
          tmem_ld32(tm_o[i] + lane_addr + c + 32, o + 32);
          tmem_ld_wait();
          if (traced) B200_TRACE_EVENT(p.status, i, 0xA);
          if (lane == 0) tma_store_wait_read<0>();  // the previous store has read the staging buffer
          __syncwarp();
          if (traced) B200_TRACE_EVENT(p.status, i, 0xB);
#pragma unroll
          for (int ch = 0; ch < 8; ++ch) {
            uint32_t wv[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              wv[k] = pack2<BF16>(__uint_as_float(o[8 * ch + 2 * k]) * inv_l, __uint_as_float(o[8 * ch + 2 * k + 1]) * inv_l);
            *reinterpret_cast<uint4*>(stg + sw128_offset(lane, ch)) = make_uint4(wv[0], wv[1], wv[2], wv[3]);
          }
          if constexpr (PACKED) {
            if (!boxed) {
              // rows stored one by one, eight lanes (128 bytes) to a row: what a box cannot take
              __syncwarp();
#pragma unroll
              for (int r4 = 0; r4 < 32; r4 += 4) {
                const int r = r4 + (lane >> 3);
                uint16_t* dst = reinterpret_cast<uint16_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(orow), r));
                const uint4 x = *reinterpret_cast<const uint4*>(stg + sw128_offset(r, lane & 7));
                if ((rows_valid >> r) & 1u) *reinterpret_cast<uint4*>(dst + c + (lane & 7) * 8) = x;
              }
              __syncwarp();
              continue;
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (traced) B200_TRACE_EVENT(p.status, i, 0xC);
          if (lane == 0 && (PACKED || warp_row0 < N)) {
            if constexpr (PACKED) tma_store_4d(&tm_o_map, stg, c, it.h, it.row0 + row, 0);  // (lane 0's position)
            else tma_store_4d(&tm_o_map, stg, c, warp_row0, it.h, it.z);
            tma_store_commit();
          }
        }
      } else if constexpr (!PACKED) {
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tmem_ld32(tm_o[i] + lane_addr + c, o);
          tmem_ld_wait();
          if (valid && FP8) {
            uint8_t* brow = reinterpret_cast<uint8_t*>(p.o) + (long long)it.z * p.o_sz + (long long)it.h * p.o_sh +
                            (long long)row * p.o_sn + c;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint32_t wq = pack4_e5m2(__uint_as_float(o[4 * k]) * inv_l, __uint_as_float(o[4 * k + 1]) * inv_l,
                                             __uint_as_float(o[4 * k + 2]) * inv_l, __uint_as_float(o[4 * k + 3]) * inv_l);
              for (int b = 0; b < 4; ++b) brow[4 * k + b] = (uint8_t)(wq >> (8 * b));
            }
          } else if (valid) {
            uint32_t wv[16];
#pragma unroll
            for (int k = 0; k < 16; ++k)
              wv[k] = pack2<BF16>(__uint_as_float(o[2 * k]) * inv_l, __uint_as_float(o[2 * k + 1]) * inv_l);
            if (vec_ok) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                reinterpret_cast<uint4*>(orow + c)[k] = make_uint4(wv[4 * k], wv[4 * k + 1], wv[4 * k + 2], wv[4 * k + 3]);
            } else {
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                orow[c + 2 * k] = (uint16_t)(wv[k] & 0xFFFFu);
                orow[c + 2 * k + 1] = (uint16_t)(wv[k] >> 16);
              }
            }
          }
        }
      }
      if constexpr (PACKED) {
        if (valid && p.m) p.m[(long long)head * p.N + it.row0 + row] = m_ref + log2f(l);
      } else if (valid) {
        p.m[(long long)it.zh * p.N + row] = m_ref + log2f(l);
      }
      if (!PACKED && valid && p.row_max) p.row_max[(long long)it.zh * p.N + row] = m_true == -FLT_MAX ? -INFINITY : m_true;
      if (traced) B200_TRACE_EVENT(p.status, i, 9);
    }
    if ((PACKED || p.o_tma) && lane == 0) tma_store_wait_read<0>();  // the staging buffer has been read: the CTA may exit, the writes land on their own
    teardown(false);
  }
}

}  // namespace

}  // namespace tb
