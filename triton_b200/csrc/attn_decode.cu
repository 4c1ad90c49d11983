// Attention of single tokens over the paged 8-bit cache.
//
//   s_j = sm_scale * ks_j * (q . k8_j),  o = sum_j 2^(s_j log2 e) * vs_j * v8_j / sum_j 2^(s_j log2 e)
// with k8, v8 the stored e4m3 values and ks, vs the scale (a power of two) of their page and head.
//
// Bound by memory: every cached byte is read once per group of 8 or 16 query heads, 4 * 8 flops per byte.
// CUDA cores could not keep up with that, and a tcgen05 tile has 128 rows where a group has a few, so the
// products run on warp-level MMAs (m16n8k16, fp32 accumulators) with the cache as the 16-row operand:
//   S^T = K Q^T   (16 tokens x 8 query heads),   O^T += V^T P^T   (16 head-dim indices x 8 query heads).
// A head dimension is a contraction in any order and tokens may take any slot, so each lane loads 16
// consecutive bytes of a row into the operand's registers: no transposes of K or V (P^T is turned by two
// 8 x 8 register transposes).  e4m3 -> fp16 is exact.  Each warp sends for the bytes of its next slabs (cp.async into
// shared memory of its own) as soon as it has read the current ones.
//
// Roundings to 16 bits: q in fp16 as it is, in bf16 times a power of two of its row that brings the row's
// largest value near fp16's top (8 significant bits fit; what lies 2^-29 below the largest loses bits);
// P to fp16, relative to a running reference that leaves the largest weight at 2^7 when it moves and lets it grow
// to 2^15 before it moves again, so that the weights of a long flat cache stay normal beside one large key (down to
// 2^-14, 21 log2 units below the largest just after a move).  The denominator sums the weights before this rounding.
// Scores, maxima, sums and O: fp32.
// The scale of V's page joins the weight's exponent before it is rounded (w = 2^(s + log2 vs - ref)), and
// the denominator keeps a reference of its own, so pages of very different scales cannot overflow fp16.
//
// A CTA takes one (sequence, k/v head, 8 or 16 query heads, chunk of tokens); its warps take 16-token
// slabs in turn and join at the end.  Several chunks of a sequence join as a cluster or in a second kernel.
//
// Measured (32/8 heads of 128 unless said; device time): 131000 tokens 48 us = 5.6 TB/s of the 6.55 a copy reaches;
// 24 sequences of 700 to 3900 tokens with 48/48 heads of 64 52 us = 5.0 TB/s, bound by its instructions (one query
// row in eight uses what the softmax computes); 96 sequences of 40 to 8000 tokens at 32/4 heads 42 us = 3.8 TB/s (about
// 750 chunks for 592 places); one of 1900 tokens 6.3 us, a row of latencies.
#include <cfloat>

#include "common.cuh"
#include "serving.h"

namespace tb {

namespace {

constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int SLAB = 16;             // tokens of one MMA
constexpr int MAX_CHUNK_SLABS = 256;  // page entries a CTA keeps in shared memory
constexpr float REF_NONE = -1.7e38f;   // reference point before the first token: finite, below every score
constexpr float LOG2E = 1.4426950408889634f;

// A warp takes STEP slabs at once (two: independent chains of MMAs) and owns room for one such step in shared
// memory; K's and V's half are refilled as soon as each has been read, so their bytes have the rest of the
// step to arrive.  (Room for two steps, hence 12 warps an SM instead of 16, was slower: the loop waits for
// its own instructions more than for memory.)
template <int D> constexpr int STEP = D == 256 ? 1 : 2;
template <int D> constexpr int ROOM = STEP<D> * SLAB * D * 2;
// the warps' rooms, in whose place their outputs are joined at the end
template <int D, int NT> constexpr int AREA = WARPS * (ROOM<D> > 8 * NT * (D + 4) * 4 ? ROOM<D> : 8 * NT * (D + 4) * 4);
// CTAs an SM holds (registers)
template <int D, int NT> constexpr int CTAS = D == 64 ? (NT == 1 ? 6 : 4) : D == 128 ? (NT == 1 ? 4 : 3) : 3;

struct DecodePlan {
  int nt;            // groups of 8 query heads per CTA
  int row_blocks;    // CTAs over the query heads of one k/v head
  int chunk;         // slabs per CTA
  int splits;        // chunks of the longest sequence the page table has room for
  bool cluster;      // a sequence's chunks are one cluster and join in shared memory
};

DecodePlan decode_plan(int B, int Hq, int Hkv, int D, int page_size, int max_pages) {
  DecodePlan p;
  const int G = Hq / Hkv;
  p.nt = (G > 8 && D <= 128) ? 2 : 1;
  p.row_blocks = (G + 8 * p.nt - 1) / (8 * p.nt);
  const int slabs = max_pages * (page_size / SLAB);
  const double pairs = (double)B * Hkv * p.row_blocks;
  const double room = 148.0 * (D == 64 ? (p.nt == 1 ? CTAS<64, 1> : CTAS<64, 2>) : D == 128 ? (p.nt == 1 ? CTAS<128, 1> : CTAS<128, 2>) : CTAS<256, 1>);
  // The chunk that is done first by this estimate, in slab times: a CTA takes its slabs and about 10 more for
  // its start and its join.  One sequence fills `room` CTAs at once; of several the lengths are not known here,
  // so half the table is taken as their mean, and the last CTAs to start run half a chunk alone.
  const int one_wave = pairs < room ? (int)((slabs + (int)(room / pairs) - 1) / (int)(room / pairs)) : MAX_CHUNK_SLABS;
  const int sizes[] = {8, 16, 24, 32, 48, 64, 96, 128, 192, 256, one_wave};
  double best = 0;
  p.chunk = 0;
  for (int chunk : sizes) {
    chunk = chunk < 8 ? 8 : chunk > MAX_CHUNK_SLABS ? MAX_CHUNK_SLABS : (chunk + 1) / 2 * 2;
    const double ctas = pairs * ((slabs + chunk - 1) / chunk);
    double t;
    if (B == 1) t = (ctas <= room ? 1.0 : ctas / room + 0.5) * (chunk + 10);
    else t = ctas * (0.5 * chunk + 10) / room + 0.5 * (chunk + 10);
    if (p.chunk == 0 || t < best) { best = t; p.chunk = chunk; }
  }
  p.splits = (slabs + p.chunk - 1) / p.chunk;
  if (p.splits < 1) p.splits = 1;
  // Few CTAs: up to eight chunks as a cluster, without workspace and second kernel.  Chunks twice as long cost the
  // GPU about what the second kernel does (1900 tokens of 32/8 heads: 8 slabs and a join 6.3 us, 16 in a cluster of
  // eight 6.2 us) and the host a launch and an allocation less (9.3 against 5.9 us).  Only where all CTAs
  // are resident at once: those without tokens wait for their cluster's others.
  p.cluster = false;
  if (p.splits > 1) {
    int size = 2;
    while (size < 8 && (slabs + size - 1) / size > 8) size *= 2;
    const int chunk = ((slabs + size - 1) / size + 1) / 2 * 2;
    if (pairs * size <= room && chunk <= p.chunk + 16 && chunk <= MAX_CHUNK_SLABS) {
      p.cluster = true;
      p.chunk = chunk;
      p.splits = size;
    }
  }
  return p;
}

struct DecodeParams {
  const uint8_t *k, *v;
  const float *k_scale, *v_scale;
  const int* table;
  long long table_stride;
  int pages, page_size, page_shift, max_pages, Hkv;  // page_size: 16 << page_shift
  const uint16_t* q;
  uint16_t* o;
  float* m;
  long long q_sb, q_sh, o_sb, o_sh;
  const int* lens;
  int B, Hq, G, row_blocks;
  float sm_scale_log2;
  int chunk, splits;
  float* ws_o;    // [B, Hq, splits, D] outputs of the chunks
  float* ws_lse;  // [B, Hq, splits] their base-2 log-sum-exp
};

struct __align__(8) SlabEntry {
  unsigned slab;    // index of 16-token slabs in the cache (times 16 * D bytes); ~0u: no page
  unsigned scales;  // exponent fields of K's scale and, 8 bits up, of V's
};

__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t x) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(x));
  return r;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// One slab (16 tokens of K, then of V) in shared memory: rows of D bytes, the 16-byte parts of a row XORed
// with bits of the row so that the loads below meet no bank twice (V at head dim 64: twice).
template <int D>
__device__ __forceinline__ uint32_t part_offset(int row, int part) {
  if constexpr (D == 64) return row * 64 + ((part ^ ((row >> 1) & 3)) << 4);
  else return row * D + ((part ^ (row & 7)) << 4);
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const uint8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// one slab's K or V into shared memory: consecutive lanes, consecutive 16 bytes
template <int D>
__device__ __forceinline__ void fetch_slab(uint32_t dst, const uint8_t* src, unsigned slab, int lane) {
  src += (unsigned long long)slab * (SLAB * D) + lane * 16;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const int q = i * 32 + lane;
    cp_async16(dst + part_offset<D>(q / (D / 16), q % (D / 16)), src + i * 512);
  }
}

// head-dim index of K's word w for lane c, and of V's byte pair i for lane g
template <int D>
__device__ __forceinline__ int k_index(int c, int w) { return (w >> 3) * 128 + c * (D == 64 ? 16 : 32) + (w & 7) * 4; }
template <int D>
__device__ __forceinline__ int v_index(int g, int i) { return (i >> 3) * 128 + g * (D == 64 ? 8 : 16) + (i & 7) * 2; }

// K in registers: rows g and g + 8 (g = lane / 4); of every 128 bytes of the row (or the 64 of head dim 64) the
// quarter of c = lane % 4.
template <int D>
__device__ __forceinline__ void read_k(uint32_t (&k)[2][D / 16], const uint8_t* at, int g, int c) {
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const int part = (D == 64) ? c : (i >> 1) * 8 + 2 * c + (i & 1);
      const uint4 x = *reinterpret_cast<const uint4*>(at + part_offset<D>(g + 8 * half, part));
      k[half][4 * i] = x.x; k[half][4 * i + 1] = x.y; k[half][4 * i + 2] = x.z; k[half][4 * i + 3] = x.w;
    }
}
// V in registers: of tokens 2c, 2c + 1, 2c + 8, 2c + 9 the D / 8 bytes of g, at head dim 256 16 in each half of the row
template <int D>
__device__ __forceinline__ void read_v(uint32_t (&v)[4][D / 32], const uint8_t* at, int g, int c) {
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int row = 2 * c + (t & 1) + (t >> 1) * 8;
    if constexpr (D == 64) {
      const uint2 x = *reinterpret_cast<const uint2*>(at + part_offset<D>(row, g >> 1) + (g & 1) * 8);
      v[t][0] = x.x; v[t][1] = x.y;
    } else {
#pragma unroll
      for (int i = 0; i < D / 128; ++i) {
        const uint4 x = *reinterpret_cast<const uint4*>(at + part_offset<D>(row, i * 8 + g));
        v[t][4 * i] = x.x; v[t][4 * i + 1] = x.y; v[t][4 * i + 2] = x.z; v[t][4 * i + 3] = x.w;
      }
    }
  }
}

// shared memory of the cluster's CTA `rank`, at the place of this CTA's `p`
__device__ __forceinline__ uint32_t in_cluster(const float* p, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ float4 ld_cluster4(const float* p, int rank) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(in_cluster(p, rank)) : "memory");
  return x;
}
__device__ __forceinline__ float ld_cluster(const float* p, int rank) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(in_cluster(p, rank)) : "memory");
  return x;
}

template <int D, int NT, bool BF16, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, CTAS<D, NT>) attn_decode_kernel(const DecodeParams p) {
  constexpr int ROWS = 8 * NT, KSTEPS = D / 16, MT = D / 16;
  constexpr int OSTRIDE = D + 4;  // floats; + 4 spreads the rows over the banks
  constexpr int SL = STEP<D>, SIDE = SLAB * D;
  extern __shared__ __align__(128) uint8_t smem[];  // [WARPS] SL slabs of K, then of V; then the chunk's page entries
  SlabEntry* table = reinterpret_cast<SlabEntry*>(smem + AREA<D, NT>);
  __shared__ float s_refw[WARPS][ROWS], s_refp[WARPS][ROWS], s_l[WARPS][ROWS];
  __shared__ int s_seen[WARPS];
  __shared__ float s_lse[ROWS];
  float* so = reinterpret_cast<float*>(smem);                                     // [WARPS][ROWS][OSTRIDE], after the loop

  if constexpr (!CLUSTER) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (none waiting: nothing)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int split = blockIdx.x, b = blockIdx.z;
  const int h = blockIdx.y / p.row_blocks, rb = blockIdx.y % p.row_blocks;
  const int row0 = rb * ROWS, nrows = min(ROWS, p.G - row0);  // query heads h * G + row0 + [0, nrows)
  // Every load of the start that needs no other goes out first: the length, q, the chunk's pages (the table has
  // room for the chunk whatever the length is); then the bytes are sent for, and the scales after them.
  const int len_given = __ldg(p.lens + b);
  const int s0 = split * p.chunk, sh = p.page_shift, room = p.max_pages << sh;  // 2^sh slabs a page
  int pages[MAX_CHUNK_SLABS / THREADS];
#pragma unroll
  for (int k = 0; k < MAX_CHUNK_SLABS / THREADS; ++k) {
    const int i = threadIdx.x + k * THREADS;
    pages[k] = (i < p.chunk && s0 + i < room) ? __ldg(p.table + b * p.table_stride + ((s0 + i) >> sh)) : -1;
  }
  // q as the B operand: for k-step s the four head-dim indices of K's word s
  uint2 raw[NT][KSTEPS];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const uint16_t* qr = p.q + b * p.q_sb + (long long)(h * p.G + row0 + min(t * 8 + g, nrows - 1)) * p.q_sh;
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) raw[t][s] = __ldg(reinterpret_cast<const uint2*>(qr + k_index<D>(c, s)));
  }
  const int len = min(max(len_given, 0), p.max_pages * p.page_size);
  const int nslabs = (len + SLAB - 1) / SLAB;
  const int s1 = min(s0 + p.chunk, nslabs), count = s1 - s0;
  const bool whole = nslabs <= p.chunk;
  if (split > 0 && s0 >= nslabs) {  // (chunk 0 of an empty sequence writes the zeros)
    if constexpr (CLUSTER)
      if (!whole) { cluster_sync(); cluster_sync(); }
    return;
  }
#pragma unroll
  for (int k = 0; k < MAX_CHUNK_SLABS / THREADS; ++k) {
    const int i = threadIdx.x + k * THREADS;
    // any entry that is no page's number names no page: its tokens are left out
    if (i < count) table[i].slab = (pages[k] >= 0 && pages[k] < p.pages) ? (((unsigned)pages[k] * p.Hkv + h) << sh) + ((s0 + i) & ((1 << sh) - 1)) : ~0u;
    else if (i < (count + SL - 1) / SL * SL) table[i].slab = ~0u;  // a step may reach past the last slab
  }
  const uint8_t* room_k = smem + warp * ROOM<D>;
  const uint8_t* room_v = room_k + SL * SIDE;
  SlabEntry ahead[SL];  // the step whose bytes are being sent for
  auto look = [&](int i) {
#pragma unroll
    for (int u = 0; u < SL; ++u) ahead[u] = SlabEntry{~0u, 0u};
    if (i < count) {
      if constexpr (SL == 2) {
        const uint4 e = *reinterpret_cast<const uint4*>(table + i);
        ahead[0] = SlabEntry{e.x, e.y};
        ahead[1] = SlabEntry{e.z, e.w};
      } else {
        ahead[0] = table[i];
      }
    }
  };
  auto fetch = [&](const uint8_t* dst, const uint8_t* src) {
#pragma unroll
    for (int u = 0; u < SL; ++u)
      if (ahead[u].slab != ~0u) fetch_slab<D>(smem_u32(dst) + u * SIDE, src, ahead[u].slab, lane);
    cp_async_commit();
  };
  __syncthreads();
  look(warp * SL);
  fetch(room_k, p.k);
  fetch(room_v, p.v);
  for (int i = threadIdx.x; i < count; i += THREADS)
    if (table[i].slab != ~0u) {
      const unsigned ph = table[i].slab >> sh;
      const unsigned ks = __float_as_uint(__ldg(p.k_scale + ph)), vs = __float_as_uint(__ldg(p.v_scale + ph));
      table[i].scales = (ks >> 23 & 0xFFu) | (vs >> 23 & 0xFFu) << 8;
    }

  uint32_t qf[KSTEPS][NT][2];
  float fac[NT][2];  // per query row 2c, 2c + 1 of each group: score of one unit of the product, log2 units
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (t * 8 + g >= nrows) {
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s) raw[t][s] = make_uint2(0, 0);
    }
    float f = p.sm_scale_log2;
    if constexpr (!BF16) {
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s) { qf[s][t][0] = raw[t][s].x; qf[s][t][1] = raw[t][s].y; }
    } else {
      float mx = 0.f;
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s) {
        mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(raw[t][s].x << 16)), fabsf(__uint_as_float(raw[t][s].x & 0xFFFF0000u))));
        mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(raw[t][s].y << 16)), fabsf(__uint_as_float(raw[t][s].y & 0xFFFF0000u))));
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // 2^up brings the largest value into [2^14, 2^15), or as near as a factor of 2^126 does; a row with an infinity stays put
      const int ex = (int)(__float_as_uint(mx) >> 23) - 127;
      const int up = ex > 127 ? 0 : min(14 - ex, 126);
      const float mul = __uint_as_float((uint32_t)(up + 127) << 23);
      f *= __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s) {
        qf[s][t][0] = pack2<false>(__uint_as_float(raw[t][s].x << 16) * mul, __uint_as_float(raw[t][s].x & 0xFFFF0000u) * mul);
        qf[s][t][1] = pack2<false>(__uint_as_float(raw[t][s].y << 16) * mul, __uint_as_float(raw[t][s].y & 0xFFFF0000u) * mul);
      }
    }
    // row r's factor sits in the lanes 4r .. 4r + 3; this lane's scores are of rows 2c and 2c + 1
    fac[t][0] = __shfl_sync(0xffffffffu, f, 8 * c);
    fac[t][1] = __shfl_sync(0xffffffffu, f, 8 * c + 4);
  }

  float o[MT][NT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][t][j] = 0.f;
  float refw[NT][2], refp[NT][2], l[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 2; ++j) { refw[t][j] = REF_NONE; refp[t][j] = REF_NONE; l[t][j] = 0.f; }
  int seen = 0;

  __syncthreads();
  look(warp * SL);  // with the scales
  for (int i = warp * SL; i < count; i += WARPS * SL) {
    float ks[SL], ev[SL];
    int left[SL];  // tokens of the slab that exist
    bool any_here = false;
#pragma unroll
    for (int u = 0; u < SL; ++u) {
      const SlabEntry e = ahead[u];
      ks[u] = __uint_as_float((e.scales & 0xFFu) << 23);
      ev[u] = __uint_as_float(0x4B000000u | (e.scales >> 8 & 0xFFu)) - (8388608.f + 127.f);  // the field as a number, less its bias
      left[u] = e.slab != ~0u ? len - (s0 + i + u) * SLAB : 0;
      any_here |= e.slab != ~0u;
    }
    look(i + WARPS * SL);
    float s[SL][NT][4];
    cp_async_wait<1>();  // K is here, V may be under way
    __syncwarp();
    if (any_here) {
      uint32_t kr[SL][2][D / 16];
#pragma unroll
      for (int u = 0; u < SL; ++u) read_k<D>(kr[u], room_k + u * SIDE, g, c);
#pragma unroll
      for (int u = 0; u < SL; ++u)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[u][t][j] = 0.f;
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
        for (int u = 0; u < SL; ++u) {
          const uint32_t x = kr[u][0][k], y = kr[u][1][k];
          const uint32_t a0 = e4m3x2_to_f16x2((uint16_t)x), a1 = e4m3x2_to_f16x2((uint16_t)y);
          const uint32_t a2 = e4m3x2_to_f16x2((uint16_t)(x >> 16)), a3 = e4m3x2_to_f16x2((uint16_t)(y >> 16));
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_f16(s[u][t], a0, a1, a2, a3, qf[k][t][0], qf[k][t][1]);
        }
    }
    __syncwarp();
    fetch(room_k, p.k);
    uint32_t pb[SL][NT][2];
    if (any_here) {
      seen = 1;
      // scores in log2 units; those behind the last token and of pages that do not exist vanish
#pragma unroll
      for (int u = 0; u < SL; ++u) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          // the factors first: a large q over small keys (2^120 and 2^-120, say) is an ordinary score, its product with
          // q's factor alone is infinite.  Finite, so that a product of 0 stays 0 under factors that pass fp32's range.
          float f0, f1;
          upk2(mul2(pk2(fac[t][0], fac[t][1]), pk2(ks[u], ks[u])), f0, f1);
          const uint64_t f = pk2(fminf(f0, FLT_MAX), fminf(f1, FLT_MAX));
#pragma unroll
          for (int j = 0; j < 4; j += 2)  // two query rows at a time
            upk2(mul2(pk2(s[u][t][j], s[u][t][j + 1]), f), s[u][t][j], s[u][t][j + 1]);
        }
        if (left[u] < SLAB) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (g + (j >> 1) * 8 >= left[u]) s[u][t][j] = -INFINITY;
        }
      }
      // new reference points where a weight would pass 2^15 (numerators) or 2^40 (denominator)
      float topw[NT][2], topp[NT][2];
      bool grow = false;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float a = fmaxf(s[0][t][j], s[0][t][j + 2]);
          topp[t][j] = a;
          topw[t][j] = a + ev[0];
#pragma unroll
          for (int u = 1; u < SL; ++u) {
            a = fmaxf(s[u][t][j], s[u][t][j + 2]);
            topp[t][j] = fmaxf(topp[t][j], a);
            topw[t][j] = fmaxf(topw[t][j], a + ev[u]);
          }
          grow |= (topw[t][j] - refw[t][j] > 15.f) || (topp[t][j] - refp[t][j] > 40.f);
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float tw = topw[t][j], tp = topp[t][j];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
              tw = fmaxf(tw, __shfl_xor_sync(0xffffffffu, tw, x));
              tp = fmaxf(tp, __shfl_xor_sync(0xffffffffu, tp, x));
            }
            const float w = fmaxf(refw[t][j], tw - 7.f), q = fmaxf(refp[t][j], tp);
            const float alpha = ex2(refw[t][j] - w);
            l[t][j] *= ex2(refp[t][j] - q);
            refw[t][j] = w;
            refp[t][j] = q;
#pragma unroll
            for (int k = 0; k < MT; ++k) { o[k][t][j] *= alpha; o[k][t][j + 2] *= alpha; }
          }
      }
#pragma unroll
      for (int u = 0; u < SL; ++u)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float w[4], q[4];
          const uint64_t ew = pk2(ev[u] - refw[t][0], ev[u] - refw[t][1]), ep = pk2(-refp[t][0], -refp[t][1]);
          uint64_t sum = pk2(l[t][0], l[t][1]);
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            const uint64_t x = pk2(s[u][t][j], s[u][t][j + 1]);
            upk2(add2(x, ew), w[j], w[j + 1]);
            upk2(add2(x, ep), q[j], q[j + 1]);
            w[j] = ex2(w[j]);
            w[j + 1] = ex2(w[j + 1]);
            sum = add2(sum, pk2(ex2(q[j]), ex2(q[j + 1])));
          }
          upk2(sum, l[t][0], l[t][1]);
          pb[u][t][0] = transpose8x8(pack2<false>(w[0], w[1]));
          pb[u][t][1] = transpose8x8(pack2<false>(w[2], w[3]));
        }
    }
    cp_async_wait<1>();  // V is here
    __syncwarp();
    if (any_here) {
#pragma unroll
      for (int u = 0; u < SL; ++u) {
        uint32_t vr[4][D / 32];
        read_v<D>(vr, room_v + u * SIDE, g, c);
        if (left[u] < SLAB) {  // what an earlier owner of the page left, NaN perhaps: 0 * NaN is not 0
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (2 * c + (t & 1) + (t >> 1) * 8 >= left[u]) {
#pragma unroll
              for (int k = 0; k < D / 32; ++k) vr[t][k] = 0u;
            }
        }
#pragma unroll
        for (int k = 0; k < MT; ++k) {
          const uint32_t sel = (k & 1) ? 0x7362u : 0x5140u;
          const uint32_t x = __byte_perm(vr[0][k >> 1], vr[1][k >> 1], sel);
          const uint32_t y = __byte_perm(vr[2][k >> 1], vr[3][k >> 1], sel);
          const uint32_t a0 = e4m3x2_to_f16x2((uint16_t)x), a1 = e4m3x2_to_f16x2((uint16_t)(x >> 16));
          const uint32_t a2 = e4m3x2_to_f16x2((uint16_t)y), a3 = e4m3x2_to_f16x2((uint16_t)(y >> 16));
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_f16(o[k][t], a0, a1, a2, a3, pb[u][t][0], pb[u][t][1]);
        }
      }
    }
    __syncwarp();
    fetch(room_v, p.v);
  }
  cp_async_wait<0>();

  // join the warps
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[t][j] += __shfl_xor_sync(0xffffffffu, l[t][j], x);
      if (g == 0) {
        s_refw[warp][t * 8 + 2 * c + j] = refw[t][j];
        s_refp[warp][t * 8 + 2 * c + j] = refp[t][j];
        s_l[warp][t * 8 + 2 * c + j] = l[t][j];
      }
    }
  if (lane == 0) s_seen[warp] = seen;
  __syncthreads();  // also: every warp is done with its ring, whose memory takes O now
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = t * 8 + 2 * c + j;
      float top = s_refw[0][row];
#pragma unroll
      for (int w = 1; w < WARPS; ++w) top = fmaxf(top, s_refw[w][row]);
      const float alpha = ex2(refw[t][j] - top);
      float* dst = so + (warp * ROWS + row) * OSTRIDE;
#pragma unroll
      for (int k = 0; k < MT; ++k)
        *reinterpret_cast<float2*>(dst + v_index<D>(g, k)) = make_float2(o[k][t][j] * alpha, o[k][t][j + 2] * alpha);
    }
  __syncthreads();
  int any = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) any |= s_seen[w];
  for (int i = threadIdx.x; i < nrows * (D / 4); i += THREADS) {
    const int row = i / (D / 4), d = i % (D / 4) * 4;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    float topw = REF_NONE, topp = REF_NONE, sum = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float4 y = *reinterpret_cast<const float4*>(so + (w * ROWS + row) * OSTRIDE + d);
      x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
      topw = fmaxf(topw, s_refw[w][row]);
      topp = fmaxf(topp, s_refp[w][row]);
    }
#pragma unroll
    for (int w = 0; w < WARPS; ++w) sum += s_l[w][row] * ex2(s_refp[w][row] - topp);
    const float f = any ? ex2(topw - topp) / sum : 0.f;  // no token: zeros
    x.x *= f; x.y *= f; x.z *= f; x.w *= f;
    const float lse = any ? topp + log2f(sum) : -INFINITY;
    const long long hq = h * p.G + row0 + row;
    if (whole) {
      uint16_t* dst = p.o + b * p.o_sb + hq * p.o_sh + d;
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<BF16>(x.x, x.y), pack2<BF16>(x.z, x.w));
      if (d == 0 && p.m) p.m[(long long)b * p.Hq + hq] = lse;
    } else if constexpr (CLUSTER) {
      *reinterpret_cast<float4*>(so + row * OSTRIDE + d) = x;  // (only this thread has read the place)
      if (d == 0) s_lse[row] = lse;
    } else {
      const long long at = ((long long)b * p.Hq + hq) * p.splits + split;
      *reinterpret_cast<float4*>(p.ws_o + at * D + d) = x;
      if (d == 0) p.ws_lse[at] = lse;
    }
  }
  if constexpr (CLUSTER) {
    if (whole) return;  // the same for every CTA of the cluster: none waits
    __syncwarp();
    cluster_sync();  // every chunk's output and log-sum-exp are in its CTA's shared memory
    const int parts = (nslabs + p.chunk - 1) / p.chunk;
    for (int i = split * THREADS + threadIdx.x; i < nrows * (D / 4); i += parts * THREADS) {
      const int row = i / (D / 4), d = i % (D / 4) * 4;
      float4 part[8];
      float lse[8], top = -INFINITY;
      bool nan = false;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        part[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        lse[k] = -INFINITY;
        if (k < parts) {
          part[k] = ld_cluster4(so + row * OSTRIDE + d, k);
          lse[k] = ld_cluster(s_lse + row, k);
        }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        nan |= lse[k] != lse[k];
        top = fmaxf(top, lse[k]);
      }
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float w = lse[k] == -INFINITY ? 0.f : ex2(lse[k] - top);  // (-inf: none of its pages exists)
        sum += w;
        x.x += w * part[k].x; x.y += w * part[k].y; x.z += w * part[k].z; x.w += w * part[k].w;
      }
      const bool tokens = top != -INFINITY || nan;
      const float f = tokens ? 1.f / sum : 0.f;
      const long long hq = h * p.G + row0 + row;
      *reinterpret_cast<uint2*>(p.o + b * p.o_sb + hq * p.o_sh + d) =
          make_uint2(pack2<BF16>(x.x * f, x.y * f), pack2<BF16>(x.z * f, x.w * f));
      if (d == 0 && p.m) p.m[(long long)b * p.Hq + hq] = tokens ? top + log2f(sum) : -INFINITY;
    }
    __syncwarp();
    cluster_sync();  // nobody reads this CTA's shared memory any more
  }
}

// Joins the chunks of a (sequence, query head): o = sum_i 2^(lse_i - max) o_i / sum_i 2^(lse_i - max).  A CTA
// each, D / 4 threads over the head dim and the groups of them over the chunks, several loads in flight (one warp
// that walked 147 chunks took 73 us); a group's first eight are sent for before the weights are known.  It is
// launched while the chunks still run, so its launch latency is hidden.
constexpr int JOIN_MOST = 512;  // weights kept at a time
constexpr int JOIN_AHEAD = 8;
template <int D, bool BF16, int THREADS>
__global__ void __launch_bounds__(THREADS) attn_decode_join_kernel(const DecodeParams p) {
  constexpr int LANES = D / 4, GROUPS = THREADS / LANES, WARPS = THREADS / 32;
  __shared__ float s_w[JOIN_MOST], s_red[WARPS];
  __shared__ __align__(16) float s_acc[GROUPS][D];
  asm volatile("griddepcontrol.wait;" ::: "memory");  // until the chunks' kernel has ended and its writes are seen
  const int tid = threadIdx.x, lane = tid & 31, d = (tid % LANES) * 4, grp = tid / LANES;
  const long long row = blockIdx.x;
  const int b = (int)(row / p.Hq), hq = (int)(row % p.Hq);
  const int len = min(max(p.lens[b], 0), p.max_pages * p.page_size);
  const int nslabs = (len + SLAB - 1) / SLAB;
  if (nslabs <= p.chunk) return;  // its only chunk has written the output
  const int n = (nslabs + p.chunk - 1) / p.chunk;
  const float* lse = p.ws_lse + row * p.splits;
  const float* src = p.ws_o + row * p.splits * D + d;
  auto reduce = [&](float x, bool sum) {  // over the CTA, the same bits in every thread
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, x, i);
      x = sum ? x + y : fmaxf(x, y);
    }
    __syncthreads();
    if (lane == 0) s_red[tid >> 5] = x;
    __syncthreads();
    x = s_red[0];
#pragma unroll
    for (int i = 1; i < WARPS; ++i) x = sum ? x + s_red[i] : fmaxf(x, s_red[i]);
    return x;
  };
  float4 ahead[JOIN_AHEAD];
#pragma unroll
  for (int k = 0; k < JOIN_AHEAD; ++k) {
    ahead[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (grp + k * GROUPS < n) ahead[k] = __ldcg(reinterpret_cast<const float4*>(src + (long long)(grp + k * GROUPS) * D));
  }
  float top = -INFINITY;
  bool nan = false;  // a chunk of NaN: its row is NaN, which a maximum would pass over
  for (int i = tid; i < n; i += THREADS) {
    const float x = lse[i];
    nan |= x != x;
    top = fmaxf(top, x);
  }
  top = reduce(top, false);
  nan = __syncthreads_or(nan);
  const bool any = top != -INFINITY || nan;  // -inf: none of the pages exists
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
  for (int i0 = 0; i0 < n; i0 += JOIN_MOST) {
    const int m = min(JOIN_MOST, n - i0);
    __syncthreads();
    for (int i = tid; i < m; i += THREADS) {
      const float x = lse[i0 + i], w = x == -INFINITY ? 0.f : ex2(x - top);
      s_w[i] = w;
      sum += w;
    }
    __syncthreads();
    int i = grp;
    if (i0 == 0) {
#pragma unroll
      for (int k = 0; k < JOIN_AHEAD; ++k, i += GROUPS) {
        const float w = i < m ? s_w[i] : 0.f;
        acc.x += w * ahead[k].x; acc.y += w * ahead[k].y; acc.z += w * ahead[k].z; acc.w += w * ahead[k].w;
      }
    }
#pragma unroll 8
    for (; i < m; i += GROUPS) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(src + (long long)(i0 + i) * D));
      const float w = s_w[i];
      acc.x += w * x.x; acc.y += w * x.y; acc.z += w * x.z; acc.w += w * x.w;
    }
  }
  sum = reduce(sum, true);
  *reinterpret_cast<float4*>(&s_acc[grp][d]) = acc;
  __syncthreads();
  if (grp == 0) {
#pragma unroll
    for (int i = 1; i < GROUPS; ++i) {
      const float4 x = *reinterpret_cast<const float4*>(&s_acc[i][d]);
      acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
    }
    const float f = any ? 1.f / sum : 0.f;
    *reinterpret_cast<uint2*>(p.o + b * p.o_sb + hq * p.o_sh + d) =
        make_uint2(pack2<BF16>(acc.x * f, acc.y * f), pack2<BF16>(acc.z * f, acc.w * f));
    if (tid == 0 && p.m) p.m[row] = any ? top + log2f(sum) : -INFINITY;
  }
}

template <int D, int NT, bool BF16, bool CLUSTER>
int launch_t(DeviceCtx* ctx, cudaStream_t stream, const DecodeParams& p) {
  constexpr size_t most = (size_t)AREA<D, NT> + (MAX_CHUNK_SLABS + STEP<D>) * sizeof(SlabEntry);
  static std::atomic<bool> attr_done[64];
  if (int rc = ensure_dynamic_smem(attn_decode_kernel<D, NT, BF16, CLUSTER>, most, ctx->device, attr_done, "attn decode")) return rc;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3((unsigned)p.splits, (unsigned)(p.Hkv * p.row_blocks), (unsigned)p.B);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = (size_t)AREA<D, NT> + (size_t)(p.chunk + STEP<D>) * sizeof(SlabEntry);
  cfg.stream = stream;
  cfg.attrs = attr;
  if constexpr (CLUSTER) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)p.splits, 1, 1};
    cfg.numAttrs = 1;
  }
  cudaError_t e = cudaLaunchKernelEx(&cfg, attn_decode_kernel<D, NT, BF16, CLUSTER>, p);
  if (!CLUSTER && e == cudaSuccess && p.splits > 1) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3((unsigned)(p.B * p.Hq));
    cfg.dynamicSmemBytes = 0;
    // many chunks, hence few sequences: more threads, so that all of a row's loads are still ahead
    if (p.splits > 32) {
      cfg.blockDim = dim3(512);
      e = cudaLaunchKernelEx(&cfg, attn_decode_join_kernel<D, BF16, 512>, p);
    } else {
      e = cudaLaunchKernelEx(&cfg, attn_decode_join_kernel<D, BF16, THREADS>, p);
    }
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(B200_ERR_CUDA, "attn decode launch: %s", cudaGetErrorString(e));
  }
  return B200_OK;
}

template <int D, int NT, bool BF16>
int launch_c(DeviceCtx* ctx, cudaStream_t stream, const DecodeParams& p, bool cluster) {
  return cluster ? launch_t<D, NT, BF16, true>(ctx, stream, p) : launch_t<D, NT, BF16, false>(ctx, stream, p);
}

template <bool BF16>
int launch_d(DeviceCtx* ctx, cudaStream_t stream, const DecodeParams& p, int D, const DecodePlan& pl) {
  if (D == 64) return pl.nt == 2 ? launch_c<64, 2, BF16>(ctx, stream, p, pl.cluster) : launch_c<64, 1, BF16>(ctx, stream, p, pl.cluster);
  if (D == 128) return pl.nt == 2 ? launch_c<128, 2, BF16>(ctx, stream, p, pl.cluster) : launch_c<128, 1, BF16>(ctx, stream, p, pl.cluster);
  return launch_c<256, 1, BF16>(ctx, stream, p, pl.cluster);
}

}  // namespace

size_t attn_decode_workspace_bytes(int B, int Hq, int Hkv, int D, int page_size, int max_pages) {
  const DecodePlan pl = decode_plan(B, Hq, Hkv, D, page_size, max_pages);
  return pl.splits > 1 && !pl.cluster ? (size_t)B * Hq * pl.splits * (D + 1) * sizeof(float) : 0;
}

int launch_attn_decode(DeviceCtx* ctx, cudaStream_t stream, const AttnDecodeArgs& a) {
  const DecodePlan pl = decode_plan(a.B, a.Hq, a.c.Hkv, a.c.D, a.c.page_size, a.c.max_pages);
  DecodeParams p{};
  p.k = a.c.k; p.v = a.c.v; p.k_scale = a.c.k_scale; p.v_scale = a.c.v_scale;
  p.table = a.c.table; p.table_stride = a.c.table_stride;
  p.pages = a.c.pages; p.page_size = a.c.page_size; p.page_shift = a.c.page_size == 16 ? 0 : a.c.page_size == 32 ? 1 : a.c.page_size == 64 ? 2 : 3; p.max_pages = a.c.max_pages; p.Hkv = a.c.Hkv;
  p.q = static_cast<const uint16_t*>(a.q); p.o = static_cast<uint16_t*>(a.o); p.m = a.m;
  p.q_sb = a.q_sb; p.q_sh = a.q_sh; p.o_sb = a.o_sb; p.o_sh = a.o_sh;
  p.lens = a.lens; p.B = a.B; p.Hq = a.Hq; p.G = a.Hq / a.c.Hkv; p.row_blocks = pl.row_blocks;
  p.sm_scale_log2 = a.sm_scale * LOG2E;
  p.chunk = pl.chunk; p.splits = pl.splits;
  p.ws_o = a.workspace;
  p.ws_lse = a.workspace ? a.workspace + (size_t)a.B * a.Hq * pl.splits * a.c.D : nullptr;
  return a.dtype == B200_BF16 ? launch_d<true>(ctx, stream, p, a.c.D, pl) : launch_d<false>(ctx, stream, p, a.c.D, pl);
}

}  // namespace tb
