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
// consecutive bytes of a row straight from global memory into the operand's registers: no shared memory,
// no transposes of K or V (P^T is turned by two 8 x 8 register transposes).  e4m3 -> fp16 is exact.
//
// Roundings to 16 bits: q in fp16 as it is, in bf16 times a power of two of its row that brings the row's
// largest value near fp16's top (8 significant bits fit; what lies 2^-29 below the largest loses bits);
// P to fp16, relative to a running reference that leaves weights 2^-7 .. 2^15 at the top, so that the
// weights of a long flat cache stay normal beside one large key.  Scores, maxima, sums and O: fp32.
// The scale of V's page joins the weight's exponent before it is rounded (w = 2^(s + log2 vs - ref)), and
// the denominator keeps a reference of its own, so pages of very different scales cannot overflow fp16.
//
// A CTA takes one (sequence, k/v head, 8 or 16 query heads, chunk of tokens); its warps take 16-token
// slabs in turn and join at the end.  With more than one chunk a second kernel joins those.
#include "common.cuh"
#include "serving.h"

namespace tb {

namespace {

constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int SLAB = 16;             // tokens of one MMA
constexpr int MAX_CHUNK_SLABS = 1024;  // page-table entries a CTA keeps in shared memory
constexpr float REF_NONE = -1.7e38f;   // reference point before the first token: finite, below every score
constexpr float LOG2E = 1.4426950408889634f;

struct DecodePlan {
  int nt;            // groups of 8 query heads per CTA
  int row_blocks;    // CTAs over the query heads of one k/v head
  int chunk;         // slabs per CTA
  int splits;        // chunks of the longest sequence the page table has room for
};

DecodePlan decode_plan(int B, int Hq, int Hkv, int D, int page_size, int max_pages) {
  DecodePlan p;
  const int G = Hq / Hkv;
  p.nt = (G > 8 && D <= 128) ? 2 : 1;
  p.row_blocks = (G + 8 * p.nt - 1) / (8 * p.nt);
  const long long slabs = (long long)max_pages * (page_size / SLAB);
  const long long ctas = (long long)B * Hkv * p.row_blocks;
  const long long want = 148 * 8;
  long long splits = (want + ctas - 1) / ctas;
  long long chunk = (slabs + splits - 1) / splits;
  if (chunk < 16) chunk = 16;
  if (chunk > MAX_CHUNK_SLABS) chunk = MAX_CHUNK_SLABS;
  p.chunk = (int)chunk;
  p.splits = (int)((slabs + chunk - 1) / chunk);
  if (p.splits < 1) p.splits = 1;
  return p;
}

struct DecodeParams {
  const uint8_t *k, *v;
  const float *k_scale, *v_scale;
  const int* table;
  long long table_stride;
  int pages, page_size, max_pages, Hkv;
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

struct SlabEntry {
  unsigned slab;  // index of 16-token slabs in the cache (times 16 * D bytes); ~0u: no page
  float ks;
  float ev;       // log2 of V's scale
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
__device__ __forceinline__ uint4 ldg_stream(const uint8_t* p) {  // read once: no room in L1
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
__device__ __forceinline__ uint2 ldg_stream8(const uint8_t* p) {
  uint2 r;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}

// One slab's bytes in registers.  K: words of rows g and g + 8 (g = lane / 4), for each 64-byte part of the
// row the 16 bytes at 16 * (lane % 4).  V: of tokens 2c, 2c + 1, 2c + 8, 2c + 9 (c = lane % 4) the D / 8
// bytes at (D / 8) * g.
template <int D>
struct SlabRegs {
  uint32_t k[2][D / 16];
  uint32_t v[4][D / 32];
};

template <int D>
__device__ __forceinline__ void load_slab(SlabRegs<D>& r, const DecodeParams& p, unsigned slab, int g, int c) {
  const unsigned long long at = (unsigned long long)slab * (SLAB * D);
  const uint8_t* kp = p.k + at + g * D + c * 16;
#pragma unroll
  for (int part = 0; part < D / 64; ++part) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint4 x = ldg_stream(kp + half * 8 * D + part * 64);
      r.k[half][4 * part] = x.x; r.k[half][4 * part + 1] = x.y; r.k[half][4 * part + 2] = x.z; r.k[half][4 * part + 3] = x.w;
    }
  }
  const uint8_t* vp = p.v + at + g * (D / 8);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint8_t* row = vp + (2 * c + (i & 1) + (i >> 1) * 8) * D;
    if constexpr (D == 64) {
      const uint2 x = ldg_stream8(row);
      r.v[i][0] = x.x; r.v[i][1] = x.y;
    } else {
#pragma unroll
      for (int part = 0; part < D / 128; ++part) {
        const uint4 x = ldg_stream(row + part * 16);
        r.v[i][4 * part] = x.x; r.v[i][4 * part + 1] = x.y; r.v[i][4 * part + 2] = x.z; r.v[i][4 * part + 3] = x.w;
      }
    }
  }
}

template <bool BF16>
__device__ __forceinline__ float to_f32(uint16_t x) {
  if constexpr (BF16) return __uint_as_float((uint32_t)x << 16);
  else return __half2float(__ushort_as_half(x));
}
template <bool BF16>
__device__ __forceinline__ uint16_t from_f32(float x) {
  if constexpr (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(x));
  else return __half_as_ushort(__float2half_rn(x));
}

template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(THREADS) attn_decode_kernel(const DecodeParams p) {
  constexpr int ROWS = 8 * NT, KSTEPS = D / 16, MT = D / 16;
  constexpr int OSTRIDE = D + 4;  // floats; + 4 spreads the rows over the banks
  extern __shared__ __align__(16) uint8_t smem[];
  SlabEntry* table = reinterpret_cast<SlabEntry*>(smem);                          // [chunk]
  __shared__ float s_refw[WARPS][ROWS], s_refp[WARPS][ROWS], s_l[WARPS][ROWS];
  __shared__ int s_seen[WARPS];
  float* so = reinterpret_cast<float*>(smem);                                     // [WARPS][ROWS][OSTRIDE], after the loop

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int split = blockIdx.x, b = blockIdx.z;
  const int h = blockIdx.y / p.row_blocks, rb = blockIdx.y % p.row_blocks;
  const int row0 = rb * ROWS, nrows = min(ROWS, p.G - row0);  // query heads h * G + row0 + [0, nrows)
  const int len = min(max(p.lens[b], 0), p.max_pages * p.page_size);
  const int nslabs = (len + SLAB - 1) / SLAB;
  const int s0 = split * p.chunk, s1 = min(s0 + p.chunk, nslabs);
  if (split > 0 && s0 >= nslabs) return;  // (chunk 0 of an empty sequence writes the zeros)
  const bool whole = nslabs <= p.chunk;

  // this chunk's pages and their scales
  const int spp = p.page_size / SLAB;
  for (int i = threadIdx.x; i < s1 - s0; i += THREADS) {
    const int slab = s0 + i, pg = p.table[b * p.table_stride + slab / spp];
    SlabEntry e;
    e.slab = ~0u; e.ks = 0.f; e.ev = 0.f;
    if (pg >= 0 && pg < p.pages) {  // any other entry names no page: its tokens are left out
      const unsigned ph = (unsigned)pg * p.Hkv + h;
      e.slab = ph * spp + slab % spp;
      e.ks = p.k_scale[ph];
      e.ev = (float)((int)((__float_as_uint(p.v_scale[ph]) >> 23) & 0xFFu) - 127);
    }
    table[i] = e;
  }

  // q as the B operand: for the 64-byte part and word of k-step s, the four head-dim indices of that word
  uint32_t qf[KSTEPS][NT][2];
  float fac[NT][2];  // per query row 2c, 2c + 1 of each group: score of one unit of the product, log2 units
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int row = t * 8 + g;
    const uint16_t* qr = p.q + b * p.q_sb + (long long)(h * p.G + row0 + min(row, nrows - 1)) * p.q_sh;
    uint2 raw[KSTEPS];
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) {
      raw[s] = __ldg(reinterpret_cast<const uint2*>(qr + (s >> 2) * 64 + c * 16 + (s & 3) * 4));
      if (row >= nrows) raw[s] = make_uint2(0, 0);
    }
    float f = p.sm_scale_log2;
    if constexpr (!BF16) {
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s) { qf[s][t][0] = raw[s].x; qf[s][t][1] = raw[s].y; }
    } else {
      float mx = 0.f;
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s) {
        mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(raw[s].x << 16)), fabsf(__uint_as_float(raw[s].x & 0xFFFF0000u))));
        mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(raw[s].y << 16)), fabsf(__uint_as_float(raw[s].y & 0xFFFF0000u))));
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // 2^up brings the largest value into [2^14, 2^15); a row of zeros or with an infinity stays put
      const int ex = (int)(__float_as_uint(mx) >> 23) - 127;
      const int up = (ex < -112 || ex > 127) ? 0 : min(14 - ex, 126);
      const float mul = __uint_as_float((uint32_t)(up + 127) << 23);
      f *= __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s) {
        qf[s][t][0] = pack2<false>(__uint_as_float(raw[s].x << 16) * mul, __uint_as_float(raw[s].x & 0xFFFF0000u) * mul);
        qf[s][t][1] = pack2<false>(__uint_as_float(raw[s].y << 16) * mul, __uint_as_float(raw[s].y & 0xFFFF0000u) * mul);
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
  const int count = s1 - s0;
  SlabRegs<D> cur, nxt;
  if (warp < count && table[warp].slab != ~0u) load_slab<D>(cur, p, table[warp].slab, g, c);
  for (int i = warp; i < count; i += WARPS) {
    const SlabEntry e = table[i];
    if (i + WARPS < count && table[i + WARPS].slab != ~0u) load_slab<D>(nxt, p, table[i + WARPS].slab, g, c);
    if (e.slab != ~0u) {
      seen = 1;
      float s[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[t][j] = 0.f;
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k) {
        const uint32_t x = cur.k[0][k], y = cur.k[1][k];
        const uint32_t a0 = e4m3x2_to_f16x2((uint16_t)x), a1 = e4m3x2_to_f16x2((uint16_t)y);
        const uint32_t a2 = e4m3x2_to_f16x2((uint16_t)(x >> 16)), a3 = e4m3x2_to_f16x2((uint16_t)(y >> 16));
#pragma unroll
        for (int t = 0; t < NT; ++t) mma_f16(s[t], a0, a1, a2, a3, qf[k][t][0], qf[k][t][1]);
      }
      // scores in log2 units; columns behind the last token vanish, and so do V's rows there (their bytes
      // are whatever an earlier owner of the page left)
      const int left = len - (s0 + i) * SLAB;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[t][j] = (s[t][j] * fac[t][j & 1]) * e.ks;
      if (left < SLAB) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (g + (j >> 1) * 8 >= left) s[t][j] = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (2 * c + (j & 1) + (j >> 1) * 8 >= left) {
#pragma unroll
            for (int k = 0; k < D / 32; ++k) cur.v[j][k] = 0u;
          }
      }
      // new reference points where a weight would pass 2^15 (numerators) or 2^40 (denominator)
      bool grow = false;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float top = fmaxf(s[t][j], s[t][j + 2]);
          grow |= (top + e.ev - refw[t][j] > 15.f) || (top - refp[t][j] > 40.f);
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float top = fmaxf(s[t][j], s[t][j + 2]);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            const float w = fmaxf(refw[t][j], top + e.ev - 7.f), q = fmaxf(refp[t][j], top);
            const float alpha = ex2(refw[t][j] - w);
            l[t][j] *= ex2(refp[t][j] - q);
            refw[t][j] = w;
            refp[t][j] = q;
#pragma unroll
            for (int k = 0; k < MT; ++k) { o[k][t][j] *= alpha; o[k][t][j + 2] *= alpha; }
          }
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w[j] = ex2(s[t][j] + e.ev - refw[t][j & 1]);
          l[t][j & 1] += ex2(s[t][j] - refp[t][j & 1]);
        }
        pb[t][0] = transpose8x8(pack2<false>(w[0], w[1]));
        pb[t][1] = transpose8x8(pack2<false>(w[2], w[3]));
      }
#pragma unroll
      for (int k = 0; k < MT; ++k) {
        const uint32_t sel = (k & 1) ? 0x7362u : 0x5140u;
        const uint32_t x = __byte_perm(cur.v[0][k >> 1], cur.v[1][k >> 1], sel);
        const uint32_t y = __byte_perm(cur.v[2][k >> 1], cur.v[3][k >> 1], sel);
        const uint32_t a0 = e4m3x2_to_f16x2((uint16_t)x), a1 = e4m3x2_to_f16x2((uint16_t)(x >> 16));
        const uint32_t a2 = e4m3x2_to_f16x2((uint16_t)y), a3 = e4m3x2_to_f16x2((uint16_t)(y >> 16));
#pragma unroll
        for (int t = 0; t < NT; ++t) mma_f16(o[k][t], a0, a1, a2, a3, pb[t][0], pb[t][1]);
      }
    }
    cur = nxt;
  }

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
  __syncthreads();  // also: every warp is done with the page entries, whose memory takes O now
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
      for (int k = 0; k < MT; ++k)  // head-dim indices of lane (g, c), tile k: (D / 8) g + 2k and + 1
        *reinterpret_cast<float2*>(dst + g * (D / 8) + 2 * k) = make_float2(o[k][t][j] * alpha, o[k][t][j + 2] * alpha);
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
    } else {
      const long long at = ((long long)b * p.Hq + hq) * p.splits + split;
      *reinterpret_cast<float4*>(p.ws_o + at * D + d) = x;
      if (d == 0) p.ws_lse[at] = lse;
    }
  }
}

// Joins the chunks of one (sequence, query head) per warp: o = sum_i 2^(lse_i - max) o_i / sum_i 2^(lse_i - max).
template <int D, bool BF16>
__global__ void __launch_bounds__(THREADS) attn_decode_join_kernel(const DecodeParams p) {
  constexpr int PER = D / 32;
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5);
  if (row >= (long long)p.B * p.Hq) return;
  const int b = (int)(row / p.Hq), hq = (int)(row % p.Hq);
  const int len = min(max(p.lens[b], 0), p.max_pages * p.page_size);
  const int nslabs = (len + SLAB - 1) / SLAB;
  if (nslabs <= p.chunk) return;  // its only chunk has written the output
  const int n = (nslabs + p.chunk - 1) / p.chunk;
  const float* lse = p.ws_lse + row * p.splits;
  float top = REF_NONE;
  for (int i = lane; i < n; i += 32) top = fmaxf(top, lse[i]);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
  float acc[PER], sum = 0.f;
  bool any = false;
#pragma unroll
  for (int j = 0; j < PER; ++j) acc[j] = 0.f;
  const float* src = p.ws_o + row * p.splits * D + lane * PER;
  for (int i = 0; i < n; ++i) {
    const float li = lse[i];
    if (li == -INFINITY) continue;  // a chunk none of whose pages exists
    any = true;
    const float w = ex2(li - top);
    sum += w;
#pragma unroll
    for (int j = 0; j < PER; ++j) acc[j] += w * src[(long long)i * D + j];
  }
  const float f = any ? 1.f / sum : 0.f;
  uint16_t* dst = p.o + b * p.o_sb + hq * p.o_sh + lane * PER;
#pragma unroll
  for (int j = 0; j < PER; j += 2)
    *reinterpret_cast<uint32_t*>(dst + j) = pack2<BF16>(acc[j] * f, acc[j + 1] * f);
  if (lane == 0 && p.m) p.m[row] = any ? top + log2f(sum) : -INFINITY;
}

template <int D, int NT, bool BF16>
int launch_t(DeviceCtx* ctx, cudaStream_t stream, const DecodeParams& p) {
  constexpr size_t out_bytes = (size_t)WARPS * 8 * NT * (D + 4) * sizeof(float);
  constexpr size_t most = MAX_CHUNK_SLABS * sizeof(SlabEntry) > out_bytes ? MAX_CHUNK_SLABS * sizeof(SlabEntry) : out_bytes;
  static std::atomic<bool> attr_done[64];
  if (int rc = ensure_dynamic_smem(attn_decode_kernel<D, NT, BF16>, most, ctx->device, attr_done, "attn decode")) return rc;
  const size_t table_bytes = (size_t)p.chunk * sizeof(SlabEntry);
  const size_t smem = table_bytes > out_bytes ? table_bytes : out_bytes;
  const dim3 grid((unsigned)p.splits, (unsigned)(p.Hkv * p.row_blocks), (unsigned)p.B);
  attn_decode_kernel<D, NT, BF16><<<grid, THREADS, smem, stream>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess && p.splits > 1) {
    attn_decode_join_kernel<D, BF16><<<(unsigned)(((long long)p.B * p.Hq + WARPS - 1) / WARPS), THREADS, 0, stream>>>(p);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return fail(B200_ERR_CUDA, "attn decode launch: %s", cudaGetErrorString(e));
  return B200_OK;
}

template <bool BF16>
int launch_d(DeviceCtx* ctx, cudaStream_t stream, const DecodeParams& p, int D, int nt) {
  if (D == 64) return nt == 2 ? launch_t<64, 2, BF16>(ctx, stream, p) : launch_t<64, 1, BF16>(ctx, stream, p);
  if (D == 128) return nt == 2 ? launch_t<128, 2, BF16>(ctx, stream, p) : launch_t<128, 1, BF16>(ctx, stream, p);
  return launch_t<256, 1, BF16>(ctx, stream, p);
}

}  // namespace

size_t attn_decode_workspace_bytes(int B, int Hq, int Hkv, int D, int page_size, int max_pages) {
  const DecodePlan pl = decode_plan(B, Hq, Hkv, D, page_size, max_pages);
  return pl.splits > 1 ? (size_t)B * Hq * pl.splits * (D + 1) * sizeof(float) : 0;
}

int launch_attn_decode(DeviceCtx* ctx, cudaStream_t stream, const AttnDecodeArgs& a) {
  const DecodePlan pl = decode_plan(a.B, a.Hq, a.c.Hkv, a.c.D, a.c.page_size, a.c.max_pages);
  DecodeParams p{};
  p.k = a.c.k; p.v = a.c.v; p.k_scale = a.c.k_scale; p.v_scale = a.c.v_scale;
  p.table = a.c.table; p.table_stride = a.c.table_stride;
  p.pages = a.c.pages; p.page_size = a.c.page_size; p.max_pages = a.c.max_pages; p.Hkv = a.c.Hkv;
  p.q = static_cast<const uint16_t*>(a.q); p.o = static_cast<uint16_t*>(a.o); p.m = a.m;
  p.q_sb = a.q_sb; p.q_sh = a.q_sh; p.o_sb = a.o_sb; p.o_sh = a.o_sh;
  p.lens = a.lens; p.B = a.B; p.Hq = a.Hq; p.G = a.Hq / a.c.Hkv; p.row_blocks = pl.row_blocks;
  p.sm_scale_log2 = a.sm_scale * LOG2E;
  p.chunk = pl.chunk; p.splits = pl.splits;
  p.ws_o = a.workspace;
  p.ws_lse = a.workspace ? a.workspace + (size_t)a.B * a.Hq * pl.splits * a.c.D : nullptr;
  return a.dtype == B200_BF16 ? launch_d<true>(ctx, stream, p, a.c.D, pl.nt) : launch_d<false>(ctx, stream, p, a.c.D, pl.nt);
}

}  // namespace tb
