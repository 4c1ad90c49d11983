// Writing new rows of k and v into the paged 8-bit cache.
//
// A page and head share one scale 2^e per side (k or v): e is the smallest integer >= -126 with
//   max over the page's rows of |x| <= 448 * 2^e        (finite x only; 448 is e4m3's largest value)
// and a row is stored as e4m3(x * 2^-e), round to nearest even.  With powers of two every product by a
// scale is exact in fp32, so the stored bytes do not depend on how the work is split, and an e4m3 value
// keeps its relative precision under any of them (a finer scale would gain no bits).  A page that holds
// rows already keeps max(e_old, e_new); when that grew, the held rows are rounded to the new scale: exact
// but for values that fall below e4m3's normal range.  Values that are not finite become NaN: e4m3 has no
// infinity, and saturating would hide it.
//
// Bound by memory (read 2 bytes, write 1 per value) for prompts: 21325 rows of 8 heads x 128 in 27.4 us = 4.8 TB/s (with
// a CTA per page, head and side and the maxima in fp32 43.7 us).  Single tokens are bound by latency: 2.1 us for one,
// 2.8 for 200.
#include <algorithm>

#include "common.cuh"
#include "serving.h"

namespace tb {

namespace {

__device__ __forceinline__ float pow2f(int e) {  // 2^e; 0 below the normal range (e > 127 does not occur)
  return e < -126 ? 0.f : __uint_as_float((uint32_t)(e + 127) << 23);
}
// smallest e >= -126 with amax <= 448 * 2^e; 448 = 1.75 * 2^8 (a subnormal amax lands on the bound)
__device__ __forceinline__ int exponent_for(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return max(e, -126);
}
__device__ __forceinline__ int scale_exponent(float s) { return max((int)((__float_as_uint(s) >> 23) & 0xFFu) - 127, -126); }

template <bool BF16>
__device__ __forceinline__ float to_f32(uint32_t bits16) {
  if constexpr (BF16) return __uint_as_float(bits16 << 16);
  else return __half2float(__ushort_as_half((unsigned short)bits16));
}
template <bool BF16> constexpr uint32_t INF16 = BF16 ? 0x7F80u : 0x7C00u;  // bits of infinity; NaN's are above

// The largest of eight values' magnitudes as bits: magnitudes order like their bits, two at a time.  At INF16 or
// above some value is not finite and finite_amax_bits has to look again.
__device__ __forceinline__ uint32_t amax_bits(const uint4& x) {
  constexpr uint32_t M = 0x7FFF7FFFu;
  return __vmaxu2(__vmaxu2(x.x & M, x.y & M), __vmaxu2(x.z & M, x.w & M));
}
__device__ __forceinline__ uint32_t higher_half(uint32_t two) { return max(two & 0xFFFFu, two >> 16); }
template <bool BF16>
__device__ __noinline__ uint32_t finite_amax_bits(uint4 x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t m = 0;
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = (w[i >> 1] >> (16 * (i & 1))) & 0x7FFFu;
    if (a < INF16<BF16>) m = max(m, a);
  }
  return m;
}
__device__ __forceinline__ uint32_t pack4_e4m3(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
// eight 16-bit values times 2^-e as eight e4m3 bytes
template <bool BF16>
__device__ __noinline__ uint2 quantize8_slow(uint4 x, int e) {  // any values, any e
  const float inv = pow2f(-e);
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  float f[8];
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = (w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu;
    f[i] = (b & 0x7FFFu) < INF16<BF16> ? to_f32<BF16>(b) * inv : __uint_as_float(0x7FC00000u);
  }
  return make_uint2(pack4_e4m3(f[0], f[1], f[2], f[3]), pack4_e4m3(f[4], f[5], f[6], f[7]));
}
__device__ __forceinline__ uint32_t e4m3x2_of_f16x2(uint32_t x) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(x));
  return r;
}
// Finite values, and for fp16 -15 <= -e <= 14, so that 2^-e is an fp16 number: the product is exact down to
// fp16's normal range, and what lies below that is below half of e4m3's smallest step.
template <bool BF16>
__device__ __forceinline__ uint2 quantize8(const uint4& x, int e) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  if constexpr (BF16) {
    const float inv = pow2f(-e);
    const uint64_t inv2 = pk2(inv, inv);
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      upk2(mul2(pk2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u)), inv2), f[2 * i], f[2 * i + 1]);
    return make_uint2(pack4_e4m3(f[0], f[1], f[2], f[3]), pack4_e4m3(f[4], f[5], f[6], f[7]));
  } else {
    const __half2 inv = __float2half2_rn(pow2f(-e));
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&w[i]), inv);
      r[i] = e4m3x2_of_f16x2(*reinterpret_cast<const uint32_t*>(&y));
    }
    return make_uint2(r[0] | (r[1] << 16), r[2] | (r[3] << 16));
  }
}
template <bool BF16>
__device__ __forceinline__ bool quantizes_fast(uint32_t bits, int e) {
  return bits < INF16<BF16> && (BF16 || (e >= -14 && e <= 15));
}
__device__ __forceinline__ uint32_t requantize4(uint32_t w, float factor) {
  const __half2 lo(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xFFFFu), __NV_E4M3));
  const __half2 hi(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3));
  const float2 a = __half22float2(lo), b = __half22float2(hi);
  return pack4_e4m3(a.x * factor, a.y * factor, b.x * factor, b.y * factor);
}
__device__ __forceinline__ uint4 requantize16(uint4 w, float factor) {
  return make_uint4(requantize4(w.x, factor), requantize4(w.y, factor), requantize4(w.z, factor), requantize4(w.w, factor));
}

constexpr int TOKEN_THREADS = 128;

// One row per sequence: a warp per (sequence, head, side).
template <bool BF16>
__global__ void __launch_bounds__(TOKEN_THREADS) kv_append_token_kernel(const KvAppendArgs a) {
  const int lane = threadIdx.x & 31;
  const int unit = blockIdx.x * (TOKEN_THREADS / 32) + (threadIdx.x >> 5);
  if (unit >= a.batch * a.c.Hkv * 2) return;
  const int side = unit & 1, h = (unit >> 1) % a.c.Hkv, b = (unit >> 1) / a.c.Hkv;
  const int D = a.c.D, P = a.c.page_size;
  const uint16_t* src = side ? reinterpret_cast<const uint16_t*>(a.v) + b * a.v_st + h * a.v_sh
                             : reinterpret_cast<const uint16_t*>(a.k) + b * a.k_st + h * a.k_sh;
  const bool mine = lane * 8 < D;
  uint4 x = make_uint4(0, 0, 0, 0);
  if (mine) x = __ldg(reinterpret_cast<const uint4*>(src) + lane);
  const int pos = a.lens[b] - 1;
  if (pos < 0 || pos >= a.c.max_pages * P) return;
  const int page = a.c.table[b * a.c.table_stride + pos / P], slot = pos % P;
  if (page < 0 || page >= a.c.pages) return;  // names no page: nothing is written
  const long long ph = (long long)page * a.c.Hkv + h;
  float* scale = (side ? a.c.v_scale : a.c.k_scale) + ph;
  uint8_t* rows = (side ? a.c.v : a.c.k) + ph * P * D;
  const float held = *scale;

  const uint32_t bits = __reduce_max_sync(0xffffffffu, higher_half(amax_bits(x)));
  uint32_t top = bits;
  if (bits >= INF16<BF16>) top = __reduce_max_sync(0xffffffffu, finite_amax_bits<BF16>(x));
  int e = exponent_for(to_f32<BF16>(top));
  if (slot > 0) {
    const int before = scale_exponent(held);
    if (e > before) {
      const float factor = pow2f(before - e);
      uint4* old = reinterpret_cast<uint4*>(rows);
      for (int i = lane; i < slot * D / 16; i += 32) old[i] = requantize16(old[i], factor);
    } else {
      e = before;
    }
  }
  if (mine)
    reinterpret_cast<uint2*>(rows + slot * D)[lane] = quantizes_fast<BF16>(bits, e) ? quantize8<BF16>(x, e) : quantize8_slow<BF16>(x, e);
  if (lane == 0) *scale = pow2f(e);
}

constexpr int PAGE_THREADS = 256;

// Prompts: a CTA per page that gets rows, over some of its (head, side) pairs; the loads of the next pair are under
// way while the current one, held in registers between the pass that finds the maximum and the one that rounds,
// is worked on.  The pages of the batch are numbered without a scan: a sequence with n new rows touches at most
// n / P + 2 pages, so numbering sequence b's from cu[b] / P + 2 b leaves no two sequences the same number; the few
// numbers in between belong to no page.
template <bool BF16, int ITEMS>
__global__ void __launch_bounds__(PAGE_THREADS) kv_append_page_kernel(const KvAppendArgs a, int pairs) {
  constexpr bool AHEAD = ITEMS <= 8;  // (16 items twice would not fit the registers)
  __shared__ int s_seq, s_t0, s_n, s_len;
  __shared__ uint32_t s_max[2][PAGE_THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31;
  const int unit = blockIdx.x, D = a.c.D, P = a.c.page_size;
  if (tid == 0) s_seq = -1;
  __syncthreads();
  int found = -1, f_t0 = 0, f_n = 0, f_len = 0;
  for (int b = tid; b < a.batch; b += PAGE_THREADS) {
    const int t0 = min(max(__ldg(a.cu + b), 0), a.T), t1 = min(max(__ldg(a.cu + b + 1), 0), a.T), len = __ldg(a.lens + b);
    if (t0 / P + 2 * b <= unit && (b + 1 == a.batch || unit < t1 / P + 2 * (b + 1))) {
      found = b; f_t0 = t0; f_n = t1 - t0; f_len = len;
      atomicMax(&s_seq, b);
    }
  }
  __syncthreads();
  if (found >= 0 && found == s_seq) { s_t0 = f_t0; s_n = f_n; s_len = f_len; }  // (decreasing offsets can match twice)
  __syncthreads();
  const int b = s_seq, t0 = s_t0, n = s_n, len = s_len, start = len - n;
  if (b < 0 || n <= 0 || start < 0) return;
  const int p = start / P + (unit - (t0 / P + 2 * b));
  if (p >= a.c.max_pages || (long long)p * P >= len) return;
  const int page = __ldg(a.c.table + b * a.c.table_stride + p);
  if (page < 0 || page >= a.c.pages) return;  // names no page: its rows are not written
  const int lo = max(start - p * P, 0), hi = min(len - p * P, P);
  const long long t = t0 + (p * P + lo - start);
  const int shift = 31 - __clz(D / 8), items = (hi - lo) << shift;  // of 16 bytes, D / 8 (a power of two) a row
  const int row = tid >> shift, col = (tid & (D / 8 - 1)) * 8;      // of this thread's first
  const int first = blockIdx.y * pairs, last = min(first + pairs, 2 * a.c.Hkv);

  auto load = [&](uint4 (&x)[ITEMS], float& held, int pair) {
    const int side = pair & 1, h = pair >> 1;
    const long long st = side ? a.v_st : a.k_st;
    const uint16_t* src = (side ? reinterpret_cast<const uint16_t*>(a.v) + h * a.v_sh
                                : reinterpret_cast<const uint16_t*>(a.k) + h * a.k_sh) + (t + row) * st + col;
    const long long step = (PAGE_THREADS >> shift) * st;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      x[i] = make_uint4(0, 0, 0, 0);
      if (i * PAGE_THREADS + tid < items) x[i] = __ldg(reinterpret_cast<const uint4*>(src + i * step));
    }
    held = (side ? a.c.v_scale : a.c.k_scale)[(long long)page * a.c.Hkv + h];
  };
  uint4 x[ITEMS];
  float held;
  load(x, held, first);
  for (int pair = first; pair < last; ++pair) {
    uint4 y[AHEAD ? ITEMS : 1];
    float held_y = 0.f;
    if constexpr (AHEAD)
      if (pair + 1 < last) load(y, held_y, pair + 1);
    uint32_t two = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) two = __vmaxu2(two, amax_bits(x[i]));
    // the maximum over the CTA; a second time, without what is not finite, when that is what it found
    uint32_t bits = higher_half(two), top;
    auto over_cta = [&](uint32_t v, int buf) {
      v = __reduce_max_sync(0xffffffffu, v);
      if (lane == 0) s_max[buf][tid >> 5] = v;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < PAGE_THREADS / 32; ++i) v = max(v, s_max[buf][i]);
      return v;
    };
    bits = top = over_cta(bits, pair & 1);
    if (bits >= INF16<BF16>) {
      top = 0;
      for (int i = 0; i < ITEMS; ++i) top = max(top, finite_amax_bits<BF16>(x[i]));
      __syncthreads();
      top = over_cta(top, pair & 1);
    }
    const int side = pair & 1;
    const long long ph = (long long)page * a.c.Hkv + (pair >> 1);
    uint8_t* rows = (side ? a.c.v : a.c.k) + ph * P * D;
    int e = exponent_for(to_f32<BF16>(top));
    if (lo > 0) {
      const int before = scale_exponent(held);
      if (e > before) {
        const float factor = pow2f(before - e);
        uint4* old = reinterpret_cast<uint4*>(rows);
        for (int i = tid; i < lo * D / 16; i += PAGE_THREADS) old[i] = requantize16(old[i], factor);
      } else {
        e = before;
      }
    }
    uint2* dst = reinterpret_cast<uint2*>(rows + lo * D);
    const bool fast = quantizes_fast<BF16>(bits, e);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int w = i * PAGE_THREADS + tid;
      if (w < items) dst[w] = fast ? quantize8<BF16>(x[i], e) : quantize8_slow<BF16>(x[i], e);
    }
    if (tid == 0) (side ? a.c.v_scale : a.c.k_scale)[ph] = pow2f(e);  // (every thread had read it before the barrier above)
    if (pair + 1 < last) {
      if constexpr (AHEAD) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) x[i] = y[i];
        held = held_y;
      } else {
        load(x, held, pair + 1);
      }
    }
  }
}

template <bool BF16>
int launch_t(cudaStream_t stream, const KvAppendArgs& a) {
  if (!a.cu) {
    const long long units = (long long)a.batch * a.c.Hkv * 2;
    const int per = TOKEN_THREADS / 32;
    kv_append_token_kernel<BF16><<<(unsigned)((units + per - 1) / per), TOKEN_THREADS, 0, stream>>>(a);
  } else {
    // pairs of head and side per CTA: enough CTAs for the GPU first, then loads ahead of the work
    const long long units = (long long)a.T / a.c.page_size + 2 * a.batch, all = 2LL * a.c.Hkv;
    const int pairs = (int)std::max(1LL, std::min({8LL, all, units * all / (148 * 6)}));
    const dim3 grid((unsigned)units, (unsigned)((all + pairs - 1) / pairs));
    const int items = a.c.page_size * a.c.D / 8 / PAGE_THREADS;
    if (items <= 1) kv_append_page_kernel<BF16, 1><<<grid, PAGE_THREADS, 0, stream>>>(a, pairs);
    else if (items <= 2) kv_append_page_kernel<BF16, 2><<<grid, PAGE_THREADS, 0, stream>>>(a, pairs);
    else if (items <= 4) kv_append_page_kernel<BF16, 4><<<grid, PAGE_THREADS, 0, stream>>>(a, pairs);
    else if (items <= 8) kv_append_page_kernel<BF16, 8><<<grid, PAGE_THREADS, 0, stream>>>(a, pairs);
    else kv_append_page_kernel<BF16, 16><<<grid, PAGE_THREADS, 0, stream>>>(a, pairs);  // page 128 at head dim 256
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(B200_ERR_CUDA, "kv append launch: %s", cudaGetErrorString(e));
  return B200_OK;
}

}  // namespace

int launch_kv_append(DeviceCtx*, cudaStream_t stream, const KvAppendArgs& a) {
  return a.dtype == B200_BF16 ? launch_t<true>(stream, a) : launch_t<false>(stream, a);
}

}  // namespace tb
