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
// Bound by memory (read 2 bytes, write 1 per value) for prompts and by latency for single tokens.
#include <cstring>

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
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi) {
  if constexpr (BF16) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xFFFF0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = f.x;
    hi = f.y;
  }
}
__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }
__device__ __forceinline__ float finite_abs(float x) { return finite(x) ? fabsf(x) : 0.f; }
__device__ __forceinline__ uint32_t pack4_e4m3(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
template <bool BF16>
__device__ __forceinline__ float amax8(const uint4& x) {
  float m = 0.f;
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    unpack2<BF16>(w[i], a, b);
    m = fmaxf(m, fmaxf(finite_abs(a), finite_abs(b)));
  }
  return m;
}
// eight 16-bit values times `inv` (a power of two) as eight e4m3 bytes
template <bool BF16>
__device__ __forceinline__ uint2 quantize8(const uint4& x, float inv) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unpack2<BF16>(w[i], f[2 * i], f[2 * i + 1]);
    f[2 * i] = finite(f[2 * i]) ? f[2 * i] * inv : __uint_as_float(0x7FC00000u);
    f[2 * i + 1] = finite(f[2 * i + 1]) ? f[2 * i + 1] * inv : __uint_as_float(0x7FC00000u);
  }
  return make_uint2(pack4_e4m3(f[0], f[1], f[2], f[3]), pack4_e4m3(f[4], f[5], f[6], f[7]));
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

  float m = amax8<BF16>(x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  int e = exponent_for(m);
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
  if (mine) reinterpret_cast<uint2*>(rows + slot * D)[lane] = quantize8<BF16>(x, pow2f(-e));
  if (lane == 0) *scale = pow2f(e);
}

constexpr int PAGE_THREADS = 256;

// Prompts: a CTA per (page that gets rows, head, side).  The pages of the batch are numbered without a
// scan: a sequence with n new rows touches at most n / P + 2 pages, so numbering sequence b's from
// cu[b] / P + 2 b leaves no two sequences the same number; the few numbers in between belong to no page.
// The page's new rows stay in registers between the pass that finds the maximum and the one that rounds.
template <bool BF16, int ITEMS>
__global__ void __launch_bounds__(PAGE_THREADS) kv_append_page_kernel(const KvAppendArgs a) {
  __shared__ int s_seq;
  __shared__ float s_max[PAGE_THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31;
  const int unit = blockIdx.x, h = blockIdx.y, side = blockIdx.z;
  const int D = a.c.D, P = a.c.page_size;
  if (tid == 0) s_seq = -1;
  __syncthreads();
  auto offset = [&](int b) { return min(max(a.cu[b], 0), a.T); };
  for (int b = tid; b < a.batch; b += PAGE_THREADS) {
    if (offset(b) / P + 2 * b <= unit && (b + 1 == a.batch || unit < offset(b + 1) / P + 2 * (b + 1))) s_seq = b;
  }
  __syncthreads();
  const int b = s_seq;
  if (b < 0) return;
  const int t0 = offset(b), n = offset(b + 1) - t0;
  const int len = a.lens[b], start = len - n;
  if (n <= 0 || start < 0) return;
  const int p = start / P + (unit - (t0 / P + 2 * b));
  if (p >= a.c.max_pages || (long long)p * P >= len) return;
  const int page = a.c.table[b * a.c.table_stride + p];
  if (page < 0 || page >= a.c.pages) return;  // names no page: its rows are not written
  const int lo = max(start - p * P, 0), hi = min(len - p * P, P);
  const long long t = t0 + (p * P + lo - start);
  const long long st = side ? a.v_st : a.k_st;
  const uint16_t* src = (side ? reinterpret_cast<const uint16_t*>(a.v) + h * a.v_sh
                              : reinterpret_cast<const uint16_t*>(a.k) + h * a.k_sh) + t * st;
  const long long ph = (long long)page * a.c.Hkv + h;
  float* scale = (side ? a.c.v_scale : a.c.k_scale) + ph;
  uint8_t* rows = (side ? a.c.v : a.c.k) + ph * P * D;
  const int per_row = D / 8, items = (hi - lo) * per_row;  // 16 bytes each; per_row is a power of two

  uint4 x[ITEMS];
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int w = i * PAGE_THREADS + tid;
    x[i] = make_uint4(0, 0, 0, 0);
    if (w < items) x[i] = __ldg(reinterpret_cast<const uint4*>(src + (w / per_row) * st) + w % per_row);
  }
  const float held = *scale;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) m = fmaxf(m, amax8<BF16>(x[i]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) s_max[tid >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PAGE_THREADS / 32; ++i) m = fmaxf(m, s_max[i]);
  int e = exponent_for(m);
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
  const float inv = pow2f(-e);
  uint2* dst = reinterpret_cast<uint2*>(rows + lo * D);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int w = i * PAGE_THREADS + tid;
    if (w < items) dst[w] = quantize8<BF16>(x[i], inv);
  }
  if (tid == 0) *scale = pow2f(e);  // every thread has read it: the barrier above follows the loads
}

template <bool BF16>
int launch_t(cudaStream_t stream, const KvAppendArgs& a) {
  if (!a.cu) {
    const long long units = (long long)a.batch * a.c.Hkv * 2;
    const int per = TOKEN_THREADS / 32;
    kv_append_token_kernel<BF16><<<(unsigned)((units + per - 1) / per), TOKEN_THREADS, 0, stream>>>(a);
  } else {
    const dim3 grid((unsigned)(a.T / a.c.page_size + 2 * a.batch), (unsigned)a.c.Hkv, 2);
    const int items = a.c.page_size * a.c.D / 8 / PAGE_THREADS;
    if (items <= 1) kv_append_page_kernel<BF16, 1><<<grid, PAGE_THREADS, 0, stream>>>(a);
    else if (items <= 2) kv_append_page_kernel<BF16, 2><<<grid, PAGE_THREADS, 0, stream>>>(a);
    else if (items <= 4) kv_append_page_kernel<BF16, 4><<<grid, PAGE_THREADS, 0, stream>>>(a);
    else if (items <= 8) kv_append_page_kernel<BF16, 8><<<grid, PAGE_THREADS, 0, stream>>>(a);
    else kv_append_page_kernel<BF16, 16><<<grid, PAGE_THREADS, 0, stream>>>(a);  // page 128 at head dim 256
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
