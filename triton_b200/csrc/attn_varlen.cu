// Attention over packed prompts with grouped heads: tensor maps and launches of the packed form of the
// kernel in attn_fwd_kernel.cuh.
#include "attn_fwd_kernel.cuh"
#include "serving.h"

namespace tb {

namespace {

template <int D, bool BF16>
int launch_packed_t(DeviceCtx* ctx, cudaStream_t stream, const CUtensorMap& tq, const CUtensorMap& tk,
                    const CUtensorMap& tv, const CUtensorMap& to, const PackedFwdParams& p, long long most_items) {
  static std::atomic<bool> attr_done[64];
  constexpr size_t smem = FwdCfg<D>::SMEM + 64;  // + the published items
  if (int rc = ensure_dynamic_smem(attn_fwd_kernel<D, BF16, false, true>, smem, ctx->device, attr_done, "attn varlen")) return rc;
  const int grid = most_items < 1 ? 1 : (most_items < ctx->sm_count ? (int)most_items : ctx->sm_count);
  attn_fwd_kernel<D, BF16, false, true><<<grid, FWD_THREADS, smem, stream>>>(tq, tk, tv, to, p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(B200_ERR_CUDA, "attn varlen launch: %s", cudaGetErrorString(e));
  return B200_OK;
}

}  // namespace

int launch_attn_varlen(DeviceCtx* ctx, cudaStream_t stream, const AttnVarlenArgs& a) {
  CUtensorMap tq, tk, tv, to;
  if (!encode_qkv_map(&tq, a.dtype, a.q, 1, a.Hq, a.T, a.D, 0, a.sq[1], a.sq[0], BLK)) return B200_ERR_UNSUPPORTED;
  if (!encode_qkv_map(&tk, a.dtype, a.k, 1, a.Hkv, a.T, a.D, 0, a.sk[1], a.sk[0], BLK)) return B200_ERR_UNSUPPORTED;
  if (!encode_qkv_map(&tv, a.dtype, a.v, 1, a.Hkv, a.T, a.D, 0, a.sv[1], a.sv[0], BLK)) return B200_ERR_UNSUPPORTED;
  if (!encode_qkv_map(&to, a.dtype, a.o, 1, a.Hq, a.T, a.D, 0, a.so[1], a.so[0], 32)) return B200_ERR_UNSUPPORTED;
  PackedFwdParams p{};
  p.o_tma = 1;
  p.o = a.o;
  p.m = a.m;
  p.o_sh = a.so[1];
  p.o_sn = a.so[0];
  p.Z = 1;
  p.H = a.Hq;
  p.N = a.T;
  p.causal = a.causal;
  p.scale_log2 = a.sm_scale * 1.44269504f;
  p.cu = a.cu;
  p.batch = a.batch;
  p.group = a.Hq / a.Hkv;
  // By level evens out the end of a causal launch (2 to 8 % over by length: 16 x 2048 rows at 16/1 heads 291 against
  // 308 us, 2000 rows at 32/8 heads 39 against 52), but comes back to every K and V once per level: with a k/v
  // head per query head and more K and V than L2 keeps that costs more (4 x 4096 at 32/32 heads 569 against
  // 528 us), unless the sequences have few levels (64 x 512 at 32/32: 273 against 295).  Not causal, every block
  // of a sequence costs the same and only the reuse counts (4 x 4096 at 32/32: 1063 against 882 us).
  p.by_level = a.causal && (a.Hq > a.Hkv || (long long)a.T * a.Hkv * a.D * 4 <= (128 << 20) || (long long)a.T <= 1024LL * a.batch);
  // Two heads of a group on the same 128 rows waste no tile on short sequences (200 x 100 rows at 32/8 heads 115
  // against 212 us, 64 x 512 222 against 239, 12 of 5 to 2300 rows 100 against 105); 256 rows of one head are as
  // good or better on long ones (4 x 1024 at 48/8 heads of 64: 73 against 67 us) and spread few items over more SMs
  // (300 rows at 32/8: 22.3 against 19.5 us).
  p.pair = a.D != 256 && (a.Hq / a.Hkv) % 2 == 0 && (long long)a.T <= 640LL * a.batch &&
           ((long long)a.T / BLK + a.batch) * (a.Hq / 2) >= ctx->sm_count;
  p.zero_rest = a.zero_rest;
  p.status = ctx->status;
  p.sched_counter = next_sched_counter(ctx, stream);
  if (!p.sched_counter) return B200_ERR_CUDA;
  const int item_rows = (a.D == 256 || p.pair) ? BLK : 2 * BLK;
  const long long most_items = ((long long)a.T / item_rows + a.batch) * (p.pair ? a.Hq / 2 : a.Hq);  // the lengths are on the device
  const bool bf16 = a.dtype == B200_BF16;
  if (a.D == 256) return bf16 ? launch_packed_t<256, true>(ctx, stream, tq, tk, tv, to, p, most_items) : launch_packed_t<256, false>(ctx, stream, tq, tk, tv, to, p, most_items);
  if (a.D == 128) return bf16 ? launch_packed_t<128, true>(ctx, stream, tq, tk, tv, to, p, most_items) : launch_packed_t<128, false>(ctx, stream, tq, tk, tv, to, p, most_items);
  return bf16 ? launch_packed_t<64, true>(ctx, stream, tq, tk, tv, to, p, most_items) : launch_packed_t<64, false>(ctx, stream, tq, tk, tv, to, p, most_items);
}

}  // namespace tb
