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

// a [T, H, D] tensor as {d, head, row}, boxes of 64 columns (128 bytes, swizzled) x heads x rows
bool encode_heads_map(CUtensorMap* out, int dtype, const void* base, int T, int H, int D, const long long* stride, int heads,
                      int rows) {
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)H, (uint64_t)T, 1};
  const uint64_t eb = (uint64_t)dtype_bytes(dtype);
  const uint64_t strides[3] = {(uint64_t)stride[1] * eb, (uint64_t)stride[0] * eb, 0};
  const uint32_t box[4] = {64, (uint32_t)heads, (uint32_t)rows, 1};
  return encode_tmap(out, dtype, 4, base, dims, strides, box, 1);
}

}  // namespace

int launch_attn_varlen(DeviceCtx* ctx, cudaStream_t stream, const AttnVarlenArgs& a) {
  const int group = a.Hq / a.Hkv;
  // All heads of a group in a tile's rows leave no tile half empty on short sequences: 131 x 52 rows at 48/16 heads of 64
  // 69 against 171 us, 79 x 139 at 32/2 55 against 103, 200 x 100 at 32/8 heads of 128 114 against 205, 64 x 512 222
  // against 237, 20 x 1000 206 against 221.  Where they do not divide a warp's 32 rows (no boxes for o, tiles that
  // straddle K blocks) they pay on the shortest only: 64 x 512 rows at 24/8 heads of 64 190 against 150 us.  On long
  // sequences one head's rows are as good or better (4 x 4096 at 32/8 of 128 equal, 8 x 4096 1008 against 986).
  const int fold = (group <= 32 && (long long)a.T <= (32 % group == 0 ? 1024LL : 192LL) * a.batch) ? group : 1;
  const int tile_pos = BLK / fold;
  CUtensorMap tq, tk, tv, to;
  if (!encode_heads_map(&tq, a.dtype, a.q, a.T, a.Hq, a.D, a.sq, fold, tile_pos)) return B200_ERR_UNSUPPORTED;
  if (!encode_qkv_map(&tk, a.dtype, a.k, 1, a.Hkv, a.T, a.D, 0, a.sk[1], a.sk[0], BLK)) return B200_ERR_UNSUPPORTED;
  if (!encode_qkv_map(&tv, a.dtype, a.v, 1, a.Hkv, a.T, a.D, 0, a.sv[1], a.sv[0], BLK)) return B200_ERR_UNSUPPORTED;
  // o in boxes of a warp's 32 rows, where those are whole positions and where there is enough of o to make up for the
  // map's encoding here (0.6 us of 7.1 for 37 rows; without boxes 4 x 4096 rows at 32/8 heads take 498 us, not 487)
  const bool boxes = 32 % fold == 0 && (long long)a.T * a.Hq * a.D * 2 >= (1 << 20);
  if (boxes) {
    if (!encode_heads_map(&to, a.dtype, a.o, a.T, a.Hq, a.D, a.so, fold, 32 / fold)) return B200_ERR_UNSUPPORTED;
  } else {
    if ((reinterpret_cast<uintptr_t>(a.o) & 15) || (a.T > 1 && (a.so[0] & 7)) || (a.Hq > 1 && (a.so[1] & 7)))
      return fail(B200_ERR_UNSUPPORTED, "o must be 16-byte aligned, its strides multiples of 16 bytes");
    to = tq;
  }
  PackedFwdParams p{};
  p.o_tma = boxes ? 1 : 0;
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
  p.group = group;
  p.fold = fold;
  p.tile_pos = tile_pos;
  p.item_pos = (a.D == 256 ? 1 : 2) * tile_pos;
  p.item_shift = (p.item_pos & (p.item_pos - 1)) == 0 ? __builtin_ctz((unsigned)p.item_pos) : -1;
  p.block_items = a.Hq / fold;
  p.kv_items = group / fold;
  // By level evens out the end of a causal launch (2 to 8 % over by length: 16 x 2048 rows at 16/1 heads 291 against
  // 308 us, 2000 rows at 32/8 heads 39 against 52), but comes back to every K and V once per level: with a k/v
  // head per query head and more K and V than L2 keeps that costs more (4 x 4096 at 32/32 heads 569 against
  // 528 us), unless the sequences have few levels (64 x 512 at 32/32: 273 against 295).  Not causal, every block
  // of a sequence costs the same and only the reuse counts (4 x 4096 at 32/32: 1063 against 882 us).
  p.by_level = a.causal && (a.Hq > a.Hkv || (long long)a.T * a.Hkv * a.D * 4 <= (128 << 20) || (long long)a.T <= 1024LL * a.batch);
  p.lane_most = ((1 << 26) - 1) / p.block_items;
  p.rest = a.rest;
  p.status = ctx->status;
  bool used_up = false;
  p.sched_counter = next_sched_counter(ctx, stream, &used_up);
  if (!p.sched_counter && !used_up) return B200_ERR_CUDA;
  const long long most_items = ((long long)a.T / p.item_pos + a.batch) * p.block_items;  // the lengths are on the device
  const bool bf16 = a.dtype == B200_BF16;
  if (a.D == 256) return bf16 ? launch_packed_t<256, true>(ctx, stream, tq, tk, tv, to, p, most_items) : launch_packed_t<256, false>(ctx, stream, tq, tk, tv, to, p, most_items);
  if (a.D == 128) return bf16 ? launch_packed_t<128, true>(ctx, stream, tq, tk, tv, to, p, most_items) : launch_packed_t<128, false>(ctx, stream, tq, tk, tv, to, p, most_items);
  return bf16 ? launch_packed_t<64, true>(ctx, stream, tq, tk, tv, to, p, most_items) : launch_packed_t<64, false>(ctx, stream, tq, tk, tv, to, p, most_items);
}

}  // namespace tb
