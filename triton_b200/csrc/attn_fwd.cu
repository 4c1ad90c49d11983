// Flash-attention forward for dense [Z, H, N, D] batches: tensor maps and launches of the kernel in
// attn_fwd_kernel.cuh.
#include "attn_fwd_kernel.cuh"

namespace tb {

namespace {

template <int D, bool BF16, bool FP8 = false>
int launch_fwd_t(DeviceCtx* ctx, cudaStream_t stream, const CUtensorMap& tq, const CUtensorMap& tk,
                 const CUtensorMap& tv, const CUtensorMap& to, const FwdParams& p) {
  static std::atomic<bool> attr_done[64];
  constexpr size_t smem = FwdCfg<D, FP8>::SMEM;
  if (int rc = ensure_dynamic_smem(attn_fwd_kernel<D, BF16, FP8>, smem, ctx->device, attr_done, "attn fwd")) return rc;
  const int grid = p.total_items < ctx->sm_count ? p.total_items : ctx->sm_count;
  attn_fwd_kernel<D, BF16, FP8><<<grid, FWD_THREADS, smem, stream>>>(tq, tk, tv, to, p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(B200_ERR_CUDA, "attn fwd launch: %s", cudaGetErrorString(e));
  return B200_OK;
}

}  // namespace

bool encode_rows_map(CUtensorMap* out, int dtype, const void* base, int Z, int H, int N, int D, int64_t sz, int64_t sh,
                     int64_t sn, int box_cols, int box_rows, int swizzle) {
  uint64_t dims[4] = {(uint64_t)D, (uint64_t)N, (uint64_t)H, (uint64_t)Z};
  const uint64_t eb = (uint64_t)dtype_bytes(dtype);
  uint64_t strides[3] = {(uint64_t)sn * eb, (uint64_t)sh * eb, (uint64_t)sz * eb};
  uint32_t box[4] = {(uint32_t)box_cols, (uint32_t)box_rows, 1, 1};
  return encode_tmap(out, dtype, 4, base, dims, strides, box, swizzle);
}

// the operand maps: boxes of 64 columns (128 bytes, swizzled) x box_rows rows
bool encode_qkv_map(CUtensorMap* out, int dtype, const void* base, int Z, int H, int N, int D, int64_t sz, int64_t sh,
                    int64_t sn, int box_rows) {
  return encode_rows_map(out, dtype, base, Z, H, N, D, sz, sh, sn, 64, box_rows, true);
}

int launch_attn_fwd(DeviceCtx* ctx, cudaStream_t stream, const void* q, const void* k, const void* v, void* o,
                    float* m, float* row_max, int Z, int H, int N, int D, const int64_t* sq, const int64_t* sk, const int64_t* sv,
                    const int64_t* so, float sm_scale, int causal, int dtype) {
  if (dtype == B200_E5M2) {
    // 8-bit forward: rows of 128 bytes; V is addressed as [D rows][N keys] (keys contiguous)
    if (D != 128 && D != 64) return fail(B200_ERR_UNSUPPORTED, "the 8-bit forward has kernels for head dims 64 and 128");
    const int sw = (D == 64) ? 2 : 1;  // rows of 64 bytes take the 64-byte swizzle
    if (sq[3] != 1 || sk[3] != 1 || so[3] != 1) return fail(B200_ERR_UNSUPPORTED, "8-bit q, k, o need a contiguous head dimension");
    if (sv[2] != 1 && N != 1) return fail(B200_ERR_UNSUPPORTED, "an 8-bit v needs its key dimension contiguous (stride_v[2] == 1)");
    CUtensorMap tq8, tk8, tv8, to8;
    if (!encode_rows_map(&tq8, dtype, q, Z, H, N, D, sq[0], sq[1], sq[2], D, BLK, sw)) return B200_ERR_UNSUPPORTED;
    if (!encode_rows_map(&tk8, dtype, k, Z, H, N, D, sk[0], sk[1], sk[2], D, BLK, sw)) return B200_ERR_UNSUPPORTED;
    // "rows" of the V map are head-dim indices, "columns" are keys: a block is D rows of 128 keys
    if (!encode_rows_map(&tv8, dtype, v, Z, H, D, N, sv[0], sv[1], sv[3], 128, D, 1)) return B200_ERR_UNSUPPORTED;
    FwdParams p8{};
    p8.o_tma = encode_rows_map(&to8, dtype, o, Z, H, N, D, so[0], so[1], so[2], D, 32, sw) ? 1 : 0;
    if (!p8.o_tma) to8 = tq8;
    p8.o = o; p8.m = m; p8.row_max = row_max;
    p8.o_sz = so[0]; p8.o_sh = so[1]; p8.o_sn = so[2];
    p8.Z = Z; p8.H = H; p8.N = N; p8.causal = causal;
    p8.scale_log2 = sm_scale * 1.44269504f;
    p8.num_qb = (N + 255) / 256;
    p8.total_items = p8.num_qb * Z * H;
    p8.status = ctx->status;
    p8.sched_counter = next_sched_counter(ctx, stream);
    if (!p8.sched_counter) return B200_ERR_CUDA;
    return D == 64 ? launch_fwd_t<64, false, true>(ctx, stream, tq8, tk8, tv8, to8, p8)
                   : launch_fwd_t<128, false, true>(ctx, stream, tq8, tk8, tv8, to8, p8);
  }
  CUtensorMap tq, tk, tv;
  if (!encode_qkv_map(&tq, dtype, q, Z, H, N, D, sq[0], sq[1], sq[2], BLK)) return B200_ERR_UNSUPPORTED;
  if (!encode_qkv_map(&tk, dtype, k, Z, H, N, D, sk[0], sk[1], sk[2], BLK)) return B200_ERR_UNSUPPORTED;
  if (!encode_qkv_map(&tv, dtype, v, Z, H, N, D, sv[0], sv[1], sv[2], BLK)) return B200_ERR_UNSUPPORTED;
  CUtensorMap to;
  FwdParams p{};
  // O through TMA stores (boxes of 32 rows x 64 columns) when its layout allows, else direct stores
  p.o_tma = encode_qkv_map(&to, dtype, o, Z, H, N, D, so[0], so[1], so[2], 32) ? 1 : 0;
  if (!p.o_tma) to = tq;
  p.o = o; p.m = m; p.row_max = row_max;
  p.o_sz = so[0]; p.o_sh = so[1]; p.o_sn = so[2];
  p.Z = Z; p.H = H; p.N = N; p.causal = causal;
  p.scale_log2 = sm_scale * 1.44269504f;  // the reference's constant (06-fused-attention.py:161)
  const int item_rows = (D == 256) ? BLK : 2 * BLK;  // one 128-row tile per work item at head dim 256, two otherwise
  p.num_qb = (N + item_rows - 1) / item_rows;
  p.total_items = p.num_qb * Z * H;
  p.status = ctx->status;
  p.sched_counter = next_sched_counter(ctx, stream);
  if (!p.sched_counter) return B200_ERR_CUDA;
  const bool bf16 = dtype == B200_BF16;
  if (D == 256) return bf16 ? launch_fwd_t<256, true>(ctx, stream, tq, tk, tv, to, p) : launch_fwd_t<256, false>(ctx, stream, tq, tk, tv, to, p);
  if (D == 128) return bf16 ? launch_fwd_t<128, true>(ctx, stream, tq, tk, tv, to, p) : launch_fwd_t<128, false>(ctx, stream, tq, tk, tv, to, p);
  if (D == 64) return bf16 ? launch_fwd_t<64, true>(ctx, stream, tq, tk, tv, to, p) : launch_fwd_t<64, false>(ctx, stream, tq, tk, tv, to, p);
  return fail(B200_ERR_UNSUPPORTED, "head dim %d: the forward has kernels for 64, 128 and 256", D);
}

}  // namespace tb
