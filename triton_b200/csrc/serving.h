// Internal header of the serving kernels (packed prompts, paged 8-bit cache, single tokens): what the
// C ABI (capi.cu) hands to the launchers.  Everything has been checked there.
#pragma once
#include "host.h"

namespace tb {

// A paged cache of e4m3 values, k and v alike: [pages][Hkv][page_size][D] bytes and one fp32 scale (a
// power of two) per (page, head), [pages][Hkv]; the pages of sequence b in order are
// table[b * table_stride + 0 .. max_pages).
struct PagedCache {
  uint8_t *k, *v;
  float *k_scale, *v_scale;
  const int* table;
  long long table_stride;
  int pages, page_size, max_pages;
  int Hkv, D;
};

// New rows k, v [T, Hkv, D] (element strides of the token and head dimensions) into the cache; cu: the
// batch's offsets into T, or nullptr when every sequence has one row (T == batch).
struct KvAppendArgs {
  PagedCache c;
  const void *k, *v;
  long long k_st, k_sh, v_st, v_sh;
  const int *lens, *cu;
  int batch, T;
  int dtype;
};
int launch_kv_append(DeviceCtx* ctx, cudaStream_t stream, const KvAppendArgs& a);

// One query row per sequence and head, q and o [B, Hq, D] (element strides of the first two dimensions).
struct AttnDecodeArgs {
  PagedCache c;
  const void* q;
  void* o;
  float* m;  // optional [B, Hq]: base-2 log-sum-exp
  long long q_sb, q_sh, o_sb, o_sh;
  const int* lens;
  int B, Hq;
  float sm_scale;
  int dtype;
  float* workspace;
};
size_t attn_decode_workspace_bytes(int B, int Hq, int Hkv, int D, int page_size, int max_pages);
int launch_attn_decode(DeviceCtx* ctx, cudaStream_t stream, const AttnDecodeArgs& a);

// Packed prompts: q, o [T, Hq, D], k, v [T, Hkv, D] (element strides {t, h}), m optional [Hq, T].
struct AttnVarlenArgs {
  const void *q, *k, *v;
  void* o;
  float* m;
  const int* cu;
  int batch, T, Hq, Hkv, D;
  long long sq[2], sk[2], sv[2], so[2];
  float sm_scale;
  int causal, dtype;
  int rest;  // see PackedFwdParams
};
int launch_attn_varlen(DeviceCtx* ctx, cudaStream_t stream, const AttnVarlenArgs& a);

}  // namespace tb
