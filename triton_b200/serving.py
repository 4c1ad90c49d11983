"""Serving: attention over packed prompts, a paged 8-bit key/value cache, single tokens over it.

  attention_varlen(q, k, v, cu_seqlens, causal, sm_scale)       prompts of different lengths, grouped heads
  kv_cache_append(k_cache, v_cache, k_scale, v_scale, k, v, ...)  their keys and values into the cache
  attention_decode(q, k_cache, v_cache, k_scale, v_scale, ...)    the next token of every sequence
  PagedKVCache                                                    the cache's four tensors with both calls

The reference's attention takes dense batches of one length and one head count
(python/tutorials/06-fused-attention.py:441-475); these three are what a program that answers needs beside
it.  They are for inference: inputs that require a gradient are refused while autograd records.

All lengths, offsets and page tables are int32 CUDA tensors that the kernels read: no call synchronises, and
every call can be captured into a CUDA graph (whose replays see the tensors' current values).
"""
import torch

from . import _lib
from .ops import _DT, _on_device, _require_cuda, _stream

_HEAD_DIMS = (64, 128, 256)
_PAGE_SIZES = (16, 32, 64, 128)


def _no_grad(what, *ts):
    if torch.is_grad_enabled() and any(t.requires_grad for t in ts):
        raise RuntimeError(f"{what} has no backward: call it under torch.no_grad(), or attention() for training")


def _check_ints(name, t, shape):
    assert t.dtype == torch.int32 and tuple(t.shape) == shape, f"{name} must be an int32 tensor of shape {shape}"
    assert t.is_contiguous(), f"{name} must be contiguous"


def attention_varlen(q, k, v, cu_seqlens, causal, sm_scale, *, out=None, return_stats=False):
    """Attention of whole prompts packed behind one another, with grouped heads.

    q [T, Hq, D], k and v [T, Hkv, D], fp16 or bf16, Hq a multiple of Hkv; sequence b is the rows
    cu_seqlens[b] : cu_seqlens[b + 1] (int32, on the GPU) and attends to itself, causally or in both
    directions.  Head dims 16 .. 256 as in attention().  Any strides with a contiguous head dimension and the
    others multiples of 8 (slices of one fused projection, say).  Returns O [T, Hq, D], with
    return_stats=True (O, M): M [Hq, T] is the base-2 log-sum-exp of attention_forward.
    Rows of T that belong to no sequence (padding behind the last one) come back as zeros (-inf in M); with
    `out=` they stay as they were.
    """
    assert q.dim() == 3 and k.dim() == 3 and v.shape == k.shape, "q [T, Hq, D], k and v [T, Hkv, D]"
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    assert k.shape[0] == T and k.shape[2] == D, "q, k and v must have the same rows and head dim"
    assert Hkv > 0 and Hq % Hkv == 0, "the query heads must be a multiple of the k/v heads"
    assert D in (16, 32) + _HEAD_DIMS, f"unsupported head dim {D}"
    assert q.dtype in (torch.float16, torch.bfloat16) and k.dtype == q.dtype and v.dtype == q.dtype, "fp16 or bf16, one type"
    assert cu_seqlens.dim() == 1 and cu_seqlens.numel() >= 1, "cu_seqlens holds one offset more than there are sequences"
    _check_ints("cu_seqlens", cu_seqlens, (cu_seqlens.numel(),))
    _no_grad("attention_varlen", q, k, v)
    dev = _require_cuda(q, k, v, cu_seqlens)
    if out is not None:
        assert out.shape == q.shape and out.dtype == q.dtype and out.device == dev, "out= must look like q"
    if D in (16, 32):  # as in attention_forward: zero-padded to the kernels' head dim 64
        wide = lambda t: torch.nn.functional.pad(t, (0, 64 - D))
        res = attention_varlen(wide(q), wide(k), wide(v), cu_seqlens, causal, sm_scale,
                               out=None if out is None else wide(out), return_stats=True)
        o = res[0][..., :D].contiguous() if out is None else out.copy_(res[0][..., :D])
        return (o, res[1]) if return_stats else o
    with _on_device(dev):
        o = torch.empty((T, Hq, D), device=dev, dtype=q.dtype) if out is None else out
        M = torch.empty((Hq, T), device=dev, dtype=torch.float32) if return_stats else None
        code = _lib.lib().b200_attention_varlen_fwd(
            _stream(q), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), M.data_ptr() if return_stats else None,
            cu_seqlens.data_ptr(), cu_seqlens.numel() - 1, T, Hq, Hkv, D, _lib.strides3(q), _lib.strides3(k),
            _lib.strides3(v), _lib.strides3(o), float(sm_scale), 1 if causal else 0, _DT[q.dtype], 1 if out is None else 0)
        _lib.check(code, "attention_varlen")
    return (o, M) if return_stats else o


def _check_cache(k_cache, v_cache, k_scale, v_scale, page_table, seq_lens):
    """The cache's tensors belong together; returns (pages, Hkv, page size, head dim)."""
    assert k_cache.dim() == 4 and v_cache.shape == k_cache.shape, "caches are [pages, Hkv, page size, D]"
    assert k_cache.dtype == v_cache.dtype == torch.float8_e4m3fn, "caches hold float8_e4m3fn values"
    assert k_cache.is_contiguous() and v_cache.is_contiguous(), "caches must be contiguous"
    pages, heads, page, D = k_cache.shape
    assert page in _PAGE_SIZES, f"pages hold 16, 32, 64 or 128 tokens, not {page}"
    assert D in _HEAD_DIMS, f"a cache has head dim 64, 128 or 256, not {D}"
    for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
        assert s.dtype == torch.float32 and tuple(s.shape) == (pages, heads) and s.is_contiguous(), \
            f"{name} must be a contiguous fp32 tensor [pages, Hkv]"
    assert page_table.dim() == 2 and page_table.dtype == torch.int32 and (page_table.stride(1) == 1 or page_table.shape[1] <= 1), \
        "page_table must be an int32 tensor [batch, pages of the longest sequence] with contiguous rows"
    _check_ints("seq_lens", seq_lens, (page_table.shape[0],))
    return pages, heads, page, D


def kv_cache_append(k_cache, v_cache, k_scale, v_scale, k, v, page_table, seq_lens, cu_seqlens=None):
    """Writes new rows of k and v, [T, Hkv, D] in fp16 or bf16, into the paged cache, in place.

    k_cache, v_cache [pages, Hkv, page size, D] float8_e4m3fn, k_scale, v_scale [pages, Hkv] fp32; page_table
    [batch, n] int32 names the pages of each sequence in order (an entry outside the cache names none: its rows
    are dropped).  seq_lens [batch] int32 is each sequence's length with the new rows, which become its last
    tokens: cu_seqlens[b] : cu_seqlens[b + 1] of T (a prompt's k and v as attention_varlen takes them), or one
    row per sequence without cu_seqlens (T == batch).
    The scale of a page and head is a power of two, 2^e with the smallest e >= -126 that lets e4m3's 448 * 2^e
    reach every finite value; values are stored as x / scale rounded to nearest even, non-finite ones as NaN.
    When later rows need a larger scale the page's earlier rows are rounded to it.  The stored bytes depend on
    nothing else.  Two sequences of one call may not write to the same page.
    """
    pages, heads, page, D = _check_cache(k_cache, v_cache, k_scale, v_scale, page_table, seq_lens)
    batch = page_table.shape[0]
    assert k.dim() == 3 and tuple(k.shape[1:]) == (heads, D) and v.shape == k.shape, "k and v must be [T, Hkv, D] of the cache's heads"
    assert k.dtype in (torch.float16, torch.bfloat16) and v.dtype == k.dtype, "fp16 or bf16, one type"
    tensors = (k_cache, v_cache, k_scale, v_scale, k, v, page_table, seq_lens)
    if cu_seqlens is None:
        assert k.shape[0] == batch, "without cu_seqlens every sequence has one new row"
    else:
        _check_ints("cu_seqlens", cu_seqlens, (batch + 1,))
        tensors += (cu_seqlens,)
    _no_grad("kv_cache_append", k, v)
    dev = _require_cuda(*tensors)
    with _on_device(dev):
        code = _lib.lib().b200_kv_append(
            _stream(k), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, page,
            page_table.data_ptr(), page_table.stride(0), page_table.shape[1], seq_lens.data_ptr(), k.data_ptr(), v.data_ptr(),
            None if cu_seqlens is None else cu_seqlens.data_ptr(), batch, k.shape[0], heads, D, _lib.strides3(k),
            _lib.strides3(v), _DT[k.dtype])
        _lib.check(code, "kv_cache_append")


def attention_decode(q, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, sm_scale, *, out=None, return_stats=False):
    """Attention of one token per sequence over the paged cache: q [batch, Hq, D] in fp16 or bf16, Hq a multiple
    of the cache's heads, over the first seq_lens[b] tokens (the new one among them, once it is appended).  Tokens
    of a page that the table does not name are left out; a sequence without tokens gives zeros.  Returns O like
    q, with return_stats=True (O, M): M [batch, Hq] is the base-2 log-sum-exp (-inf without tokens)."""
    pages, heads, page, D = _check_cache(k_cache, v_cache, k_scale, v_scale, page_table, seq_lens)
    batch = page_table.shape[0]
    assert q.dim() == 3 and q.shape[0] == batch and q.shape[2] == D, "q must be [batch, Hq, D] of the cache's head dim"
    Hq = q.shape[1]
    assert heads > 0 and Hq % heads == 0, "the query heads must be a multiple of the cache's heads"
    assert q.dtype in (torch.float16, torch.bfloat16), "fp16 or bf16"
    _no_grad("attention_decode", q)
    dev = _require_cuda(q, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens)
    if out is not None:
        assert out.shape == q.shape and out.dtype == q.dtype and out.device == dev, "out= must look like q"
    with _on_device(dev):
        L = _lib.lib()
        o = torch.empty((batch, Hq, D), device=dev, dtype=q.dtype) if out is None else out
        M = torch.empty((batch, Hq), device=dev, dtype=torch.float32) if return_stats else None
        ws_bytes = L.b200_attention_decode_workspace(batch, Hq, heads, D, page, page_table.shape[1])
        ws = torch.empty(ws_bytes // 4, device=dev, dtype=torch.float32) if ws_bytes else None
        code = L.b200_attention_decode(
            _stream(q), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages,
            page, page_table.data_ptr(), page_table.stride(0), page_table.shape[1], seq_lens.data_ptr(), o.data_ptr(),
            M.data_ptr() if return_stats else None, batch, Hq, heads, D, _lib.strides3(q), _lib.strides3(o),
            float(sm_scale), _DT[q.dtype], None if ws is None else ws.data_ptr())
        _lib.check(code, "attention_decode")
    return (o, M) if return_stats else o


class PagedKVCache:
    """The four tensors of a cache (one layer's) and the calls on them.  `append` and `attend` take the page
    table and the lengths from the caller, who hands out the pages; fresh pages hold zeros with scale 1."""

    def __init__(self, pages, page_size, kv_heads, head_dim, device="cuda"):
        assert page_size in _PAGE_SIZES and head_dim in _HEAD_DIMS
        shape = (pages, kv_heads, page_size, head_dim)
        self.k = torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        self.v = torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        self.k_scale = torch.ones(shape[:2], dtype=torch.float32, device=device)
        self.v_scale = torch.ones(shape[:2], dtype=torch.float32, device=device)

    def append(self, k, v, page_table, seq_lens, cu_seqlens=None):
        kv_cache_append(self.k, self.v, self.k_scale, self.v_scale, k, v, page_table, seq_lens, cu_seqlens)

    def attend(self, q, page_table, seq_lens, sm_scale, *, out=None, return_stats=False):
        return attention_decode(q, self.k, self.v, self.k_scale, self.v_scale, page_table, seq_lens, sm_scale, out=out,
                                return_stats=return_stats)
