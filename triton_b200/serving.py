"""Serving: attention over packed prompts, a paged 8-bit key/value cache, single tokens over it.

  attention_varlen(q, k, v, cu_seqlens, causal, sm_scale)       prompts of different lengths, grouped heads
  kv_cache_append(k_cache, v_cache, k_scale, v_scale, k, v, ...)  their keys and values into the cache
  attention_decode(q, k_cache, v_cache, k_scale, v_scale, ...)    the next token of every sequence
  PagedKVCache                                                    the cache's four tensors with both calls

The reference's attention takes dense batches of one length and one head count
(python/tutorials/06-fused-attention.py:441-475); these three are what a program that answers needs beside
it.  They are for inference: inputs that require a gradient are refused while autograd records, dual tensors of
forward-mode differentiation always.

All lengths, offsets and page tables are int32 CUDA tensors that the kernels read: no call synchronises, and
every call can be captured into a CUDA graph (whose replays see the tensors' current values).
"""
import torch

from . import _lib

_HEAD_DIMS = (64, 128, 256)
_PAGE_SIZES = (16, 32, 64, 128)


def attention_varlen(q, k, v, cu_seqlens, causal, sm_scale, *, out=None, return_stats=False):
    """Attention of whole prompts packed behind one another, with grouped heads.

    q [T, Hq, D], k and v [T, Hkv, D], fp16 or bf16, Hq a multiple of Hkv; sequence b is the rows
    cu_seqlens[b] : cu_seqlens[b + 1] (int32, on the GPU) and attends to itself, causally or in both
    directions.  Head dims 16 .. 256 as in attention().  Any strides with a contiguous head dimension and the
    others multiples of 8 (slices of one fused projection, say).  Returns O [T, Hq, D], with
    return_stats=True (O, M): M [Hq, T] is the base-2 log-sum-exp of attention_forward.
    Rows of T that belong to no sequence (padding behind the last one) come back as zeros, with `out=` they stay
    as they were; in M they are -inf.  `out` may be q, but not share memory with k or v.

    Scores, their maximum and all sums are fp32.  The weights are rounded to the inputs' type before they meet V
    (at head dims 128 and 256 a quarter of them come from a cubic for 2^x, within 8.6e-5), the output once more.
    Sequences keep to themselves whatever their values; within one, a V that is not finite may also reach rows
    before its own, whose weight for it is 0 (0 * inf).
    """
    if q.dim() == 3 and q.shape[2] in (16, 32):  # as in attention_forward: zero-padded to the kernels' head dim 64
        D = q.shape[2]
        assert k.shape[-1] == v.shape[-1] == D, "q, k and v must have the same head dim"
        wide = lambda t: torch.nn.functional.pad(t, (0, 64 - D))
        res = attention_varlen(wide(q), wide(k), wide(v), cu_seqlens, causal, sm_scale,
                               out=None if out is None else wide(out), return_stats=True)
        o = res[0][..., :D].contiguous() if out is None else out.copy_(res[0][..., :D])
        return (o, res[1]) if return_stats else o
    return (_lib._binding or _lib.binding()).attention_varlen(q, k, v, cu_seqlens, causal, sm_scale, out, return_stats)


def kv_cache_append(k_cache, v_cache, k_scale, v_scale, k, v, page_table, seq_lens, cu_seqlens=None):
    """Writes new rows of k and v, [T, Hkv, D] in fp16 or bf16, into the paged cache, in place.

    k_cache, v_cache [pages, Hkv, page size, D] float8_e4m3fn, k_scale, v_scale [pages, Hkv] fp32; page_table
    [batch, n] int32 names the pages of each sequence in order (an entry outside the cache names none: its rows
    are dropped).  seq_lens [batch] int32 is each sequence's length with the new rows, which become its last
    tokens: cu_seqlens[b] : cu_seqlens[b + 1] of T (a prompt's k and v as attention_varlen takes them), or one
    row per sequence without cu_seqlens (T == batch).
    The scale of a page and head is a power of two, 2^e with the smallest e >= -126 that lets e4m3's 448 * 2^e
    reach every finite value; values are stored as x / scale rounded to nearest even, non-finite ones as NaN.
    """
    (_lib._binding or _lib.binding()).kv_cache_append(k_cache, v_cache, k_scale, v_scale, k, v, page_table, seq_lens, cu_seqlens)


def attention_decode(q, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, sm_scale, *, out=None, return_stats=False):
    """Attention of one token per sequence over the paged cache: q [batch, Hq, D] in fp16 or bf16, Hq a multiple
    of the cache's heads, over the first seq_lens[b] tokens (the new one among them, once it is appended).  Tokens
    of a page that the table does not name are left out; a sequence without tokens gives zeros.  Returns O like
    q, with return_stats=True (O, M): M [batch, Hq] is the base-2 log-sum-exp (-inf without tokens).
    The scales have to be powers of two, as kv_cache_append leaves them: only their exponents are read.  Scores,
    their maximum and all sums are fp32; the weights are rounded to fp16 before they meet V, and a bf16 row of q is
    taken as fp16 times a power of two (what lies 2^-29 below the row's largest value loses bits).
    The lengths stay on the GPU, so the launch covers what the table has room for: where that is far more than
    the longest sequence, pass its first columns (page_table[:, :n])."""
    return (_lib._binding or _lib.binding()).attention_decode(q, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, sm_scale,
                                                              out, return_stats)


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
