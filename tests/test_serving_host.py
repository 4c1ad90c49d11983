"""Serving calls on a machine without a GPU: what they refuse, and how they trace."""
import ctypes

import pytest
import torch

import triton_b200 as tb
from triton_b200 import _lib

I32 = torch.int32


def _pack(T=10, Hq=4, Hkv=2, D=64, dtype=torch.float16, batch=2):
    q = torch.zeros(T, Hq, D, dtype=dtype)
    k = torch.zeros(T, Hkv, D, dtype=dtype)
    return q, k, k.clone(), torch.zeros(batch + 1, dtype=I32)


def _cache(pages=4, heads=2, page=16, D=64, batch=3, width=2):
    kc = torch.zeros(pages, heads, page, D, dtype=torch.uint8).view(torch.float8_e4m3fn)
    sc = torch.ones(pages, heads)
    return [kc, kc.clone(), sc, sc.clone()], torch.zeros(batch, width, dtype=I32), torch.ones(batch, dtype=I32)


def test_varlen_refusals():
    q, k, v, cu = _pack()
    call = lambda q=q, k=k, v=v, cu=cu, **kw: tb.attention_varlen(q, k, v, cu, True, 0.5, **kw)
    bad = [dict(q=q[0]), dict(k=k[:9], v=v[:9]), dict(v=v[:, :1]), dict(k=k[:, :, :32], v=v[:, :, :32]),
           dict(q=torch.zeros(10, 3, 64, dtype=torch.float16)),               # 3 query heads on 2 k/v heads
           dict(q=torch.zeros(10, 4, 48, dtype=torch.float16), k=k[..., :48], v=v[..., :48]),
           dict(q=q.float(), k=k.float(), v=v.float()), dict(q=q.bfloat16()),
           dict(cu=cu.long()), dict(cu=cu[:0]), dict(cu=torch.zeros(6, dtype=I32)[::2]), dict(cu=cu[None])]
    for kw in bad:
        with pytest.raises(AssertionError):
            call(**kw)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        call()
    with pytest.raises(RuntimeError, match="no backward"):
        call(q=q.clone().requires_grad_(True))


def test_append_refusals():
    c, table, lens = _cache()
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    cu = torch.zeros(4, dtype=I32)

    def call(c=c, k=k, v=k, table=table, lens=lens, cu=None):
        tb.kv_cache_append(*c, k, v, table, lens, cu)

    other = lambda i, t: [t if j == i else x for j, x in enumerate(c)]
    bad = [dict(c=other(1, c[1][:3])), dict(c=other(0, c[0].view(torch.uint8))), dict(c=other(2, c[2].half())),
           dict(c=other(3, c[3][:, :1])), dict(c=other(2, torch.ones(2, 4).t())), dict(c=_cache(page=24)[0]), dict(c=_cache(D=96)[0]),
           dict(c=[c[0].transpose(1, 2), c[1].transpose(1, 2), *c[2:]]), dict(k=k[:2], v=k[:2]), dict(k=k[:, :1], v=k[:, :1]),
           dict(k=k.float(), v=k.float()), dict(v=k.half()), dict(v=k[:2]), dict(table=table.long()), dict(table=table[0]),
           dict(table=torch.zeros(2, 3, dtype=I32).t()), dict(lens=lens[:2]), dict(lens=lens.long()), dict(cu=cu[:3]), dict(cu=cu.long())]
    for kw in bad:
        with pytest.raises(AssertionError):
            call(**kw)
    for kw in (dict(), dict(cu=cu, k=torch.zeros(7, 2, 64, dtype=torch.bfloat16), v=torch.zeros(7, 2, 64, dtype=torch.bfloat16))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call(**kw)


def test_decode_refusals():
    c, table, lens = _cache()
    q = torch.zeros(3, 6, 64, dtype=torch.float16)
    call = lambda q=q, table=table, lens=lens, **kw: tb.attention_decode(q, *c, table, lens, 0.5, **kw)
    for kw in (dict(q=q[:2]), dict(q=q[:, :5]), dict(q=q[..., :32]), dict(q=q.float()), dict(q=q[0]), dict(lens=lens[:1])):
        with pytest.raises(AssertionError):
            call(**kw)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        call()
    with pytest.raises(RuntimeError, match="no backward"):
        call(q=q.clone().requires_grad_(True))
    with pytest.raises(AssertionError):
        tb.PagedKVCache(4, 8, 2, 64, device="cpu")
    cache = tb.PagedKVCache(4, 16, 2, 64, device="cpu")
    assert cache.k.float().abs().sum() == 0 and cache.k_scale.min() == 1


S3 = ctypes.c_int64 * 3


def test_c_entry_points_check_their_arguments():
    """Arguments are checked before a device is looked for: 1 = bad argument, 2 = unsupported layout or size."""
    L = _lib.lib()
    ok = S3(128, 64, 1)

    def varlen(batch=1, T=8, Hq=2, Hkv=2, D=64, s=(ok,) * 4, scale=0.5, dtype=0):
        return L.b200_attention_varlen_fwd(None, 16, 16, 16, 16, None, 16, batch, T, Hq, Hkv, D, *s, scale, 1, dtype, 0)

    assert varlen(T=-1) == 1 and varlen(batch=-1) == 1 and varlen(Hq=3) == 1 and varlen(Hkv=0) == 1 and varlen(scale=0.0) == 1
    assert varlen(dtype=3) == 1 and varlen(scale=float("nan")) == 1 and varlen(D=48) == 2
    assert varlen(s=(ok, ok, S3(128, 64, 2), ok)) == 2 and varlen(T=2 ** 31 - 1, Hq=4096, Hkv=1) == 2

    def append(pages=4, page=16, width=2, batch=2, T=2, heads=2, D=64, s=(ok, ok), dtype=0, kc=16, k=16, cu=None):
        return L.b200_kv_append(None, kc, 16, 16, 16, pages, page, 16, width, width, 16, k, 16, cu, batch, T, heads, D, *s, dtype)

    assert append(batch=-1) == 1 and append(T=3) == 1 and append(dtype=2) == 1 and append(pages=-1) == 1 and append(heads=-2) == 1
    assert append(page=48) == 2 and append(D=32) == 2 and append(s=(S3(129, 64, 1), ok)) == 2 and append(s=(ok, S3(128, 64, 2))) == 2
    assert append(kc=24) == 2 and append(k=8) == 2 and append(width=2 ** 28) == 2 and append(pages=2 ** 31 - 1, heads=65535) == 2

    def decode(pages=4, page=16, width=2, batch=2, Hq=4, heads=2, D=64, s=(ok, ok), scale=0.5, dtype=0, q=16):
        return L.b200_attention_decode(None, q, 16, 16, 16, 16, pages, page, 16, width, width, 16, 16, None, batch, Hq, heads, D,
                                       *s, scale, dtype, None)

    assert decode(batch=-1) == 1 and decode(Hq=3) == 1 and decode(dtype=4) == 1 and decode(scale=-1.0) == 1 and decode(heads=0) == 1
    assert decode(page=17) == 2 and decode(D=100) == 2 and decode(q=4) == 2 and decode(s=(S3(4, 64, 1), ok)) == 2
    assert decode(batch=70000) == 2
    assert L.b200_attention_decode_workspace(0, 4, 2, 64, 16, 2) == 0
    # few heads and a long table: split over tokens, so there is something to join
    assert L.b200_attention_decode_workspace(1, 8, 2, 128, 64, 1024) >= 8 * 2 * 129 * 4
    if not torch.cuda.is_available():
        assert varlen() == 4 and append() == 4 and decode() == 4  # no device


def test_custom_ops_trace_on_meta_tensors():
    ns = torch.ops.triton_b200
    meta = lambda *s, dtype=torch.float16: torch.empty(*s, dtype=dtype, device="meta")
    q, k, cu = meta(10, 4, 64), meta(10, 2, 64), meta(3, dtype=I32)
    assert ns.attention_varlen(q, k, k, cu, True, 0.5).shape == q.shape
    c = [meta(4, 2, 16, 64, dtype=torch.float8_e4m3fn)] * 2 + [meta(4, 2, dtype=torch.float32)] * 2
    table, lens = meta(10, 2, dtype=I32), meta(10, dtype=I32)
    assert ns.kv_cache_append(*c, k, k, table, lens) is None
    o = ns.attention_decode(q, *c, table, lens, 0.5)
    assert o.shape == q.shape and o.dtype == q.dtype


def test_docstrings_end_where_their_sentences_do():
    for f in (tb.attention_varlen, tb.kv_cache_append, tb.attention_decode, tb.PagedKVCache):
        assert f.__doc__.rstrip().endswith("."), f.__name__


def test_dual_tensors_are_refused():
    """A dual tensor of forward-mode differentiation does not pass a call in silence, neither while autograd records nor
    under no_grad."""
    from torch.autograd import forward_ad
    q, k, v, cu = _pack()
    c, table, lens = _cache()
    q1 = torch.zeros(3, 4, 64, dtype=torch.float16)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        calls = [lambda: tb.attention_varlen(dual(q), k, v, cu, True, 0.5), lambda: tb.attention_varlen(q, k, dual(v), cu, True, 0.5),
                 lambda: tb.kv_cache_append(*c, dual(q1[:, :2]), q1[:, :2], table, lens), lambda: tb.attention_decode(dual(q1), *c, table, lens, 0.5)]
        for call in calls:
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode derivative"):  # which ends backward recording only
                call()


def test_a_cache_that_requires_a_gradient_is_refused():
    from torch.autograd import forward_ad
    c, table, lens = _cache()
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    for i in range(4):
        d = [x.clone().requires_grad_(True) if j == i else x for j, x in enumerate(c)]
        with pytest.raises(RuntimeError, match="no backward"):
            tb.attention_decode(q, *d, table, lens, 0.5)
        with pytest.raises(RuntimeError, match="no backward"):
            tb.kv_cache_append(*d, q[:, :2], q[:, :2], table, lens)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):
            tb.attention_decode(q, *d, table, lens, 0.5)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
        tb.attention_decode(q, *c[:3], forward_ad.make_dual(c[3], torch.ones_like(c[3])), table, lens, 0.5)


def test_binding_is_rebuilt_for_another_torch(tmp_path, monkeypatch):
    """The binding is linked against torch's libraries: built for another version of it, it is stale."""
    from triton_b200 import build
    made = []

    class Done:
        returncode, stdout, stderr = 0, "", ""

    def compiler(cmd, **kw):
        made.append(cmd)
        open(build.BINDING, "w").close()
        return Done

    monkeypatch.setattr(build, "BINDING", str(tmp_path / "_binding.so"))
    monkeypatch.setattr(build, "OBJ", str(tmp_path / "_obj"))
    monkeypatch.setattr(build.subprocess, "run", compiler)
    build.build_binding()
    build.build_binding()
    assert len(made) == 1
    monkeypatch.setattr(torch, "__version__", torch.__version__ + "+other")
    build.build_binding()
    build.build_binding()
    assert len(made) == 2
