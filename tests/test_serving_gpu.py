"""Serving on the GPU against plain implementations in 64 bits: packed prompts, the paged 8-bit cache, single
tokens, and the three together.

Bounds (all sums below in 64 bits; eps the type's distance from 1 to the next value):
  * the output is rounded once: half a step, eps / 2 of its value;
  * the weights p are rounded to 16 bits before the second product: at most eps_p / 2 of each, i.e. eps_p / 2 times
    sum p |v| (eps_p: the type's in the packed attention, fp16's for single tokens);
  * a score is a sum of D exact products in fp32, |error| <= D 2^-23 sum |q k| (2^-23: the adder may cut); with the
    scaling and the rounding of score - maximum it moves a weight by a relative error of at most
    ds = ln-units (D + 4) 2^-23 scale max_j sum |q k_j| + |score| 2^-23, and so does the sum they are divided by;
  * 2^x: 8.6e-5 where the cubic is used, 2^-21 otherwise; both in the weight and in the sum; together below 2^-12.
"""
import math

import pytest
import torch

import triton_b200 as tb
from triton_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = torch.int32
ints = lambda *x: torch.tensor(x, dtype=I32, device=DEV)


@pytest.fixture(autouse=True)
def _status():
    yield
    torch.cuda.synchronize()
    assert _lib.status() == 0, "a bounded device-side wait ran out"


def one_head(q, k, v, scale, causal):
    """(o, lse in log2 units, sum p |v|, ds) of q [n, D] over k, v [m, D], all in 64 bits; rows see the first
    m - n + 1 + i keys when causal."""
    q, k, v = q.double(), k.double(), v.double()
    s = q @ k.T * scale
    if causal:
        s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(1 + k.shape[0] - q.shape[0]), -math.inf)
    p = torch.softmax(s, 1)
    size = (q.abs() @ k.abs().T).amax(1, keepdim=True) * scale
    ds = (q.shape[1] + 4) * 2.0 ** -23 * size + size * 2.0 ** -23
    return p @ v, torch.logsumexp(s, 1) / math.log(2), p @ v.abs(), ds


def check(got, want, dtype, p_dtype, what):
    o, lse, pv, ds = want
    tol = torch.finfo(dtype).eps / 2 * o.abs() + (torch.finfo(p_dtype).eps / 2 + 2.0 ** -12 + 2 * ds) * pv + 2.0 ** -24
    err = (got.double() - o).abs()
    assert bool((err <= tol).all()), f"{what}: worst {float((err / tol).max())} of the bound"


def check_lse(got, want, what):
    _, lse, _, ds = want
    tol = (2.0 ** -12 + ds[:, 0]) / math.log(2) + lse.abs() * 2.0 ** -22
    assert bool(((got.double() - lse).abs() <= tol).all()), what


# ------------------------------------------------------------------ packed prompts
def pack(lens, hq, hkv, D, dtype, seed, tail=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    T = sum(lens) + tail
    mk = lambda h: torch.randn(T, h, D, generator=g, device=DEV).to(dtype)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return mk(hq), mk(hkv), mk(hkv), torch.tensor(cu, dtype=I32, device=DEV), cu


def check_pack(o, M, q, k, v, cu, causal, scale, what=""):
    group = q.shape[1] // k.shape[1]
    for b in range(len(cu) - 1):
        a, e = cu[b], cu[b + 1]
        if a == e:
            continue
        for h in range(q.shape[1]):
            want = one_head(q[a:e, h], k[a:e, h // group], v[a:e, h // group], scale, causal)
            check(o[a:e, h], want, q.dtype, q.dtype, f"{what} sequence {b} ({e - a} rows) head {h}")
            if M is not None:
                check_lse(M[h, a:e], want, f"{what} lse of sequence {b} head {h}")


LENS = [[1], [37], [128], [129], [256, 256], [1, 2, 3, 127, 128, 129, 255, 256, 257], [700, 0, 5, 0], [0, 1025, 31]]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,D", [(4, 2, 64), (3, 1, 128), (2, 2, 256), (6, 2, 32), (1, 1, 16)])
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_varlen(lens, hq, hkv, D, dtype, causal):
    q, k, v, cu, off = pack(lens, hq, hkv, D, dtype, seed=len(lens) + D)
    scale = 1.3 * D ** -0.5
    o, M = tb.attention_varlen(q, k, v, cu, causal, scale, return_stats=True)
    assert o.shape == q.shape and o.dtype == dtype and M.shape == (hq, q.shape[0])
    check_pack(o, M, q, k, v, off, causal, scale)
    assert torch.equal(tb.attention_varlen(q, k, v, cu, causal, scale), o)  # repeatable, and the same without M


def test_varlen_equals_dense_attention_on_equal_lengths():
    Z, H, N, D = 3, 4, 640, 64
    q, k, v, cu, _ = pack([N] * Z, H, H, D, torch.bfloat16, seed=9)
    dense = lambda t: t.view(Z, N, H, D).transpose(1, 2).contiguous()
    o, M = tb.attention_forward(dense(q), dense(k), dense(v), True, 0.125)
    o2, M2 = tb.attention_varlen(q, k, v, cu, True, 0.125, return_stats=True)
    assert torch.equal(dense(o2), o) and torch.equal(M2.view(H, Z, N).transpose(0, 1), M)


def test_varlen_many_sequences():
    lens = [(7 * i) % 23 for i in range(1500)] + [900] + [3] * 40
    q, k, v, cu, off = pack(lens, 2, 1, 64, torch.float16, seed=3)
    o = tb.attention_varlen(q, k, v, cu, True, 0.125)
    some = [0, 3, 10, 700, 1499, 1500, 1501, 1540]
    for b in some:
        a, e = off[b], off[b + 1]
        for h in range(2 if e > a else 0):
            check(o[a:e, h], one_head(q[a:e, h], k[a:e, 0], v[a:e, 0], 0.125, True), q.dtype, q.dtype, f"sequence {b}")
    # every other sequence against the same rows of a pack of its own
    for b in range(0, 1541, 37):
        a, e = off[b], off[b + 1]
        if a < e:
            alone = tb.attention_varlen(q[a:e], k[a:e], v[a:e], ints(0, e - a), True, 0.125)
            assert torch.equal(o[a:e], alone)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan, 65504.0])
def test_varlen_neighbours_do_not_leak(D, what):
    """Everything around a sequence - the next one, the one before, the padding - holds infinities or NaN."""
    lens = [100, 201, 77]
    q, k, v, cu, off = pack(lens, 4, 2, D, torch.float16, seed=5, tail=60)
    want = tb.attention_varlen(q, k, v, cu, True, 0.1)
    a, e = off[1], off[2]
    for t in (q, k, v):
        t[:a] = what
        t[e:] = what
    for causal in (True, False):
        o, M = tb.attention_varlen(q, k, v, cu, causal, 0.1, return_stats=True)
        assert torch.isfinite(o[a:e]).all() and torch.isfinite(M[:, a:e]).all()
        if causal:
            assert torch.equal(o[a:e], want[a:e])
        check_pack(o[a:e], None, q[a:e], k[a:e], v[a:e], [0, e - a], causal, 0.1)


def test_varlen_nan_stays_in_its_rows():
    q, k, v, cu, off = pack([300, 200], 2, 1, 64, torch.bfloat16, seed=6)
    q[310, 1] = math.nan  # one row of one head
    o = tb.attention_varlen(q, k, v, cu, True, 0.125)
    bad = torch.isnan(o).all(-1)
    assert bool(bad[310, 1]) and int(bad.sum()) == 1 and int(torch.isnan(o).sum()) == 64
    k[400] = math.nan  # seen by rows 400.. of the second sequence only
    o = tb.attention_varlen(q, k, v, cu, True, 0.125)
    assert torch.isnan(o[400:]).all() and torch.isfinite(o[:310]).all() and torch.isfinite(o[311:400]).all()


@pytest.mark.parametrize("D", [64, 128, 32])
def test_varlen_rows_outside_the_sequences(D):
    q, k, v, cu, off = pack([130, 9], 2, 2, D, torch.float16, seed=7, tail=150)
    o, M = tb.attention_varlen(q, k, v, cu, True, 0.2, return_stats=True)
    assert (o[139:] == 0).all() and (M[:, 139:] == -math.inf).all()
    mine = torch.full_like(q, 7.0)
    got = tb.attention_varlen(q, k, v, cu, True, 0.2, out=mine)
    assert got is mine and torch.equal(mine[:139], o[:139]) and (mine[139:] == 7.0).all()
    shifted = cu + 20  # rows before the first sequence as well
    o = tb.attention_varlen(q, k, v, shifted, True, 0.2)
    assert (o[:20] == 0).all() and (o[159:] == 0).all()
    check_pack(o, None, q, k, v, [x + 20 for x in off], True, 0.2)


def test_varlen_empty_and_odd_offsets():
    q, k, v, _, _ = pack([50], 2, 1, 64, torch.float16, seed=8)
    assert (tb.attention_varlen(q, k, v, ints(0), True, 0.2) == 0).all()          # no sequence
    assert (tb.attention_varlen(q, k, v, ints(0, 0, 0), True, 0.2) == 0).all()    # empty ones
    assert tb.attention_varlen(q[:0], k[:0], v[:0], ints(0, 0), True, 0.2).shape == (0, 2, 64)
    # offsets outside the tensors are cut, so nothing is read or written beside them
    a = tb.attention_varlen(q, k, v, ints(-5, 2000), True, 0.2)
    assert torch.equal(a, tb.attention_varlen(q, k, v, ints(0, 50), True, 0.2))
    a = tb.attention_varlen(q, k, v, ints(30, 10, 20), True, 0.2)  # a decreasing pair is an empty sequence
    check_pack(a[10:20], None, q[10:20], k[10:20], v[10:20], [0, 10], True, 0.2)


def test_varlen_slices_of_a_fused_projection():
    lens, hq, hkv, D = [60, 333], 6, 2, 128
    g = torch.Generator(device=DEV).manual_seed(10)
    qkv = torch.randn(393, (hq + 2 * hkv) * D + 8, generator=g, device=DEV).bfloat16()
    rows = qkv[:, :(hq + 2 * hkv) * D].unflatten(1, (hq + 2 * hkv, D))
    q, k, v = rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:]
    out = torch.zeros(393, 2 * hq, D, dtype=torch.bfloat16, device=DEV)[:, ::2]
    o = tb.attention_varlen(q, k, v, ints(0, 60, 393), True, 0.09, out=out)
    assert torch.equal(o, tb.attention_varlen(q.contiguous(), k.contiguous(), v.contiguous(), ints(0, 60, 393), True, 0.09))
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(o, tb.attention_varlen(heads_first, k, v, ints(0, 60, 393), True, 0.09))
    with pytest.raises(RuntimeError, match="multiple of 16 bytes|aligned"):
        tb.attention_varlen(torch.zeros(10, 2, 65, dtype=torch.bfloat16, device=DEV)[..., :64], k[:10, :, :64], v[:10, :, :64],
                            ints(0, 10), True, 0.1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_varlen_peaked_scores(dtype):
    """Scores that grow along the keys, far past the first block's: the running reference has to move."""
    q, k, v, cu, off = pack([900, 500], 2, 1, 128, dtype, seed=11)
    k *= (1 + torch.arange(1400, device=DEV) / 100.0)[:, None, None].to(dtype)
    o = tb.attention_varlen(q, k, v, cu, True, 0.3)
    check_pack(o, None, q, k, v, off, True, 0.3)


# ------------------------------------------------------------------ the cache
def new_cache(pages, heads, page, D, fill=None):
    c = tb.PagedKVCache(pages, page, heads, D)
    if fill is not None:
        c.k.view(torch.uint8).fill_(fill)
        c.v.view(torch.uint8).fill_(fill)
    return c


def reference_append(cache, scale, x, table, lens, new):
    """The definition, page by page, on the CPU in 64 bits; cache uint8, scale and x on the CPU, in place."""
    page, at = cache.shape[2], 0
    e4m3 = lambda t: t.float().to(torch.float8_e4m3fn)  # exact in fp32: values times powers of two
    val = cache.view(torch.float8_e4m3fn)
    for b, n in enumerate(new):
        start = lens[b] - n
        for pos0 in range(start - start % page, lens[b], page):
            if pos0 + page <= start:
                continue
            col = pos0 // page
            p = table[b][col] if col < len(table[b]) else -1
            lo, hi = max(start, pos0) - pos0, min(lens[b] - pos0, page)
            if not 0 <= p < cache.shape[0]:
                continue
            rows = x[at + pos0 + lo - start: at + pos0 + hi - start].double()  # [n, H, D]
            for h in range(cache.shape[1]):
                r = rows[:, h]
                ok = torch.isfinite(r)
                most = float(r[ok].abs().max()) if bool(ok.any()) else 0.0
                e = -126
                if most > 0:
                    e = max(-126, math.frexp(most / 448.0)[1] - 1)
                    while most > 448.0 * 2.0 ** e:
                        e += 1
                    while e > -126 and most <= 448.0 * 2.0 ** (e - 1):
                        e -= 1
                if lo > 0:
                    held = int(math.log2(float(scale[p, h])))
                    if e > held:
                        val[p, h, :lo] = e4m3(val[p, h, :lo].double() * 2.0 ** (held - e))
                    e = max(e, held)
                q = e4m3(r * 2.0 ** -e)
                q.view(torch.uint8)[~ok] = 0x7F
                val[p, h, lo:hi] = q
                scale[p, h] = 2.0 ** e
        at += n


def same_bytes(got, want):
    """Equal values: NaN is NaN whatever its sign."""
    g, w = got.view(torch.uint8).cpu(), want.view(torch.uint8).cpu()
    return bool(((g == w) | (((g & 0x7F) == 0x7F) & ((w & 0x7F) == 0x7F))).all())


def run_append(c, k, v, table, lens, new, single=False):
    t = torch.tensor(table, dtype=I32, device=DEV)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    ref = [x.cpu().clone() for x in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale)]
    c.append(k, v, t, torch.tensor(lens, dtype=I32, device=DEV), None if single else torch.tensor(cu, dtype=I32, device=DEV))
    reference_append(ref[0], ref[2], k.cpu(), table, lens, new)
    reference_append(ref[1], ref[3], v.cpu(), table, lens, new)
    assert torch.equal(c.k_scale.cpu(), ref[2]) and torch.equal(c.v_scale.cpu(), ref[3])
    assert same_bytes(c.k, ref[0]) and same_bytes(c.v, ref[1])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_append(page, D, dtype):
    """Prompts, a second turn behind them in the same pages, then single tokens, some of them louder than what
    their page has seen."""
    g = torch.Generator(device=DEV).manual_seed(page + D)
    heads, first = 3, [1, page - 1, page, page + 1, 0, 3 * page + 5]
    width = 6
    order = torch.randperm(40, generator=torch.Generator().manual_seed(1)).tolist()
    table = [order[i * width:(i + 1) * width] for i in range(6)]
    c = new_cache(40, heads, page, D, fill=0x7F)  # stale NaN everywhere
    mk = lambda n, loud=1.0: (torch.randn(n, heads, D, generator=g, device=DEV) * loud).to(dtype)
    run_append(c, mk(sum(first)), mk(sum(first)), table, first, first)
    second = [2, 1, page, 0, 5, page + 3]
    lens = [a + b for a, b in zip(first, second)]
    loud = torch.tensor([0.1, 50.0, 1.0, 9.0, 2.0, 300.0], device=DEV).repeat_interleave(torch.tensor(second, device=DEV))[:, None, None]
    run_append(c, mk(sum(second), loud), mk(sum(second), 1 / loud), table, lens, second)
    for step in range(3):
        lens = [n + 1 for n in lens]
        run_append(c, mk(6, 5.0 ** step), mk(6, 7.0 ** -step), table, lens, [1] * 6, single=True)


@pytest.mark.parametrize("single", [True, False])
def test_append_values_at_the_borders(single):
    """Largest values on and beside 448 * 2^e, subnormals, zeros, infinities, NaN."""
    for dtype in (torch.float16, torch.bfloat16):
        big = torch.finfo(dtype).max
        tiny = torch.finfo(dtype).smallest_normal
        vals = [448.0, 449.0, 450.0, 447.0, 224.0, 225.0, 1.75, 1.7509766, 0.875, 0.0, -0.0, big, -big, tiny, tiny / 16, 3e-5, math.inf,
                -math.inf, math.nan, 1.0]
        n = len(vals)
        k = torch.zeros(n, 1, 64, dtype=dtype, device=DEV)
        k[:, 0, 5] = torch.tensor(vals, device=DEV).to(dtype)
        k[:, 0, 9] = (torch.tensor(vals, device=DEV) / 3).to(dtype)
        v = torch.randn(n, 1, 64, device=DEV).to(dtype)
        v[3] = math.nan  # a row without one finite value
        v[4] = 0.0
        c = new_cache(n, 1, 16, 64)
        run_append(c, k, v, [[i] for i in range(n)], [1] * n, [1] * n, single=single)
        run_append(c, v, k, [[i] for i in range(n)], [2] * n, [1] * n, single=single)


def test_append_drops_what_no_page_holds():
    """Table entries outside the cache, lengths past the table, lengths that cannot be: nothing is written there
    and everything else is as it should be."""
    heads, page, D = 2, 16, 64
    mk = lambda n: torch.randn(n, heads, D, device=DEV).half()
    for single in (True, False):
        c = new_cache(6, heads, page, D, fill=0x11)
        table = [[0, -1], [6, 1], [2, 2 ** 31 - 1], [-2 ** 31, 3], [4, 5]]
        lens = [17, 5, 18, 20, 40]  # the last is past its two pages
        new = [1] * 5 if single else [17, 5, 18, 4, 9]
        run_append(c, mk(sum(new)), mk(sum(new)), table, lens, new, single=single)
    # a length below the number of new rows (no start) or zero: the sequence is left out
    c = new_cache(3, heads, page, D, fill=0x22)
    t = torch.tensor([[0], [1], [2]], dtype=I32, device=DEV)
    before = c.k.view(torch.uint8).clone()
    c.append(mk(9), mk(9), t, ints(2, 0, -7), ints(0, 3, 6, 9))
    c.append(mk(3), mk(3), t, ints(0, -1, 17))
    c.append(mk(9), mk(9), t, ints(3, 3, 3), ints(9, 6, 3, 0))      # offsets that decrease
    assert torch.equal(c.k.view(torch.uint8), before) and (c.k_scale == 1).all()
    c.append(mk(9)[:0], mk(9)[:0], t, ints(3, 3, 3), ints(0, 0, 0, 0))
    assert torch.equal(c.k.view(torch.uint8), before)


def test_append_many_sequences_and_strides():
    heads, page, D, batch = 2, 16, 64, 700
    new = [(5 * i) % 41 for i in range(batch)]
    held = [(11 * i) % 19 for i in range(batch)]
    lens = [a + b for a, b in zip(new, held)]
    need = [-(-n // page) for n in lens]
    at, table = 0, []
    for n in need:
        table.append(list(range(at, at + n)) + [-1] * (4 - n))
        at += n
    c = new_cache(at, heads, page, D)
    first = torch.randn(sum(held), heads, D, device=DEV).bfloat16()
    run_append(c, first, first * 2, table, held, held)
    qkv = torch.randn(sum(new), 4 * heads, D, device=DEV).bfloat16()
    run_append(c, qkv[:, heads:2 * heads], qkv[:, 2 * heads:3 * heads], table, lens, new)


# ------------------------------------------------------------------ single tokens
def filled_cache(lens, heads, page, D, seed, spread=2, stale=0x7F, pages=None):
    """A cache of random values with scales 2^(-6 +- spread); bytes behind the last token are NaN."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = pages or sum(need) + 2
    c = new_cache(pages, heads, page, D, fill=stale)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), max(need + [1])), -1, dtype=I32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        ids = order[at:at + n]
        at += n
        table[b, :n] = torch.tensor(ids, dtype=I32, device=DEV)
        for i, p in enumerate(ids):
            rows = min(page, lens[b] - i * page)
            for x, s in ((c.k, c.k_scale), (c.v, c.v_scale)):
                e = torch.randint(-6 - spread, -5 + spread, (heads,), generator=g, device=DEV)
                s[p] = torch.exp2(e.float())
                x[p, :, :rows] = (torch.randn(heads, rows, D, generator=g, device=DEV) * 64).clamp(-448, 448).to(torch.float8_e4m3fn)
    return c, table


def check_decode(o, M, q, c, table, lens, scale, what=""):
    page, heads, D = c.k.shape[2], c.k.shape[1], c.k.shape[3]
    group = q.shape[1] // heads
    for b, n in enumerate(lens):
        keep = [i for i in range(n) if i // page < table.shape[1] and 0 <= int(table[b, i // page]) < c.k.shape[0]] if n < 300 else list(range(n))
        if not keep:
            assert (o[b] == 0).all() and (M[b] == -math.inf).all(), f"{what} sequence {b} has no token"
            continue
        i = torch.tensor(keep, device=DEV)
        ids = table[b].long()[i // page]
        for h in range(heads):
            k = c.k[ids].double()[torch.arange(len(keep), device=DEV), h, i % page] * c.k_scale[ids, h].double()[:, None]
            v = c.v[ids].double()[torch.arange(len(keep), device=DEV), h, i % page] * c.v_scale[ids, h].double()[:, None]
            want = one_head(q[b, h * group:(h + 1) * group], k, v, scale, False)
            check(o[b, h * group:(h + 1) * group], want, q.dtype, torch.float16, f"{what} sequence {b} ({n} tokens) head {h}")
            check_lse(M[b, h * group:(h + 1) * group], want, f"{what} lse of sequence {b}")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("group,heads,D,page", [(1, 2, 64, 16), (4, 2, 128, 64), (8, 1, 128, 16), (9, 1, 64, 32), (16, 2, 128, 128),
                                                (7, 1, 256, 32), (20, 1, 256, 16), (35, 1, 64, 64)])
def test_decode(group, heads, D, page, dtype):
    lens = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 250, 700, 1033]
    c, table = filled_cache(lens, heads, page, D, seed=group + D)
    q = torch.randn(len(lens), group * heads, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(group)).to(dtype)
    n = torch.tensor(lens, dtype=I32, device=DEV)
    scale = 1.2 * D ** -0.5
    o, M = c.attend(q, table, n, scale, return_stats=True)
    check_decode(o, M, q, c, table, lens, scale)
    assert torch.equal(c.attend(q, table, n, scale), o)
    mine = torch.full((len(lens), 2 * group * heads, D), 3.0, dtype=dtype, device=DEV)
    qs = torch.stack([q, q], 2).flatten(1, 2)[:, ::2]  # strided heads in and out
    got = c.attend(qs, table, n, scale, out=mine[:, ::2])
    assert torch.equal(got, o) and (mine[:, 1::2] == 3.0).all()


def test_decode_one_long_sequence():
    lens = [40007]
    c, table = filled_cache(lens, 2, 64, 128, seed=21)
    q = torch.randn(1, 8, 128, device=DEV).half()
    o, M = c.attend(q, table, ints(*lens), 0.09, return_stats=True)
    check_decode(o, M, q, c, table, lens, 0.09)
    # the same tokens under a wider table, and a shorter prefix of them
    wide = torch.full((1, 4 * table.shape[1]), -1, dtype=I32, device=DEV)
    wide[:, :table.shape[1]] = table
    o2, M2 = c.attend(q, wide, ints(*lens), 0.09, return_stats=True)
    check_decode(o2, M2, q, c, table, lens, 0.09)
    o3, M3 = c.attend(q, wide, ints(333), 0.09, return_stats=True)
    check_decode(o3, M3, q, c, table, [333], 0.09)


def test_decode_batches_and_tables_wider_than_their_sequences():
    lens = [(37 * i) % 500 for i in range(130)] + [9000]
    c, table = filled_cache(lens, 1, 16, 64, seed=22)
    q = torch.randn(131, 5, 64, device=DEV).bfloat16()
    n = torch.tensor(lens, dtype=I32, device=DEV)
    o, M = c.attend(q, table, n, 0.125, return_stats=True)
    check_decode(o, M, q, c, table, lens, 0.125)


def test_decode_pages_that_do_not_exist():
    lens = [100, 40, 16, 64]
    c, table = filled_cache(lens, 2, 16, 64, seed=23)
    table[0, 1] = -1
    table[0, 6] = 10 ** 9
    table[1] = -1  # no page at all
    table[2, 0] = c.k.shape[0]
    table[3, 3] = -2 ** 31
    q = torch.randn(4, 4, 64, device=DEV).half()
    o, M = c.attend(q, table, torch.tensor(lens, dtype=I32, device=DEV), 0.2, return_stats=True)
    check_decode(o, M, q, c, table, lens, 0.2)
    # lengths outside the table are cut, negative ones empty
    o, M = c.attend(q, table, ints(-3, 10 ** 9, -2 ** 31, 2 ** 31 - 1), 0.2, return_stats=True)
    check_decode(o, M, q, c, table, [0, 112, 0, 112], 0.2)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_decode_scales_far_apart(dtype):
    """Pages whose scales differ by 2^40: the weights' exponents may not leave fp16."""
    lens = [400, 90]
    c, table = filled_cache(lens, 2, 16, 128, seed=24)
    g = torch.Generator(device=DEV).manual_seed(5)
    c.v_scale.copy_(torch.exp2(torch.randint(-30, 11, c.v_scale.shape, generator=g, device=DEV).float()))
    c.k_scale.copy_(torch.exp2(torch.randint(-20, -5, c.k_scale.shape, generator=g, device=DEV).float()))
    q = torch.randn(2, 8, 128, device=DEV, generator=g).to(dtype)
    scale = 2.0 ** -9 if dtype == torch.float16 else 0.09  # outputs of fp16 may not overflow: values up to 448 * 2^10
    if dtype == torch.float16:
        c.v_scale.clamp_(max=2.0 ** 6)
    o, M = c.attend(q, table, ints(*lens), scale, return_stats=True)
    check_decode(o, M, q, c, table, lens, scale)


def test_decode_queries_far_from_one():
    """bf16 rows of 2^60 and of 2^-60 beside each other: each is scaled on its own."""
    lens = [200]
    c, table = filled_cache(lens, 1, 32, 64, seed=25)
    g = torch.Generator(device=DEV).manual_seed(6)
    q = torch.randn(1, 4, 64, device=DEV, generator=g).bfloat16()
    for e, scale in ((60, 2.0 ** -63), (-60, 2.0 ** 57)):
        o, M = c.attend((q.double() * 2.0 ** e).bfloat16(), table, ints(200), scale, return_stats=True)
        o0, M0 = c.attend(q, table, ints(200), 0.125, return_stats=True)
        assert torch.equal(o, o0) and torch.equal(M, M0)
    # near the end of bf16's range, with values that stay normal numbers there
    q = ((1 + torch.rand(1, 4, 64, device=DEV, generator=g)) * torch.randn(1, 4, 64, device=DEV, generator=g).sign()).bfloat16()
    for e, scale in ((-118, 2.0 ** 115), (-125, 2.0 ** 122), (120, 2.0 ** -123)):
        o, M = c.attend((q.double() * 2.0 ** e).bfloat16(), table, ints(200), scale, return_stats=True)
        o0, M0 = c.attend(q, table, ints(200), 0.125, return_stats=True)
        assert torch.equal(o, o0) and torch.equal(M, M0)
    mixed = q.clone()
    mixed[0, 1] = (q[0, 1].double() * 2.0 ** -50).bfloat16()
    mixed[0, 3] = 0.0
    o, M = c.attend(mixed, table, ints(200), 0.125, return_stats=True)
    check_decode(o, M, mixed, c, table, lens, 0.125)


def test_decode_one_key_above_a_long_flat_cache():
    """A key far above 60000 equal ones whose weights add up: they may not vanish below fp16's range."""
    n, D = 60000, 64
    c = new_cache(-(-n // 64), 1, 64, D)
    table = torch.arange(c.k.shape[0], dtype=I32, device=DEV)[None]
    c.v.view(torch.uint8).fill_(0x38)  # 1.0
    c.k[0, 0, 0] = 1.0
    c.v[0, 0, 0] = -1.0
    q = torch.full((1, 1, D), 0.25, device=DEV).half()  # score 16 * scale for the key, 0 for the others
    o, M = c.attend(q, table, ints(n), 1.0, return_stats=True)
    check_decode(o, M, q, c, table, [n], 1.0)


def test_decode_nan():
    lens = [100, 100]
    c, table = filled_cache(lens, 1, 16, 64, seed=26)
    q = torch.randn(2, 3, 64, device=DEV).half()
    n = ints(100, 100)
    q[0, 1, 7] = math.nan
    o = c.attend(q, table, n, 0.125)
    assert torch.isnan(o[0, 1]).all() and int(torch.isnan(o).sum()) == 64
    c.k.view(torch.uint8)[int(table[1, 2]), 0, 3, 5] = 0x7F  # a key of the second sequence
    o = c.attend(q, table, n, 0.125)
    assert torch.isnan(o[1]).all() and torch.isfinite(o[0, 0]).all()


def test_decode_cache_past_32_bit_offsets():
    page, heads, D = 128, 4, 256
    pages = (1 << 32) // (page * heads * D) + 50  # 4.3 GB a side
    c = tb.PagedKVCache(pages, page, heads, D)
    lens = [300]
    ids = [pages - 1, pages - 30, 3]
    table = ints(*ids)[None]
    k, v = (torch.randn(300, heads, D, device=DEV).half() for _ in range(2))
    c.append(k, v, table, ints(300), ints(0, 300))
    q = torch.randn(1, 8, D, device=DEV).half()
    o, M = c.attend(q, table, ints(300), 0.07, return_stats=True)
    check_decode(o, M, q, c, table, lens, 0.07)
    for h in range(heads):  # and what was stored is k to e4m3's precision
        got = c.k[ids[0], h].float() * c.k_scale[ids[0], h]
        assert ((got - k[:128, h].float()).abs() <= k[:128, h].float().abs() * 2.0 ** -4 + c.k_scale[ids[0], h] * 2.0 ** -10).all()


# ------------------------------------------------------------------ together
def layer_reference(q, k8, v8, scale):
    group = q.shape[0] // k8.shape[1]
    return [one_head(q[h:h + 1], k8[:, h // group], v8[:, h // group], scale, False) for h in range(q.shape[0])]


def test_prompt_then_tokens():
    """A batch of prompts, their keys and values cached, then tokens one by one: each step against the same
    attention in 64 bits over what the cache stands for."""
    prompts, hq, hkv, D, page, steps = [5, 130, 64, 1], 8, 2, 128, 16, 20
    g = torch.Generator(device=DEV).manual_seed(31)
    q, k, v, cu, off = pack(prompts, hq, hkv, D, torch.bfloat16, seed=32)
    scale = D ** -0.5
    cache = tb.PagedKVCache(64, page, hkv, D)
    table = torch.randperm(64, generator=torch.Generator().manual_seed(2)).view(4, 16).to(I32).to(DEV)
    lens = torch.tensor(prompts, dtype=I32, device=DEV)
    o = tb.attention_varlen(q, k, v, cu, True, scale)
    cache.append(k, v, table, lens, cu)
    check_pack(o, None, q, k, v, off, True, scale)
    for step in range(steps):
        lens += 1
        q1, k1, v1 = (torch.randn(4, h, D, generator=g, device=DEV).bfloat16() for h in (hq, hkv, hkv))
        cache.append(k1, v1, table, lens)
        o, M = cache.attend(q1, table, lens, scale, return_stats=True)
        check_decode(o, M, q1, cache, table, [n + step + 1 for n in prompts], scale, f"step {step}")
    # the cache is still the prompt's keys to within e4m3 and its blocks' scales
    for b, n in enumerate(prompts):
        ids = table[b].long()[:-(-n // page)]
        got = (cache.k[ids].float() * cache.k_scale[ids][..., None, None]).transpose(0, 1).reshape(hkv, -1, D)[:, :n]
        want = k[off[b]:off[b + 1]].float().transpose(0, 1)
        floor = cache.k_scale[ids].amax() * 2.0 ** -10
        # twice: a page whose scale grew was rounded again
        assert ((got - want).abs() <= 2 * (want.abs() * 2.0 ** -4 + floor)).all()


def test_captured_step_replays_with_new_lengths():
    """Append and attend captured once; replays follow the tensors: lengths, tokens, pages.  Two graphs of one
    shape, replayed in turn on two streams, keep out of each other's way."""
    hq, hkv, D, page, batch = 8, 2, 64, 16, 3
    g = torch.Generator(device=DEV).manual_seed(41)

    def make():
        s = dict(c=tb.PagedKVCache(300, page, hkv, D), lens=ints(3, 700, 40),
                 table=torch.randperm(300, generator=torch.Generator().manual_seed(3)).view(3, 100).to(I32).to(DEV),
                 q=torch.zeros(batch, hq, D, device=DEV).half(), k=torch.zeros(batch, hkv, D, device=DEV).half(),
                 v=torch.zeros(batch, hkv, D, device=DEV).half())
        first = [torch.randn(743, hkv, D, generator=g, device=DEV).half() for _ in range(2)]
        s["c"].append(*first, s["table"], s["lens"], ints(0, 3, 703, 743))

        def step():
            s["lens"] += 1
            s["c"].append(s["k"], s["v"], s["table"], s["lens"])
            s["o"], s["M"] = s["c"].attend(s["q"], s["table"], s["lens"], 0.125, return_stats=True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
            side.synchronize()
            s["graph"] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(s["graph"], stream=side):
                step()
        torch.cuda.synchronize()
        return s

    both = [make(), make()]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    lens = [4, 701, 41]
    for step in range(20):
        lens = [n + 1 for n in lens]
        for s in both:
            for name in "qkv":
                s[name].copy_(torch.randn(s[name].shape, generator=g, device=DEV))
        torch.cuda.synchronize()
        for s, st in zip(both, streams):
            with torch.cuda.stream(st):
                s["graph"].replay()
        torch.cuda.synchronize()
        for s in both:
            assert s["lens"].tolist() == lens
            if step % 6 == 0:
                check_decode(s["o"], s["M"], s["q"], s["c"], s["table"], lens, 0.125, f"replay {step}")


def test_varlen_captured_with_new_offsets():
    q, k, v, cu, off = pack([100, 300], 4, 2, 64, torch.float16, seed=51)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tb.attention_varlen(q, k, v, cu, True, 0.125)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            o = tb.attention_varlen(q, k, v, cu, True, 0.125)
    torch.cuda.synchronize()
    for new in ([0, 100, 400], [0, 1, 400], [0, 399, 400], [0, 200, 200], [0, 0, 0]):
        cu.copy_(torch.tensor(new, dtype=I32))
        graph.replay()
        want = tb.attention_varlen(q, k, v, cu, True, 0.125)
        torch.cuda.synchronize()
        assert torch.equal(o, want)
        check_pack(o, None, q, k, v, new, True, 0.125)


def test_custom_ops_run():
    q, k, v, cu, off = pack([20, 60], 4, 2, 64, torch.float16, seed=61)
    ns = torch.ops.triton_b200
    assert torch.equal(ns.attention_varlen(q, k, v, cu, True, 0.125), tb.attention_varlen(q, k, v, cu, True, 0.125))
    a, b = tb.PagedKVCache(8, 16, 2, 64), tb.PagedKVCache(8, 16, 2, 64)
    table, lens = torch.arange(8, dtype=I32, device=DEV).view(2, 4), ints(20, 60)
    a.append(k, v, table, lens, cu)
    ns.kv_cache_append(b.k, b.v, b.k_scale, b.v_scale, k, v, table, lens, cu)
    assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8)) and torch.equal(a.v_scale, b.v_scale)
    x = torch.randn(2, 4, 64, device=DEV).half()
    assert torch.equal(ns.attention_decode(x, b.k, b.v, b.k_scale, b.v_scale, table, lens, 0.125), a.attend(x, table, lens, 0.125))


def test_inputs_that_require_grad_under_no_grad():
    q, k, v, cu, off = pack([33], 2, 1, 64, torch.float16, seed=71)
    want = tb.attention_varlen(q, k, v, cu, True, 0.125)
    q.requires_grad_(True)
    with pytest.raises(RuntimeError, match="no backward"):
        tb.attention_varlen(q, k, v, cu, True, 0.125)
    with torch.no_grad():
        assert torch.equal(tb.attention_varlen(q, k, v, cu, True, 0.125), want)


def test_empty_batches_tables_and_caches():
    c = tb.PagedKVCache(4, 16, 2, 64)
    x = lambda *s: torch.randn(*s, device=DEV).half()
    none = torch.zeros(0, dtype=I32, device=DEV)
    assert c.attend(x(0, 4, 64), none.view(0, 3), none, 0.1).shape == (0, 4, 64)          # no sequence
    c.append(x(0, 2, 64), x(0, 2, 64), none.view(0, 3), none)
    o, M = c.attend(x(3, 4, 64), none.view(3, 0), ints(5, 0, 70), 0.1, return_stats=True)  # a table without a column
    assert (o == 0).all() and (M == -math.inf).all()
    c.append(x(3, 2, 64), x(3, 2, 64), none.view(3, 0), ints(5, 1, 70))
    assert (c.k.view(torch.uint8) == 0).all() and (c.k_scale == 1).all()
    e = tb.PagedKVCache(0, 16, 2, 64)                                                      # a cache without a page
    table = torch.zeros(3, 2, dtype=I32, device=DEV)
    e.append(x(3, 2, 64), x(3, 2, 64), table, ints(1, 2, 3))
    assert (e.attend(x(3, 4, 64), table, ints(1, 2, 3), 0.1) == 0).all()


@pytest.mark.parametrize("D,group,lens", [(128, 4, [20000, 3, 15001]), (64, 1, [5000] * 30), (256, 2, [9000, 0])])
def test_decode_captured_where_chunks_are_joined_by_a_second_kernel(D, group, lens):
    """Wide tables: the chunks' results go through a workspace.  Two graphs and eager calls in turn on streams of
    their own give what each gives alone."""
    c, table = filled_cache(lens, 2, 64, D, seed=D)
    assert _lib.lib().b200_attention_decode_workspace(len(lens), 2 * group, 2, D, 64, table.shape[1]) > 0
    g = torch.Generator(device=DEV).manual_seed(8)
    qs = [torch.randn(len(lens), 2 * group, D, generator=g, device=DEV).half() for _ in range(3)]
    n = torch.tensor(lens, dtype=I32, device=DEV)
    want = [c.attend(q, table, n, 0.1, return_stats=True) for q in qs]
    torch.cuda.synchronize()
    check_decode(*want[0], qs[0], c, table, lens, 0.1)
    streams, graphs, outs = [torch.cuda.Stream() for _ in qs], [], []
    for q, st in zip(qs[:2], streams):
        st.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            outs.append(c.attend(q, table, n, 0.1, return_stats=True))
        graphs.append(graph)
    for _ in range(10):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = c.attend(qs[2], table, n, 0.1, return_stats=True)
        torch.cuda.synchronize()
        for got, w in zip(outs + [eager], want):
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])


def test_decode_table_sliced_to_the_longest_sequence():
    """A table as wide as the longest sequence a program admits, its columns sliced to the ones in use."""
    lens = [700, 12, 350]
    c, table = filled_cache(lens, 2, 16, 128, seed=81)
    wide = torch.full((3, 4096), -1, dtype=I32, device=DEV)
    wide[:, :table.shape[1]] = table
    q = torch.randn(3, 6, 128, device=DEV).bfloat16()
    n = torch.tensor(lens, dtype=I32, device=DEV)
    o = c.attend(q, wide[:, :table.shape[1]], n, 0.1)
    assert torch.equal(o, c.attend(q, table, n, 0.1))
    o2, M2 = c.attend(q, wide, n, 0.1, return_stats=True)
    check_decode(o2, M2, q, c, table, lens, 0.1)


def test_decode_a_sequence_does_not_depend_on_the_others():
    """Its bits are those of the sequence alone under a table of the same width and a batch of the same size."""
    lens = [1500, 900, 40, 1501]
    c, table = filled_cache(lens, 2, 32, 64, seed=82)
    q = torch.randn(4, 8, 64, device=DEV).half()
    n = torch.tensor(lens, dtype=I32, device=DEV)
    o = c.attend(q, table, n, 0.1)
    for b in range(4):
        only = torch.zeros_like(n)
        only[b] = n[b]
        other = torch.full_like(table, -1)
        other[b] = table[b]
        assert torch.equal(c.attend(q, other, only, 0.1)[b], o[b])


def test_varlen_a_very_large_batch():
    """40000 sequences of 0 to 3 rows: finding the items stays linear in them."""
    lens = [i % 4 for i in range(40000)]
    q, k, v, cu, off = pack(lens, 2, 1, 64, torch.float16, seed=91)
    o = tb.attention_varlen(q, k, v, cu, True, 0.125)
    first = torch.tensor([off[b] for b in range(40000) if lens[b]], device=DEV)
    assert torch.equal(o[first], v[first].expand(-1, 2, -1))  # a first row sees itself alone
    second = torch.tensor([off[b] + 1 for b in range(40000) if lens[b] >= 2], device=DEV)
    with_first = (q[second].double() * k[second - 1].double()).sum(-1) * 0.125
    own = (q[second].double() * k[second].double()).sum(-1) * 0.125
    p = torch.softmax(torch.stack([with_first, own], -1), -1)
    want = p[..., :1] * v[second - 1].double() + p[..., 1:] * v[second].double()
    bound = 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -12 + 2.0 ** -14) * (v[second - 1].double().abs() + v[second].double().abs())
    assert bool(((o[second].double() - want).abs() <= bound).all())


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hq,hkv,D", [(16, 8, 64), (24, 4, 128), (32, 1, 128), (9, 3, 64), (21, 3, 256), (40, 1, 64), (26, 2, 128)])
def test_varlen_short_sequences_all_heads_of_a_group_to_a_tile(hq, hkv, D, causal):
    """Short sequences: a tile's rows are positions times the heads of a group (up to 32 of them), whether those
    divide a warp's rows (2, 6, 32) or not (3, 7, 13); 40 heads stay one by one."""
    lens = [1, 127, 128, 129, 300, 5, 0, 640, 77, 256] + [(13 * i) % 200 for i in range(60)]
    q, k, v, cu, off = pack(lens, hq, hkv, D, torch.bfloat16, seed=hq + D, tail=9)
    assert q.shape[0] <= 192 * len(lens)
    o, M = tb.attention_varlen(q, k, v, cu, causal, 0.1, return_stats=True)
    some = list(range(0, hq, 5)) + [hq - 1]
    for b in list(range(10)) + [33, 69]:
        a, e = off[b], off[b + 1]
        for h in some if e > a else []:
            kh = h // (hq // hkv)
            want = one_head(q[a:e, h], k[a:e, kh], v[a:e, kh], 0.1, causal)
            check(o[a:e, h], want, q.dtype, q.dtype, f"sequence {b} head {h}")
            check_lse(M[h, a:e], want, f"lse of sequence {b} head {h}")
    # a short sequence's bits are those it has alone
    for b in range(0, 70, 7):
        a, e = off[b], off[b + 1]
        if 0 < e - a <= 192:
            assert torch.equal(o[a:e], tb.attention_varlen(q[a:e], k[a:e], v[a:e], ints(0, e - a), causal, 0.1))
    assert (o[off[-1]:] == 0).all() and (M[:, off[-1]:] == -math.inf).all()
    mine = torch.full_like(q, 5.0)
    tb.attention_varlen(q, k, v, cu, causal, 0.1, out=mine)
    assert torch.equal(mine[:off[-1]], o[:off[-1]]) and (mine[off[-1]:] == 5.0).all()
    q[off[4]:off[5]] = math.nan  # neighbours stay as they are
    k[off[4]:off[5]] = math.inf
    v[off[4]:off[5]] = math.nan
    v[off[-1]:] = math.nan
    again = tb.attention_varlen(q, k, v, cu, causal, 0.1)
    assert torch.equal(again[:off[4]], o[:off[4]]) and torch.equal(again[off[5]:], o[off[5]:])


def test_calls_on_several_streams_at_once():
    """Eager packed calls on two streams and a replayed graph on a third, over and over: each gives its own result."""
    packs = [pack([900, 40, 333], 8, 2, 64, torch.float16, seed=101), pack([5] * 50, 4, 4, 64, torch.bfloat16, seed=102),
             pack([2000], 4, 1, 128, torch.float16, seed=103)]
    want = [tb.attention_varlen(q, k, v, cu, True, 0.1) for q, k, v, cu, _ in packs]
    streams = [torch.cuda.Stream() for _ in packs]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[2]):
        q, k, v, cu, _ = packs[2]
        captured = tb.attention_varlen(q, k, v, cu, True, 0.1)
    for _ in range(20):
        got = []
        for (q, k, v, cu, _), st in zip(packs[:2], streams):
            with torch.cuda.stream(st):
                got.append(tb.attention_varlen(q, k, v, cu, True, 0.1))
        with torch.cuda.stream(streams[2]):
            captured.zero_()
            graph.replay()
        torch.cuda.synchronize()
        for g, w in zip(got + [captured], want):
            assert torch.equal(g, w)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_every_length_around_the_chunks_and_slabs(D):
    """Lengths on and beside multiples of 16 and of the chunks, under tables that make one chunk, a cluster, a join."""
    for width, batch in ((8, 40), (64, 12), (700, 9)):
        lens = [max(0, width * 16 - d) for d in range(batch)]
        lens[-1] = 16 * (width // 2) + 1
        c, table = filled_cache(lens, 1, 16, D, seed=width + D)
        q = torch.randn(batch, 3, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(width)).bfloat16()
        o, M = c.attend(q, table, torch.tensor(lens, dtype=I32, device=DEV), 0.11, return_stats=True)
        check_decode(o, M, q, c, table, lens, 0.11, f"width {width}")


def test_varlen_refuses_an_unaligned_out():
    q, k, v, cu, _ = pack([10], 2, 1, 64, torch.float16, seed=111)
    odd = torch.zeros(10 * 2 * 64 + 8, dtype=torch.float16, device=DEV)
    wide = torch.zeros(10, 2, 68, dtype=torch.float16, device=DEV)
    for out in (odd[1:1281].view(10, 2, 64), wide[..., :64]):
        with pytest.raises(RuntimeError, match="aligned|multiple"):
            tb.attention_varlen(q, k, v, cu, True, 0.1, out=out)
    big = pack([3000], 4, 1, 64, torch.float16, seed=112)  # through boxes
    with pytest.raises(RuntimeError, match="aligned|multiple"):
        tb.attention_varlen(*big[:4], True, 0.1, out=torch.zeros(3000, 4, 68, dtype=torch.float16, device=DEV)[..., :64])
    assert (odd == 0).all() and (wide == 0).all()


# ------------------------------------------------------------------ values that are not finite, and masked places
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("hq,hkv,D", [(2, 2, 64), (2, 2, 128), (4, 2, 128), (2, 2, 256)])
def test_varlen_bad_keys_at_every_column(hq, hkv, D, bad, causal):
    """A key of NaN, or one whose score is +inf, at every position mod 16 of the first and the second block: every
    row that sees it is NaN, and only those."""
    n, group = 160, hq // hkv
    q, k, v, cu, off = pack([n] * 32, hq, hkv, D, torch.bfloat16, seed=121 + D)
    q[..., 0] = 1.0
    clean = k.clone()
    at = [b % 16 + 16 + (112 if b >= 16 else 0) for b in range(32)]
    for b in range(32):
        k[off[b] + at[b], :, 0] = bad
    o, M = tb.attention_varlen(q, k, v, cu, causal, 0.1, return_stats=True)
    dense = lambda t: t.view(32, n, -1, D).transpose(1, 2).repeat_interleave(hq // t.shape[1], 1).contiguous()
    o2, M2 = tb.attention_forward(dense(q), dense(k), dense(v), causal, 0.1)  # the dense form of the kernel
    o2, M2 = o2.transpose(1, 2).reshape(o.shape), M2.transpose(0, 1).reshape(M.shape)
    assert torch.equal(torch.isnan(o2), torch.isnan(o)) and torch.equal(torch.isnan(M2), torch.isnan(M))
    for b in range(32):
        first = off[b] + at[b] if causal else off[b]
        assert torch.isnan(o[first:off[b + 1]]).all(), f"a key at position {at[b]} is not seen"
        assert torch.isnan(M[:, first:off[b + 1]]).all()
        check_pack(o[off[b]:first], None, q[off[b]:first], clean[off[b]:first], v[off[b]:first], [0, first - off[b]], True, 0.1)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_masked_weights_are_zero(D):
    """Values near bf16's largest behind a row, where causal masking hides them, add nothing to it."""
    q, k, v, cu, off = pack([100, 300], 2, 2, D, torch.bfloat16, seed=131)
    v[50:100] = 1e38
    v[300:] = 1e38
    o = tb.attention_varlen(q, k, v, cu, True, 0.1)
    check_pack(o[:50], None, q[:50], k[:50], v[:50], [0, 50], True, 0.1)
    check_pack(o[100:300], None, q[100:300], k[100:300], v[100:300], [0, 200], True, 0.1)
    dense = lambda t: t[100:].transpose(0, 1)[None].contiguous()
    o, _ = tb.attention_forward(dense(q), dense(k), dense(v), True, 0.1)
    check_pack(o[0, :, :200].transpose(0, 1), None, q[100:300], k[100:300], v[100:300], [0, 200], True, 0.1)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_varlen_a_first_block_of_minus_infinity(D, dtype):
    """Scores of -inf have weight 0, also where a whole block of keys has nothing else."""
    q, k, v, cu, off = pack([400], 2, 1, D, dtype, seed=141)
    q = q.abs() + 0.1
    k[:128] = -math.inf
    o, M = tb.attention_varlen(q, k, v, cu, False, 0.1, return_stats=True)
    for h in range(2):
        want = one_head(q[:, h], k[128:, 0], v[128:, 0], 0.1, False)
        check(o[:, h], want, dtype, dtype, f"head {h}")
        check_lse(M[h], want, f"lse of head {h}")
    o = tb.attention_varlen(q, k, v, cu, True, 0.1)
    assert torch.isnan(o[:128]).all()  # nothing but -inf: 0 / 0
    for h in range(2):
        want = one_head(q[128:, h], k[128:, 0], v[128:, 0], 0.1, True)
        check(o[128:, h], want, dtype, dtype, f"causal, head {h}")


def test_varlen_statistics_of_rows_outside_the_sequences_with_out():
    """M is the call's own tensor: -inf for rows that belong to no sequence, whether O is or not."""
    for D in (64, 32):
        q, k, v, cu, off = pack([130, 9], 2, 2, D, torch.float16, seed=151, tail=150)
        for offsets, inside in ((cu, slice(0, 139)), (cu + 20, slice(20, 159)), (ints(0), slice(0, 0))):
            before = torch.full((2, 289), 5.0, device=DEV)  # what the allocator hands out next
            del before
            mine = torch.full_like(q, 7.0)
            o, M = tb.attention_varlen(q, k, v, offsets, True, 0.2, out=mine, return_stats=True)
            rest = torch.ones(289, dtype=torch.bool, device=DEV)
            rest[inside] = False
            assert (M[:, rest] == -math.inf).all() and torch.isfinite(M[:, inside]).all()
            assert (mine[rest] == 7.0).all()


def test_decode_large_queries_over_small_keys():
    """q near the end of bf16's range, keys at the other: the score is an ordinary number and so is the output."""
    lens = [200]
    c, table = filled_cache(lens, 1, 32, 64, seed=161)
    g = torch.Generator(device=DEV).manual_seed(7)
    q = ((1 + torch.rand(1, 4, 64, device=DEV, generator=g)) * torch.randn(1, 4, 64, device=DEV, generator=g).sign()).bfloat16()
    o0, M0 = c.attend(q, table, ints(200), 8.0, return_stats=True)
    check_decode(o0, M0, q, c, table, lens, 8.0)
    k_scale = c.k_scale.clone()  # 2^-8 .. 2^-3
    for e in (100, 117):
        c.k_scale.copy_(k_scale * 2.0 ** -e)
        o, M = c.attend((q.double() * 2.0 ** e).bfloat16(), table, ints(200), 8.0, return_stats=True)
        assert torch.equal(o, o0) and torch.equal(M, M0)
        if e == 100:
            c.k_scale.copy_(k_scale * 2.0 ** e)
            o, M = c.attend((q.double() * 2.0 ** -e).bfloat16(), table, ints(200), 8.0, return_stats=True)
            assert torch.equal(o, o0) and torch.equal(M, M0)
    # keys of zero under the largest scales
    c.k_scale.fill_(2.0 ** 119)
    c.k.view(torch.uint8).zero_()
    o, M = c.attend((q.double() * 2.0 ** 126).bfloat16(), table, ints(200), 0.125, return_stats=True)
    check_decode(o, M, torch.zeros_like(q), c, table, lens, 0.125)


CAPTURE_MANY = """
import gc, time, torch, triton_b200 as tb
dev = "cuda"
g = torch.Generator(device=dev).manual_seed(1)
q, k, v = (torch.randn(2000, h, 64, generator=g, device=dev).half() for h in (8, 2, 2))
cu = torch.tensor([0, 1500, 1500, 2000], dtype=torch.int32, device=dev)
want = tb.attention_varlen(q, k, v, cu, True, 0.1)
dq, dk, dv = (torch.randn(1, 2, 300, 64, generator=g, device=dev).half() for _ in range(3))
dwant = tb.attention_forward(dq, dk, dv, True, 0.1)[0]

def capture(n, call, want):
    outs, graph = [], torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i in range(n):
            o = call()
            if i % 500 == 0:
                outs.append(o)
    for _ in range(2):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)
    return graph, outs

packed = lambda: tb.attention_varlen(q, k, v, cu, True, 0.1)
# graphs that are destroyed give their launches' counters back, packed and dense ones
for call, w in ((packed, want), (lambda: tb.attention_forward(dq, dk, dv, True, 0.1)[0], dwant)):
    for _ in range(3):
        kept = capture(2000, call, w)
        del kept
        gc.collect()
        torch.cuda.synchronize()
        time.sleep(0.2)
# more at a time than there are counters
kept = [capture(1500, packed, want) for _ in range(3)]
cu.copy_(torch.tensor([0, 0, 3, 2000], dtype=torch.int32))
want = packed()
for graph, outs in kept:
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
assert tb._lib.status() == 0
print("fine")
"""


def test_captures_do_not_run_out_of_work_counters():
    """More captured launches than the pool of work counters holds, one graph after another and at a time; in a
    process of their own."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CAPTURE_MANY], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("fine"), r.stdout + r.stderr


def test_calls_count_as_changes_of_what_they_write():
    """autograd's version counters: a tensor saved for a backward and then written by a call is noticed."""
    q, k, v, cu, off = pack([20, 60], 4, 2, 64, torch.float16, seed=171)
    c = tb.PagedKVCache(8, 16, 2, 64)
    table, lens = torch.arange(8, dtype=I32, device=DEV).view(2, 4), ints(20, 60)
    w = torch.ones_like(c.k_scale, requires_grad=True)
    y = (w * c.k_scale).sum()
    c.append(k, v, table, lens, cu)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    for t in (c.k, c.v, c.k_scale, c.v_scale):
        assert t._version > 0
    mine = torch.zeros_like(q)
    tb.attention_varlen(q, k, v, cu, True, 0.1, out=mine)
    one = torch.zeros(2, 4, 64, device=DEV).half()
    c.attend(q[:2], table, lens, 0.1, out=one)
    assert mine._version == 1 and one._version == 1
    with torch.inference_mode():
        d = tb.PagedKVCache(8, 16, 2, 64)
        d.append(k, v, table, lens, cu)
        tb.attention_varlen(q, k, v, cu, True, 0.1, out=torch.zeros_like(q))
        assert torch.equal(d.k.view(torch.uint8), c.k.view(torch.uint8))


def test_calls_refuse_outputs_that_overlap():
    """An `out` whose elements share memory, or that lies over k, v or the cache, would be written while it is read."""
    q, k, v, cu, off = pack([20, 60], 2, 2, 64, torch.float16, seed=181)
    want = tb.attention_varlen(q, k, v, cu, True, 0.1)
    kept = k.clone(), v.clone()
    for out in (k, v, torch.zeros(1, 2, 64, device=DEV).half().expand(80, 2, 64), torch.zeros(80, 1, 64, device=DEV).half().expand(80, 2, 64)):
        with pytest.raises(RuntimeError):
            tb.attention_varlen(q, k, v, cu, True, 0.1, out=out)
    assert torch.equal(k, kept[0]) and torch.equal(v, kept[1])
    c, table = filled_cache([20, 60], 2, 16, 64, seed=182)
    x = q[:2].clone()
    one = c.attend(x, table, ints(20, 60), 0.1)
    with pytest.raises(RuntimeError):
        c.attend(x, table, ints(20, 60), 0.1, out=torch.zeros(1, 2, 64, device=DEV).half().expand(2, 2, 64))
    # q itself may take the output: a row of it is read by the tile that writes it
    assert torch.equal(c.attend(x, table, ints(20, 60), 0.1, out=x), one)
    assert torch.equal(tb.attention_varlen(q, k, v, cu, True, 0.1, out=q), want)


def test_inputs_whose_elements_share_memory():
    """Heads or rows expanded from one: a stride of zero."""
    q, k, v, cu, off = pack([20, 60], 4, 1, 128, torch.bfloat16, seed=191)
    wide = lambda t: t.expand(80, 2, 128)
    want = tb.attention_varlen(q, wide(k).contiguous(), wide(v).contiguous(), cu, True, 0.1)
    assert torch.equal(tb.attention_varlen(q, wide(k), wide(v), cu, True, 0.1), want)
    one_q = q[:1].expand(80, 4, 128)
    assert torch.equal(tb.attention_varlen(one_q, k, v, cu, True, 0.1), tb.attention_varlen(one_q.contiguous(), k, v, cu, True, 0.1))
    a, b = tb.PagedKVCache(8, 16, 2, 128), tb.PagedKVCache(8, 16, 2, 128)
    table, lens = torch.arange(8, dtype=I32, device=DEV).view(2, 4), ints(20, 60)
    a.append(wide(k), wide(v), table, lens, cu)
    b.append(wide(k).contiguous(), wide(v).contiguous(), table, lens, cu)
    assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8)) and torch.equal(a.v_scale, b.v_scale)
    x = q[:1].expand(2, 4, 128)
    assert torch.equal(a.attend(x, table, lens, 0.1), a.attend(x.contiguous(), table, lens, 0.1))


def test_out_of_memory_is_torchs():
    """An output that cannot be had is torch's OutOfMemoryError, as everywhere else."""
    q = torch.zeros(1, 1, 64, device=DEV).half().expand(1 << 20, 1 << 16, 64)
    k = torch.zeros(1, 1, 64, device=DEV).half().expand(1 << 20, 1, 64)
    with pytest.raises(torch.OutOfMemoryError):
        tb.attention_varlen(q, k, k, ints(0, 1), True, 0.1)


@pytest.mark.parametrize("causal", [True, False])
def test_varlen_offsets_that_name_the_same_rows_over_and_over(causal):
    """Decreasing offsets that add up to more work than an int counts: no work, and nothing breaks."""
    T, H, batch = 16384, 32, (1 << 21) + 2
    q = torch.zeros(T, H, 64, dtype=torch.float16, device=DEV)
    cu = torch.zeros(batch + 1, dtype=I32, device=DEV)
    cu[1::2] = T
    mine = torch.full_like(q, 7.0)
    tb.attention_varlen(q, q, q, cu, causal, 0.1, out=mine)
    torch.cuda.synchronize()
    assert _lib.status() == 0 and (mine == 7.0).all()
    # a few of them are fine: the same rows, computed twice
    q.normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    o = tb.attention_varlen(q[:300], q[:300], q[:300], ints(0, 300, 0, 300), causal, 0.1)
    assert torch.equal(o, tb.attention_varlen(q[:300], q[:300], q[:300], ints(0, 300), causal, 0.1))
