"""Serving operators: attention over packed prompts, writing a paged 8-bit cache, attention of single tokens over it.

`run` computes an operator in its plain form (elementary torch operations in 32 bits) or, where `own` is true, by
the framework's call.  Sizes are those of the repository's attention benchmarks (32 and 48 heads, head dims 64
and 128, lengths 1024 and 4096) and generic ones around them.
"""
import math
import random

import torch

own = False

E4M3_MAX = 448.0


def listed():
    """Every case is a pass of one layer of a serving program."""
    return [
        # a question of a few words, alone: latency
        dict(name="prompt_one_short", op="prompt", batch=1, shortest=37, longest=37, hq=8, hkv=2, d=64, dtype="float16", causal=True, lens_seed=1),
        # one medium prompt, alone
        dict(name="prompt_one_medium", op="prompt", batch=1, shortest=2000, longest=2000, hq=32, hkv=8, d=128, dtype="bfloat16", causal=True, lens_seed=2),
        # a batch of prompts as they arrive: lengths from a few tokens to some thousand
        dict(name="prompt_ragged", op="prompt", batch=12, shortest=5, longest=2300, hq=32, hkv=8, d=128, dtype="bfloat16", causal=True, lens_seed=3),
        # the repository's large attention shape (4 x 32 heads x 4096 x 128) as a pack with grouped heads
        dict(name="prompt_4x4096", op="prompt", batch=4, shortest=4096, longest=4096, hq=32, hkv=8, d=128, dtype="float16", causal=True, lens_seed=4),
        # texts read in both directions (an encoder's batch), a k/v head for each q head, head dim 64
        dict(name="prompt_both_ways", op="prompt", batch=6, shortest=300, longest=1100, hq=48, hkv=48, d=64, dtype="bfloat16", causal=False, lens_seed=5),
        # the new token of one conversation: latency
        dict(name="append_token", op="append", batch=1, held_most=3000, shortest=1, longest=1, hkv=8, d=128, page=16, dtype="bfloat16", lens_seed=6),
        # the new tokens of a full batch
        dict(name="append_tokens_200", op="append", batch=200, held_most=2000, shortest=1, longest=1, hkv=8, d=128, page=64, dtype="bfloat16", lens_seed=7),
        # prompts of a batch, some behind a conversation's earlier turns
        dict(name="append_prompts", op="append", batch=24, held_most=1000, shortest=10, longest=4096, hkv=8, d=128, page=64, dtype="float16", lens_seed=8),
        # one conversation of medium length: latency, few heads to share the work
        dict(name="decode_one", op="decode", batch=1, shortest=1900, longest=1900, hq=32, hkv=8, d=128, page=16, dtype="bfloat16", lens_seed=9),
        # one long document
        dict(name="decode_one_long", op="decode", batch=1, shortest=131000, longest=131000, hq=32, hkv=8, d=128, page=64, dtype="float16", lens_seed=10),
        # a full batch of unequal conversations
        dict(name="decode_ragged_96", op="decode", batch=96, shortest=40, longest=8000, hq=32, hkv=4, d=128, page=64, dtype="bfloat16", lens_seed=11),
        # a k/v head for each q head, head dim 64
        dict(name="decode_heads_48", op="decode", batch=24, shortest=700, longest=3900, hq=48, hkv=48, d=64, page=32, dtype="float16", lens_seed=12),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread evenly over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    op = rng.choice(["prompt", "append", "decode"])
    hkv = rng.choice([1, 2, 3, 4, 6, 8, 16])
    group = rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 12, 16])
    c = dict(op=op, hkv=hkv, d=rng.choice([64, 128]), dtype=rng.choice(["float16", "bfloat16"]), lens_seed=rng.randrange(1 << 30))
    if op == "prompt":
        group = min(group, max(1, 48 // hkv))
        longest = _between(rng, 1, 8192)
        most = 4 * 32 * 4096 ** 2 // (hkv * group * longest ** 2)  # no more pairs than the largest listed case
        while most < 1:
            longest //= 2
            most = 4 * 32 * 4096 ** 2 // (hkv * group * longest ** 2)
        batch = _between(rng, 1, min(most, 200, max(1, 65536 // longest)))
        return dict(c, batch=batch, hq=hkv * group, longest=longest, shortest=rng.choice([1, max(1, longest // 8), longest]),
                    causal=rng.random() < 0.8)
    c["page"] = rng.choice([16, 32, 64, 128])
    if op == "append":
        token = rng.random() < 0.5
        longest = 1 if token else _between(rng, 1, 8192)
        batch = _between(rng, 1, min(256, max(1, 32768 // longest)))
        return dict(c, batch=batch, longest=longest, shortest=rng.choice([1, longest]), held_most=_between(rng, 1, max(1, min(4000, 200000 // batch))))
    longest = _between(rng, 1, 131000)
    batch = _between(rng, 1, max(1, min(256, 100000 * 8 // (longest * hkv))))
    return dict(c, batch=batch, hq=hkv * group, longest=longest, shortest=rng.choice([1, max(1, longest // 4), longest]))


def _lengths(case):
    """The tokens of each sequence (of the call, where a cache holds earlier ones), and how many are held before them."""
    rng = random.Random(case["lens_seed"])
    n = [_between(rng, case["shortest"], case["longest"]) for _ in range(case["batch"])]
    n[rng.randrange(len(n))] = case["longest"]
    held = [rng.choice([0, _between(rng, 1, case["held_most"])]) if case["op"] == "append" else 0 for _ in n]
    if case["op"] == "append" and case["longest"] == 1:
        held = [max(1, h) for h in held]  # a new token follows a prompt
    return n, held


def _up(a, b):
    return -(-a // b)


def _page_table(lens, page, spare, g, dev):
    """Pages in no order, as a long-running program's free list hands them out; -1 behind a sequence's last."""
    need = [_up(n, page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def _held_pages(pages, heads, page, d, g, dev):
    """What earlier tokens left in a cache: values of about unit size, a power of two as the scale of each page and head."""
    e = torch.randint(-8, -5, (pages, heads), generator=g, device=dev)
    bytes_ = torch.empty((pages, heads, page, d), dtype=torch.float8_e4m3fn, device=dev)
    step = max(1, (1 << 26) // (heads * page * d))
    for at in range(0, pages, step):
        x = torch.randn((min(step, pages - at), heads, page, d), generator=g, device=dev)
        x = x * torch.exp2(-e[at:at + step].float())[:, :, None, None]
        bytes_[at:at + step] = x.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return bytes_, torch.exp2(e.float())


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = getattr(torch, case["dtype"])
    n, held = _lengths(case)
    cu = [0]
    for x in n:
        cu.append(cu[-1] + x)
    rows = lambda t, h: torch.randn((t, h, case["d"]), generator=g, device=dev).to(dt)
    s = dict(case=dict(case), longest=max(n), scale=case["d"] ** -0.5)
    if case["op"] == "prompt":
        s.update(q=rows(cu[-1], case["hq"]), k=rows(cu[-1], case["hkv"]), v=rows(cu[-1], case["hkv"]),
                 cu=torch.tensor(cu, dtype=torch.int32, device=dev))
        return s
    total = [a + b for a, b in zip(n, held)]
    table, pages = _page_table(total, case["page"], 3, g, dev)
    kc, ks = _held_pages(pages, case["hkv"], case["page"], case["d"], g, dev)
    vc, vs = _held_pages(pages, case["hkv"], case["page"], case["d"], g, dev)
    s.update(k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, table=table, lens=torch.tensor(total, dtype=torch.int32, device=dev))
    if case["op"] == "append":
        # keys have some large channels, which a page that held few tokens has not seen yet
        loud = 1.0 + 7.0 * (torch.rand((case["hkv"], case["d"]), generator=g, device=dev) < 0.03)
        s.update(k=(rows(cu[-1], case["hkv"]) * loud).to(dt), v=rows(cu[-1], case["hkv"]),
                 cu=None if max(n) == 1 else torch.tensor(cu, dtype=torch.int32, device=dev))
    else:
        s.update(q=rows(case["batch"], case["hq"]))
    return s


# ------------------------------------------------------------------ plain forms
def _softmax(scores, seen):
    scores = scores.masked_fill(~seen, float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True)).masked_fill(~seen, 0.0)
    return p / p.sum(-1, keepdim=True)


def _prompt(s):
    """The pack padded to [batch, longest], every pair of a sequence computed, then the rows packed again."""
    q, k, v, cu = s["q"], s["k"], s["v"], s["cu"].long()
    group = q.shape[1] // k.shape[1]
    at = torch.arange(s["longest"], device=q.device)
    inside = at < (cu[1:] - cu[:-1])[:, None]  # [B, L]
    row = (cu[:-1, None] + at).clamp(max=q.shape[0] - 1)
    spread = lambda t, g: t[row].float().transpose(1, 2).repeat_interleave(g, 1)  # [B, H, L, D]
    seen = inside[:, None, None, :]
    if s["case"]["causal"]:
        seen = seen & (at[:, None] >= at)
    p = _softmax(torch.matmul(spread(q, 1), spread(k, group).transpose(2, 3)) * s["scale"], seen)
    t = torch.arange(q.shape[0], device=q.device)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return torch.matmul(p, spread(v, group))[b, :, t - cu[b]].to(q.dtype)


def _exponents(amax):
    """The smallest e >= -126 with amax <= 448 * 2^e."""
    m, e = torch.frexp(amax)  # amax = m * 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = e - 9 + (m > 0.875).int()
    return torch.where(amax > 0, e, torch.full_like(e, -126)).clamp(min=-126)


def _append_one(cache, scale, x, page_of, slot, opened, slot0):
    """`x` [T, H, D] to (page_of, slot) [T]; opened [B]: each sequence's first page of the call, which holds slot0 [B] rows."""
    pages, heads, page, d = cache.shape
    amax = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).float().abs().amax(-1)  # [T, H]
    most = torch.zeros((pages, heads), device=x.device).scatter_reduce(0, page_of[:, None].expand(-1, heads), amax, "amax")
    e = _exponents(most)
    rows = slot0[:, None] > torch.arange(page, device=x.device)  # [B, page] rows held before
    before = torch.frexp(scale[opened])[1] - 1  # [B, H]
    first = torch.where(slot0[:, None] > 0, torch.maximum(e[opened], before), e[opened])
    e[opened] = first
    old = cache[opened].float()
    again = (old * torch.exp2((before - first).float())[:, :, None, None]).to(cache.dtype)
    grown = rows[:, None, :, None] & (first > before)[:, :, None, None]
    cache[opened] = torch.where(grown, again.float(), old).to(cache.dtype)
    cache[page_of, :, slot] = (x.float() * torch.exp2(-e[page_of].float())[:, :, None]).to(cache.dtype)
    scale[page_of] = torch.exp2(e[page_of].float())


def _append(s):
    x, table, lens = s["k"], s["table"].long(), s["lens"].long()
    batch, page = lens.shape[0], s["k_cache"].shape[2]
    cu = torch.arange(batch + 1, device=x.device) if s["cu"] is None else s["cu"].long()
    t = torch.arange(x.shape[0], device=x.device)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    start = lens - (cu[1:] - cu[:-1])
    pos = start[b] + t - cu[b]
    page_of, opened = table[b, pos // page], table.gather(1, (start // page)[:, None])[:, 0]
    for side in ("k", "v"):
        _append_one(s[side + "_cache"], s[side + "_scale"], s[side], page_of, pos % page, opened, start % page)


def _decode(s):
    q, table, lens = s["q"], s["table"].long().clamp(min=0), s["lens"]
    batch, hq, d = q.shape
    heads, page = s["k_cache"].shape[1:3]
    values = lambda c, sc: (c[table].float() * sc[table][..., None, None]).transpose(1, 2).reshape(batch, heads, -1, d)
    seen = torch.arange(table.shape[1] * page, device=q.device) < lens[:, None]
    qf = q.float().view(batch, heads, hq // heads, d)
    p = _softmax(torch.matmul(qf, values(s["k_cache"], s["k_scale"]).transpose(2, 3)) * s["scale"], seen[:, None, None, :])
    return torch.matmul(p, values(s["v_cache"], s["v_scale"])).view(batch, hq, d).to(q.dtype)


# ------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if own:
        import triton_b200 as tb
        if op == "prompt":
            return tb.attention_varlen(s["q"], s["k"], s["v"], s["cu"], s["case"]["causal"], s["scale"])
        cache = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
        if op == "append":
            tb.kv_cache_append(*cache, s["k"], s["v"], s["table"], s["lens"], s["cu"])
        else:
            return tb.attention_decode(s["q"], *cache, s["table"], s["lens"], s["scale"])
    elif op == "append":
        _append(s)
    else:
        return _prompt(s) if op == "prompt" else _decode(s)
    return {name: s[name] for name in ("k_cache", "v_cache", "k_scale", "v_scale")}


def work(case):
    n, held = _lengths(case)
    d, t = case["d"], sum(n)
    if case["op"] == "prompt":
        pairs = sum(x * (x + 1) // 2 if case["causal"] else x * x for x in n)
        return {"bytes": 2 * d * t * 2 * (case["hq"] + case["hkv"]), "flops": 4 * d * pairs * case["hq"]}
    if case["op"] == "append":
        pages = sum(_up(a + b, case["page"]) - b // case["page"] for a, b in zip(n, held))
        return {"bytes": 2 * case["hkv"] * (3 * d * t + 4 * pages), "flops": 4 * case["hkv"] * d * t}
    pages = sum(_up(x, case["page"]) for x in n)
    return {"bytes": 2 * case["hkv"] * (d * t + 4 * pages) + 4 * case["batch"] * case["hq"] * d, "flops": 4 * d * t * case["hq"]}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    n, held = _lengths(case)
    if case["op"] == "prompt":
        out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        group, at = case["hq"] // case["hkv"], 0
        for x in n:
            for h in range(case["hq"]):
                z = s["q"][at:at + x, h].double() @ s["k"][at:at + x, h // group].double().T * s["scale"]
                if case["causal"]:
                    z = z.masked_fill(torch.ones_like(z, dtype=torch.bool).triu(1), -math.inf)
                out[at:at + x, h] = torch.softmax(z, 1) @ s["v"][at:at + x, h // group].double()
            at += x
        return out
    page = case["page"]
    table = s["table"].cpu().tolist()
    if case["op"] == "decode":
        out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        group = case["hq"] // case["hkv"]
        for b, x in enumerate(n):
            ids = s["table"][b, :_up(x, page)].long()
            k, v = ((s[c + "_cache"][ids].double() * s[c + "_scale"][ids].double()[:, :, None, None]).transpose(0, 1).reshape(case["hkv"], -1, case["d"])[:, :x]
                    for c in "kv")
            z = torch.einsum("hgd,hnd->hgn", s["q"][b].double().view(case["hkv"], group, -1), k) * s["scale"]
            out[b] = torch.einsum("hgn,hnd->hgd", torch.softmax(z, 2), v).reshape(case["hq"], -1)
        return out
    if len(n) * max(n) > 200000:
        return None
    found = {}
    for c in "kv":
        cache, scale, x = (s[name].cpu().double() for name in (c + "_cache", c + "_scale", c))
        at = 0
        for b, (new, old) in enumerate(zip(n, held)):
            done = 0
            while done < new:
                pos = old + done
                p, lo = table[b][pos // page], pos % page
                take = min(page - lo, new - done)
                rows = x[at + done:at + done + take].transpose(0, 1)  # [H, take, D]
                most = rows.abs().amax((1, 2))
                e = torch.ceil(torch.log2(most / E4M3_MAX)).clamp(min=-126)
                e = torch.where(most > E4M3_MAX * 2.0 ** e, e + 1, torch.where(most <= E4M3_MAX * 2.0 ** (e - 1), e - 1, e)).clamp(min=-126)
                unit = 2.0 ** e
                if lo:
                    unit = torch.maximum(unit, scale[p])
                    cache[p, :, :lo] = _nearest(cache[p, :, :lo] * (scale[p] / unit)[:, None, None])
                scale[p] = unit
                cache[p, :, lo:lo + take] = _nearest(rows / unit[:, None, None])
                done += take
            at += new
        found[c + "_cache"], found[c + "_scale"] = cache, scale
    return found


def _nearest(x):
    """The e4m3 value next to x (|x| <= 448), ties to the even one: three bits behind the leading one, steps of 2^-9 below 2^-6."""
    lead = torch.frexp(x)[1] - 1
    step = torch.exp2(lead.clamp(min=-6).double() - 3)
    return torch.round(x / step) * step
