"""Cases, plain forms and 64-bit definitions of the operators around the attention:

* ``norm_rope``: RMS norm of every query and key head with the position rotation in the same
  pass (``m3_qk_norm_rope``), forward, and forward with backward;
* ``append``: new keys and values into a paged cache, keys rotated on the way
  (``m3_cache_append``), caches in the inputs' type or in e4m3 with one scale per page and head;
* ``decode8``: one new token per request against its selected blocks of an e4m3 cache
  (``m3_sparse_decode`` with ``k_scale`` / ``v_scale``).

``own`` selects between the plain torch form and the framework's calls; ``prepare`` makes the same state for both.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "fp8": 1}
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
DEV = "cuda"


# --------------------------------------------------------------------------------------- cases
def listed():
    n = dict(op="norm_rope", eps=1e-6, interleaved=False, table=131072)
    a = dict(op="append", interleaved=False, table=131072)
    d = dict(op="decode8", block=128)
    return [
        # one request's decode step: 64 query and 8 key heads, latency only
        dict(n, name="norm_rope decode 1", form="decode", tokens=1, sequences=1, q_heads=64, groups=8, dim=128,
             rotary=64, dtype="bf16"),
        # prefill of the long-context configuration (32768 tokens, 64 / 8 heads)
        dict(n, name="norm_rope prefill 32k", form="prefill", tokens=32768, sequences=1, q_heads=64, groups=8, dim=128,
             rotary=64, dtype="bf16"),
        # a training step on the packed 16-sequence configuration (32 / 8 heads), every dimension rotated
        dict(n, name="norm_rope train 71k packed", form="train", tokens=71168, sequences=16, q_heads=32, groups=8,
             dim=128, rotary=128, dtype="bf16"),
        # the indexer's heads (64 wide, one shared key) in float32, adjacent pairs, odd sequence lengths
        dict(n, name="norm_rope train index", form="train", tokens=8191, sequences=5, q_heads=8, groups=1, dim=64,
             rotary=32, dtype="fp32", interleaved=True),
        # one request's newest key and value into the 8-bit cache
        dict(a, name="append8 decode 1", form="decode", tokens=1, requests=1, past=4000, groups=8, dim=128, rotary=64,
             page=128, cache="fp8", dtype="bf16"),
        # a large decode batch into a 16-bit cache of short pages
        dict(a, name="append decode 256", form="decode", tokens=256, requests=256, past=500, groups=8, dim=128,
             rotary=64, page=16, cache="bf16", dtype="bf16"),
        # prefill of one long request into the 8-bit cache
        dict(a, name="append8 prefill 32k", form="prefill", tokens=32768, requests=1, past=0, groups=8, dim=128,
             rotary=64, page=128, cache="fp8", dtype="bf16"),
        # chunks of several requests that go on in half-filled pages, adjacent pairs
        dict(a, name="append8 chunks", form="prefill", tokens=5000, requests=13, past=900, groups=4, dim=128,
             rotary=128, page=64, cache="fp8", dtype="fp16", interleaved=True),
        # one request, 16 selected blocks: latency
        dict(d, name="decode8 1", requests=1, empty=0, min_len=8192, max_len=8192, q_heads=64, groups=8, dim=128,
             topk=16, page=128, dtype="bf16"),
        # an ordinary decode batch
        dict(d, name="decode8 64", requests=64, empty=0, min_len=1000, max_len=16384, q_heads=64, groups=8, dim=128,
             topk=16, page=128, dtype="bf16"),
        # the largest: long requests in short pages, a cache past 2^32 elements, 4 heads per group
        dict(d, name="decode8 256 long", requests=256, empty=0, min_len=4096, max_len=32768, q_heads=32, groups=8,
             dim=128, topk=32, page=16, dtype="fp16"),
        # narrow heads, 16 per group, float32, requests without a token (a padded batch) and very short ones
        dict(d, name="decode8 ragged", requests=24, empty=3, min_len=1, max_len=5000, q_heads=32, groups=2, dim=64,
             topk=12, page=64, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm_rope", "append", "decode8"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    dim = rng.choice((64, 96, 128, 128, 128, 192))
    groups = rng.choice((1, 2, 4, 8))
    if op == "norm_rope":
        form = rng.choice(("decode", "prefill", "train"))
        tokens = _log(rng, 1, 512) if form == "decode" else _log(rng, 16, 20000)
        return dict(op=op, form=form, tokens=tokens, sequences=min(tokens, rng.randint(1, 12)),
                    q_heads=groups * rng.choice((1, 4, 8)), groups=groups, dim=dim,
                    rotary=rng.choice((dim // 4, dim // 2, dim)), dtype=dtype, interleaved=rng.random() < 0.3,
                    eps=rng.choice((1e-6, 1e-5)), table=131072)
    if op == "append":
        form = rng.choice(("decode", "prefill"))
        requests = _log(rng, 1, 300) if form == "decode" else rng.randint(1, 20)
        tokens = requests if form == "decode" else _log(rng, requests, 20000)
        return dict(op=op, form=form, tokens=tokens, requests=requests, past=_log(rng, 1, 2000), groups=groups,
                    dim=dim, rotary=rng.choice((dim // 4, dim // 2, dim)), page=rng.choice((16, 32, 64, 128)),
                    cache=rng.choice((dtype, "fp8", "fp8")), dtype=dtype, interleaved=rng.random() < 0.3, table=131072)
    max_len = _log(rng, 100, 32768)
    return dict(op=op, requests=_log(rng, 1, 128), empty=rng.choice((0, 0, 1)), min_len=max(1, max_len // 10),
                max_len=max_len, q_heads=groups * rng.choice((2, 4, 8, 16)), groups=groups, dim=dim,
                block=rng.choice((64, 128, 128)), topk=rng.randint(1, 32), page=rng.choice((16, 32, 64, 128)),
                dtype=dtype)


def _split(total, parts, rng):
    """`parts` positive lengths that sum to `total`."""
    cuts = sorted(rng.sample(range(1, total), parts - 1)) if parts > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def _rng(case):
    return random.Random("%s" % sorted((k, str(v)) for k, v in case.items() if k != "name"))


def _lengths(case):
    """Context lengths of a decode batch, the same for every seed (so that work() can count them)."""
    rng = _rng(case)
    lens = [rng.randint(case["min_len"], case["max_len"]) for _ in range(case["requests"])]
    for b in range(min(case["empty"], len(lens) - 1)):
        lens[(7 * b + 1) % len(lens)] = 0
    return lens


def _new_and_past(case):
    """New tokens and earlier tokens of each request of an append."""
    rng = _rng(case)
    new = _split(case["tokens"], case["requests"], rng) if case["form"] == "prefill" else [1] * case["requests"]
    return new, [rng.randint(0, case["past"]) for _ in new]


# --------------------------------------------------------------------------------------- inputs
def _table(rows, rotary):
    """cos and sin of position * base^(-2i / rotary), the angles in 64 bits: [rows, rotary] (cos half, sin half)."""
    inv = 5e6 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=DEV) / rotary)
    ang = torch.arange(rows, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.cat((ang.cos(), ang.sin()), dim=-1).float()


def _pages(lens, page, gen):
    """A block table over randomly ordered physical pages, some of them unused."""
    per = [(n + page - 1) // page for n in lens]
    total = sum(per) + 3
    order = torch.randperm(total, generator=gen, device=DEV).to(torch.int32)
    first = torch.tensor([0] + per, device=DEV).cumsum(0)[:-1]
    at = torch.arange(max(max(per), 1), device=DEV)
    own_page = at < torch.tensor(per, device=DEV)[:, None]
    return torch.where(own_page, order[(first[:, None] + at).clamp(max=total - 1)], 0).to(torch.int32), total


def _pow2(amax):
    """The smallest power of two s with amax <= 448 s (2^-126 at least)."""
    m, e = torch.frexp(amax)
    return torch.ldexp(torch.ones_like(amax), (e - 9 + (m > 0.875).to(e.dtype)).clamp(min=-126))


def _quantised_cache(pages, page, groups, dim, gen):
    """An e4m3 cache of unit-variance values with uneven channels, and its scales, filled some pages at a time."""
    codes = torch.empty(pages, page, groups, dim, dtype=FP8, device=DEV)
    scale = torch.empty(pages, groups, device=DEV)
    gain = (0.4 * torch.randn(groups, dim, generator=gen, device=DEV)).exp()
    step = max(1, 2 ** 28 // (page * groups * dim))
    for i in range(0, pages, step):
        x = torch.randn(min(step, pages - i), page, groups, dim, generator=gen, device=DEV) * gain
        s = _pow2(x.abs().amax(dim=(1, 3)))
        codes[i:i + step] = (x / s[:, None, :, None]).to(FP8)
        scale[i:i + step] = s
    return codes, scale


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = _rng(case)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    if case["op"] == "norm_rope":
        t, hq, g, d = case["tokens"], case["q_heads"], case["groups"], case["dim"]
        # q and k lie side by side, as one projection leaves them
        qkv = (randn(t, (hq + 2 * g) * d) * (0.3 * randn(t, 1)).exp()).to(dt)
        q = qkv[:, :hq * d].view(t, hq, d)
        k = qkv[:, hq * d:(hq + g) * d].view(t, g, d)
        wq, wk = ((1 + 0.2 * randn(d)).to(dt) for _ in range(2))
        s = dict(case, q=q, k=k, wq=wq, wk=wk, rope=_table(case["table"], case["rotary"]))
        if case["form"] == "decode":
            s["positions"] = torch.randint(0, case["table"], (t,), generator=gen, device=DEV, dtype=torch.int32)
        else:
            lens = _split(t, case["sequences"], rng)
            s["bounds"] = [0]
            for n in lens:
                s["bounds"].append(s["bounds"][-1] + n)
            s["cu"] = torch.tensor(s["bounds"], dtype=torch.int32, device=DEV)
        if case["form"] == "train":
            for x in (q, k, wq, wk):
                x.requires_grad_()
            s["gq"], s["gk"] = randn(t, hq, d).to(dt), randn(t, g, d).to(dt)
        return s

    if case["op"] == "append":
        new, past = _new_and_past(case)
        t, g, d, page = case["tokens"], case["groups"], case["dim"], case["page"]
        lens = [a + b for a, b in zip(new, past)]
        table, pages = _pages(lens, page, gen)
        cu = torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32)
        s = dict(case, k=randn(t, g, d).to(dt), v=(1.5 * randn(t, g, d)).to(dt), block_table=table,
                 cu=cu if case["form"] == "prefill" else None, rope=_table(case["table"], case["rotary"]),
                 seq_lens=torch.tensor(lens, dtype=torch.int32, device=DEV), k_scale=None, v_scale=None)
        if case["cache"] == "fp8":
            s["k_cache"], s["k_scale"] = _quantised_cache(pages, page, g, d, gen)
            s["v_cache"], s["v_scale"] = _quantised_cache(pages, page, g, d, gen)
        else:
            s["k_cache"], s["v_cache"] = (randn(pages, page, g, d).to(DTYPES[case["cache"]]) for _ in range(2))
        return s

    lens = _lengths(case)
    b, g, d, block = case["requests"], case["groups"], case["dim"], case["block"]
    table, pages = _pages(lens, case["page"], gen)
    k_cache, k_scale = _quantised_cache(pages, case["page"], g, d, gen)
    v_cache, v_scale = _quantised_cache(pages, case["page"], g, d, gen)
    seq_lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
    # a selection as top-k leaves it: the newest block, then others of the request's, -1 behind them
    blocks = max(1, (max(lens) + block - 1) // block)
    score = torch.rand(b, g, blocks, generator=gen, device=DEV)
    last = (seq_lens - 1).div(block, rounding_mode="floor")[:, None, None]
    at = torch.arange(blocks, device=DEV)
    score = torch.where(at == last, math.inf, torch.where(at > last, -math.inf, score))
    top = score.topk(min(case["topk"], blocks), dim=-1)
    ids = torch.full((b, g, case["topk"]), -1, dtype=torch.int32, device=DEV)
    ids[..., :top.indices.shape[-1]] = torch.where(top.values == -math.inf, -1, top.indices).to(torch.int32)
    return dict(case, q=randn(b, case["q_heads"], d).to(dt), k_cache=k_cache, v_cache=v_cache, k_scale=k_scale,
                v_scale=v_scale, block_table=table, seq_lens=seq_lens, ids=ids)


# --------------------------------------------------------------------------------------- plain forms
def _rotate(x, cs, interleaved, sign=1.0):
    """Rotates the first dims of x [T, H, D] by the rows cs [T, R] of the table (sign -1: back)."""
    r = cs.shape[-1]
    c, s = cs[:, None, :r // 2], cs[:, None, r // 2:] * sign
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack((a * c - b * s, b * c + a * s), dim=-1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat((a * c - b * s, b * c + a * s), dim=-1)
    return torch.cat((y, x[..., r:]), dim=-1)


def _positions(s):
    if s["form"] == "decode":
        return s["positions"].long()
    t = torch.arange(s["tokens"], device=DEV)
    return t - s["cu"][torch.searchsorted(s["cu"], t, right=True) - 1]


def _norm_rope(x, w, cs, s, grad=None):
    """The output, or with `grad` the gradients of x and w."""
    f = x.detach().float()
    r = torch.rsqrt(f.square().mean(-1, keepdim=True) + s["eps"])
    hat = f * r
    if grad is None:
        return _rotate(hat * w.detach().float(), cs, s["interleaved"]).to(x.dtype)
    back = _rotate(grad.float(), cs, s["interleaved"], -1.0)
    dw = (back * hat).sum((0, 1))
    u = back * w.detach().float()
    return (r * (u - hat * (u * hat).mean(-1, keepdim=True))).to(x.dtype), dw.to(w.dtype)


def _places(s):
    """Of each new token: its position, physical page and row of the page."""
    req = torch.arange(s["tokens"], device=DEV)
    end = req + 1
    if s["cu"] is not None:
        at = torch.searchsorted(s["cu"], req, right=True) - 1
        req, end, t = at, s["cu"][at + 1], req
    else:
        t = req
    pos = (s["seq_lens"][req] - (end - t)).long()
    return pos, s["block_table"][req, pos // s["page"]].long(), pos % s["page"]


def _append(x, cache, scale, page, row):
    if scale is None:
        cache[page, row] = x.to(cache.dtype)
        return
    need = torch.zeros_like(scale).index_reduce_(0, page, x.abs().amax(-1), "amax")
    first = torch.full((scale.shape[0],), cache.shape[1], device=DEV).index_reduce_(0, page, row, "amin")
    need = _pow2(need)
    grown = torch.where((first == 0)[:, None], need, torch.maximum(scale, need))
    touched = torch.unique(page)
    old = cache[touched].float() * (scale[touched] / grown[touched])[:, None, :, None]
    earlier = torch.arange(cache.shape[1], device=DEV) < first[touched][:, None]
    bits = cache.view(torch.uint8)
    bits[touched] = torch.where(earlier[:, :, None, None], old.to(FP8).view(torch.uint8), bits[touched])
    scale[touched] = grown[touched]
    bits[page, row] = (x / scale[page][:, :, None]).to(FP8).view(torch.uint8)


def _decode8(s):
    b, g, k = s["ids"].shape
    block, page_size, d = s["block"], s["page"], s["dim"]
    ids, n = s["ids"].long(), k * block
    pos = (s["seq_lens"].long() - 1)[:, None, None, None]
    again = ((ids[..., :, None] == ids[..., None, :]).tril(-1)).any(-1)
    tok = ids[..., None] * block + torch.arange(block, device=DEV)
    seen = ((ids >= 0) & ~again)[..., None] & (tok <= pos)
    tok, seen = torch.where(seen, tok, 0).view(b, g * n), seen.view(b, g, n)
    page = s["block_table"].long().gather(1, tok // page_size).view(b, g, n)
    head = torch.arange(g, device=DEV)[None, :, None]
    row = (page * page_size + tok.view(b, g, n) % page_size) * g + head

    def values(cache, scale):
        x = cache.view(torch.uint8).view(-1, d)[row].view(FP8).float() * scale[page, head][..., None]
        return torch.where(seen[..., None], x, 0.0)

    q = s["q"].float().view(b, g, -1, d)
    logit = (q @ values(s["k_cache"], s["k_scale"]).transpose(-1, -2)) * d ** -0.5
    logit = torch.where(seen[:, :, None], logit, -math.inf)
    top = logit.amax(-1, keepdim=True)
    p = torch.exp(logit - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = (p @ values(s["v_cache"], s["v_scale"])) / torch.where(total == 0, 1.0, total)
    return out.reshape(b, -1, d).to(s["q"].dtype), (top + torch.log(total)).reshape(b, -1)


def run(state):
    s = state
    if own:
        return _own(s)
    if s["op"] == "norm_rope":
        cs = s["rope"][_positions(s)]
        out = [_norm_rope(s["q"], s["wq"], cs, s), _norm_rope(s["k"], s["wk"], cs, s)]
        if s["form"] == "train":
            dq, dwq = _norm_rope(s["q"], s["wq"], cs, s, s["gq"])
            dk, dwk = _norm_rope(s["k"], s["wk"], cs, s, s["gk"])
            out += [dq, dk, dwq, dwk]
        return out
    if s["op"] == "append":
        pos, page, row = _places(s)
        _append(_rotate(s["k"].float(), s["rope"][pos], s["interleaved"]), s["k_cache"], s["k_scale"], page, row)
        _append(s["v"].float(), s["v_cache"], s["v_scale"], page, row)
        return [s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]]
    return _decode8(s)


def _own(s):
    import msa_triton_b200 as msa

    if s["op"] == "norm_rope":
        if s["form"] == "decode":
            return list(msa.m3_qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["rope"], positions=s["positions"],
                                            eps=s["eps"], interleaved=s["interleaved"]))
        prepared = msa.prepare_batch(s["cu"], bounds=s["bounds"])
        out = msa.m3_qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["rope"], s["cu"], eps=s["eps"],
                                  interleaved=s["interleaved"], prepared=prepared)
        if s["form"] != "train":
            return list(out)
        grads = torch.autograd.grad(out, (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"]))
        return [x.detach() for x in out] + list(grads)
    if s["op"] == "append":
        msa.m3_cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["block_table"], s["seq_lens"],
                            cu_seqlens=s["cu"], rope_table=s["rope"], interleaved=s["interleaved"],
                            k_scale=s["k_scale"], v_scale=s["v_scale"])
        return [s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]]
    return msa.m3_sparse_decode(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["seq_lens"], s["ids"],
                                block_size=s["block"], k_scale=s["k_scale"], v_scale=s["v_scale"], return_lse=True)


# --------------------------------------------------------------------------------------- work
def work(case):
    c = case
    size = SIZE[c["dtype"]]
    if c["op"] == "norm_rope":
        rows = c["tokens"] * (c["q_heads"] + c["groups"])
        one = rows * c["dim"] * size
        seen = c["tokens"] * c["rotary"] * 4
        if c["form"] != "train":
            return {"bytes": 2 * one + seen, "flops": rows * (5 * c["dim"] + 3 * c["rotary"])}
        # x, its gradient's source and the two results of each row
        return {"bytes": 4 * one + seen, "flops": rows * (16 * c["dim"] + 6 * c["rotary"])}
    if c["op"] == "append":
        values = c["tokens"] * c["groups"] * c["dim"]
        pages = sum((past + new - 1) // c["page"] - past // c["page"] + 1 for new, past in zip(*_new_and_past(c)))
        scales = 2 * 4 * pages * c["groups"] if c["cache"] == "fp8" else 0
        return {"bytes": 2 * values * (size + SIZE[c["cache"]]) + c["tokens"] * c["rotary"] * 4 + scales,
                "flops": c["tokens"] * c["groups"] * 3 * c["rotary"] + (4 * values if c["cache"] == "fp8" else 0)}
    keys = 0
    for n in _lengths(c):
        if n:
            blocks = min(c["topk"], (n + c["block"] - 1) // c["block"])
            keys += (blocks - 1) * c["block"] + (n - 1) % c["block"] + 1
    keys *= c["groups"]
    rows = c["requests"] * c["q_heads"]
    return {"bytes": 2 * keys * c["dim"] + 2 * rows * c["dim"] * size + 4 * rows,
            "flops": 4 * keys * c["dim"] * c["q_heads"] // c["groups"]}


# --------------------------------------------------------------------------------------- 64 bits
def _turned(x, cos, sin, interleaved):
    """R(p) x in 64 bits: pair i of x [T, H, D] as the complex number a + ib, times cos + i sin."""
    half = cos.shape[-1]
    pairs = x[..., :2 * half]
    pairs = pairs.unflatten(-1, (half, 2)) if interleaved else pairs.unflatten(-1, (2, half)).transpose(-1, -2)
    z = torch.view_as_complex(pairs.contiguous()) * torch.complex(cos, sin)[:, None]
    y = torch.view_as_real(z)
    y = (y if interleaved else y.transpose(-1, -2)).flatten(-2)
    return torch.cat((y, x[..., 2 * half:]), -1)


def _exact_norm_rope(s):
    pos = torch.cat([torch.arange(n, device=DEV) for n in
                     (b - a for a, b in zip(s["bounds"], s["bounds"][1:]))]) if "bounds" in s else s["positions"].long()
    cos, sin = s["rope"][pos].double().chunk(2, -1)
    outs, dxs, dws = [], [], []
    for x, w, g in ((s["q"], s["wq"], s.get("gq")), (s["k"], s["wk"], s.get("gk"))):
        ys, gs, dw = [], [], torch.zeros(s["dim"], dtype=torch.float64, device=DEV)
        w = w.detach().double()
        for i in range(0, x.shape[0], 4096):
            at = slice(i, i + 4096)
            f = x.detach()[at].double()
            rms = (f.pow(2).sum(-1, keepdim=True) / s["dim"] + s["eps"]).sqrt()
            ys.append(_turned(f / rms * w, cos[at], sin[at], s["interleaved"]))
            if g is not None:
                back = _turned(g[at].double(), cos[at], -sin[at], s["interleaved"])
                dw += torch.einsum("thd,thd->d", back, f / rms)
                u = back * w
                gs.append(u / rms - f * (u * f).sum(-1, keepdim=True) / (s["dim"] * rms ** 3))
        outs.append(torch.cat(ys))
        if g is not None:
            dxs.append(torch.cat(gs))
            dws.append(dw)
    return outs + dxs + dws


def _exact_codes(x):
    """The e4m3 values nearest to x (64 bits, |x| <= 448), ties to the even one."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _exact_scale(amax):
    """The smallest power of two s, at least 2^-126, with amax <= 448 s."""
    if amax == 0:
        return 2.0 ** -126
    s = 2.0 ** math.floor(math.log2(amax / FP8_MAX))
    return max(s if FP8_MAX * s >= amax else 2 * s, 2.0 ** -126)


def _exact_append(s):
    new, past = _new_and_past({k: s[k] for k in s["case_keys"]})
    out = []
    for key, x in (("k", s["k"].double()), ("v", s["v"].double())):
        cache, scale = s[key + "_cache"].double(), s[key + "_scale"]
        scale = scale.double() if scale is not None else None
        start = 0
        for b, (n, p) in enumerate(zip(new, past)):
            y = x[start:start + n]
            if key == "k":
                cos, sin = s["rope"][p:p + n].double().chunk(2, -1)
                y = _turned(y, cos, sin, s["interleaved"])
            for lp in range(p // s["page"], (p + n - 1) // s["page"] + 1):
                lo, hi = max(p, lp * s["page"]), min(p + n, (lp + 1) * s["page"])
                page, row, part = int(s["table_host"][b][lp]), lo - lp * s["page"], y[lo - p:hi - p]
                if scale is None:
                    cache[page, row:row + hi - lo] = part
                    continue
                need = torch.tensor([_exact_scale(m) for m in part.abs().amax((0, 2)).tolist()],
                                    dtype=torch.float64, device=DEV)
                grown = torch.maximum(scale[page], need) if row else need
                if row:
                    cache[page, :row] = _exact_codes(cache[page, :row] * (scale[page] / grown)[:, None])
                scale[page] = grown
                cache[page, row:row + hi - lo] = _exact_codes(part / grown[:, None])
            start += n
        out.append((cache, scale))
    return [out[0][0], out[1][0], out[0][1], out[1][1]]


def _exact_decode8(s, lens):
    outs, lses = [], []
    g, d, h = s["groups"], s["dim"], s["q_heads"] // s["groups"]
    for b, n in enumerate(lens):
        out = torch.zeros(g, h, d, dtype=torch.float64, device=DEV)
        lse = torch.full((g, h), -math.inf, dtype=torch.float64, device=DEV)
        if n:
            at = torch.arange(n, device=DEV)
            page, row = s["block_table"][b].long()[at // s["page"]], at % s["page"]
            for i in range(g):
                mine = torch.isin(at // s["block"], s["ids"][b, i])
                p, r = page[mine], row[mine]
                k = s["k_cache"].view(torch.uint8)[p, r, i].view(FP8).double() * s["k_scale"][p, i].double()[:, None]
                v = s["v_cache"].view(torch.uint8)[p, r, i].view(FP8).double() * s["v_scale"][p, i].double()[:, None]
                logit = s["q"][b, i * h:(i + 1) * h].double() @ k.T / math.sqrt(d)
                lse[i] = torch.logsumexp(logit, -1)
                out[i] = torch.exp(logit - lse[i][:, None]) @ v
        outs.append(out.view(-1, d))
        lses.append(lse.view(-1))
    return torch.stack(outs), torch.stack(lses)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm_rope":
        return _exact_norm_rope(s)
    if case["op"] == "append":
        return _exact_append(dict(s, case_keys=list(case), table_host=s["block_table"].tolist()))
    return _exact_decode8(s, _lengths(case))
