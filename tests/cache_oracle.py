"""The paged cache append and the 8-bit decode attention, one token, page and head at a time
on the CPU, for the tests."""

import math

import torch

from tests import rope_oracle as R

FP8 = torch.float8_e4m3fn


def power_of_two_scale(amax: float) -> float:
    """The smallest power of two s >= 2^-126 with amax <= 448 s."""
    s = 2.0 ** -126
    while amax > 448.0 * s:
        s *= 2
    return s


def encode(x, scale):
    """e4m3 codes of x / scale; values that are not finite become NaN."""
    y = (x.double() / scale).float()
    return torch.where(torch.isfinite(x), y, math.nan).to(FP8)


def rotated_f32(k, table, positions, interleaved):
    """The rotation in float32, every product and sum rounded by itself."""
    y = k.float().clone()
    if table is None or table.shape[1] == 0:
        return y
    inside = (positions >= 0) & (positions < table.shape[0])
    cs = table[torch.where(inside, positions, 0)]
    cos, sin = cs.split(table.shape[1] // 2, -1)
    y = R.rotate(y, cos, sin, interleaved)
    y[~inside] = math.nan
    return y


def append(k, v, k_cache, v_cache, block_table, seq_lens, cu, table, interleaved, k_scale, v_scale):
    """In place on CPU copies; the float32 arithmetic of the definition."""
    pages_total, size = k_cache.shape[:2]
    bounds = list(range(len(seq_lens) + 1)) if cu is None else cu.tolist()
    for b, total in enumerate(seq_lens.tolist()):
        first, n = bounds[b], bounds[b + 1] - bounds[b]
        pos = torch.arange(total - n, total)
        rows = torch.arange(first, first + n)[pos >= 0]
        pos = pos[pos >= 0]
        for x, cache, scale, turn in ((k, k_cache, k_scale, table), (v, v_cache, v_scale, None)):
            if x is None or not len(pos):
                continue
            y = rotated_f32(x[rows], turn, pos, interleaved)
            for lp in range(int(pos[0]) // size, int(pos[-1]) // size + 1):
                here = pos // size == lp
                if lp >= block_table.shape[1]:
                    continue
                page = int(block_table[b, lp])
                if not 0 <= page < pages_total:
                    continue
                at = pos[here] % size
                if cache.dtype != FP8:
                    cache[page, at] = y[here].to(cache.dtype)
                    continue
                for h in range(x.shape[1]):
                    part = y[here][:, h]
                    finite = part[torch.isfinite(part)].abs()
                    need = power_of_two_scale(float(finite.max()) if len(finite) else 0.0)
                    old = float(scale[page, h])
                    now = need if int(at[0]) == 0 else max(old, need)
                    if int(at[0]) and now > old:
                        kept = cache[page, :int(at[0]), h].float() * (old / now)
                        cache[page, :int(at[0]), h] = kept.to(FP8)
                    scale[page, h] = now
                    cache[page, at, h] = encode(part, now)


def attend(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, ids, block, scale):
    """float64 out [B, Hq, D] and lse [B, Hq], and what bounds their float32 errors: per row, the largest
    sum of a logit's absolute terms (each query element counted as the head's largest at least once),
    sum(p |v|) per element, and keys * 448 * max(p v_scale)."""
    batch, hq, dim = q.shape
    groups = k_cache.shape[2]
    size, h = k_cache.shape[1], hq // groups
    out, size_o = (torch.zeros(batch, hq, dim, dtype=torch.float64) for _ in range(2))
    lse = torch.full((batch, hq), -math.inf, dtype=torch.float64)
    size_s, size_w, keys = (torch.zeros(batch, hq, dtype=torch.float64) for _ in range(3))
    for b, n in enumerate(seq_lens.tolist()):
        for g in range(groups):
            chosen = [i for i in dict.fromkeys(ids[b, g].tolist()) if i >= 0 and i * block < n]
            tok = [t for i in chosen for t in range(i * block, min((i + 1) * block, n))
                   if t // size < block_table.shape[1] and 0 <= int(block_table[b, t // size]) < k_cache.shape[0]]
            if not tok:
                continue
            tok = torch.tensor(tok)
            page, row = block_table[b].long()[tok // size], tok % size
            kk = k_cache[page, row, g].float().double() * k_scale[page, g].double()[:, None]
            vs = v_scale[page, g].double()
            vv = v_cache[page, row, g].float().double() * vs[:, None]
            rows = slice(g * h, (g + 1) * h)
            x = q[b, rows].double()
            logit = x @ kk.T * scale
            lse[b, rows] = torch.logsumexp(logit, -1)
            p = torch.exp(logit - lse[b, rows][:, None])
            out[b, rows] = p @ vv
            size_o[b, rows] = p @ vv.abs()
            largest = x.abs().amax(-1, keepdim=True)
            size_s[b, rows] = ((x.abs() @ kk.abs().T + largest * kk.abs().sum(-1)) * abs(scale)).amax(-1)
            size_w[b, rows] = (p * vs).amax(-1) * 448 * len(tok)
            keys[b, rows] = len(tok)
    return out, lse, size_s, size_o, size_w, keys
