"""m3_sparse_decode over an 8-bit cache against a float64 attention on the values the cache stands for.

Tolerance, by first-order error analysis of the kernel's float32 arithmetic (u = 2^-24), with the sizes
that the oracle returns:
  * a logit (natural units): D products and sums, q's and the scales' factors, the softmax's subtraction:
    (D + 32) u of its absolute terms; elements of q far below the head's largest are kept to 2^-25 of
    that one (counted in the terms);
  * a weight: the logit's error twice (numerator and sum), exp2's 2 ulp, one rounding to fp16 (half of its
    relative step 2^-10, so 2^-11: an 11-bit significand 1.xxxxxxxxxx is off by at most 2^-11 of a number in [1, 2);
    the two-term float32 form rounds a rest of at most 2^-11 once more, 2^-22), and 2^-25 of the largest weight
    below fp16's normal range;
  * sums over the keys: one u per key, and the merges (64);
  * the output's own rounding, half a step."""

import pytest
import torch

from msa_triton_b200 import m3_cache_append, m3_sparse_decode
from tests import cache_oracle as C
from tests import rope_oracle as R

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
NAN_CODE = 0x7F


def make_cache(pages, size, heads, dim, gen, head_major=False, spread=0.0):
    x = torch.randn(pages, size, heads, dim, generator=gen)
    x *= torch.exp(spread * torch.randn(pages, 1, heads, 1, generator=gen))
    scale = x.abs().amax((1, 3)) / 448 * (1 + 0.3 * torch.rand(pages, heads, generator=gen))
    codes = (x / scale[:, None, :, None]).to(FP8)
    if head_major:
        codes = codes.view(torch.uint8).transpose(1, 2).contiguous().view(FP8).transpose(1, 2)
    return codes, scale


def make_case(lens, heads, ratio, dim, block, size, topk, dtype, seed=0, head_major=False, spread=0.0):
    gen = torch.Generator().manual_seed(seed)
    per = [max(1, -(-n // size)) for n in lens]
    total = sum(per) + 2
    order = torch.randperm(total, generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(per)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    k, ks = make_cache(total, size, heads, dim, gen, head_major, spread)
    v, vs = make_cache(total, size, heads, dim, gen, head_major, spread)
    # what lies behind a request's last token, and on no request's page, must not matter
    for x in (k, v):
        bits = x.view(torch.uint8)
        for b, n in enumerate(lens):
            bits[int(table[b, per[b] - 1]), n - (per[b] - 1) * size:] = NAN_CODE
        bits[order[at:].long()] = NAN_CODE
    q = (torch.randn(len(lens), heads * ratio, dim, generator=gen)
         * torch.exp(torch.randn(len(lens), heads * ratio, 1, generator=gen))).to(dtype)
    ids = torch.full((len(lens), heads, topk), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        blocks = -(-n // block)
        for g in range(heads):
            if blocks:
                pick = torch.randperm(blocks, generator=gen)[:topk]
                if blocks - 1 not in pick:
                    pick[0] = blocks - 1
                ids[b, g, :len(pick)] = pick.to(torch.int32)
    return q, k, v, ks, vs, table, torch.tensor(lens, dtype=torch.int32), ids


def run(case, block, dev, **kw):
    q, k, v, ks, vs, table, lens, ids = case

    def cache(x):
        if x.is_contiguous():
            return x.to(dev)
        return x.view(torch.uint8).transpose(1, 2).contiguous().to(dev).view(FP8).transpose(1, 2)

    return m3_sparse_decode(q.to(dev), cache(k), cache(v), table.to(dev), lens.to(dev), ids.to(dev), block_size=block,
                            return_lse=True, k_scale=ks.to(dev), v_scale=vs.to(dev), **kw)


def check(case, block, got, scale=None):
    q, k, v, ks, vs, table, lens, ids = case
    dim, dtype = q.shape[2], q.dtype
    eff = dim ** -0.5 if scale is None else scale
    out, lse, size_s, size_o, size_w, keys = C.attend(q, k, v, ks, vs, table, lens, ids, block, eff)
    got_out, got_lse = got[0].cpu().double(), got[1].cpu().double()
    assert got[0].dtype == dtype and got[1].dtype == torch.float32
    assert torch.equal(torch.isneginf(got_lse), torch.isneginf(lse))
    logit = (dim + 32) * R.U * size_s
    weight = 2 * logit + 2.0 ** -21 + (2.0 ** -22 if dtype == torch.float32 else 2.0 ** -11) + (keys + 64) * R.U
    bound = (R.half_step(dtype) * out.abs() * (1 + 2.0 ** -6) + weight[..., None] * size_o
             + 2.0 ** -25 * size_w[..., None] + 2.0 ** -25 * (dtype == torch.float16))
    off = (got_out - out).abs()
    assert not torch.isnan(got_out).any()
    assert float((off - bound).max()) <= 0, f"out: {float((off / bound.clamp(min=1e-300)).max())} of the bound"
    fin = torch.isfinite(lse)
    lse_bound = logit + 2.0 ** -21 + (keys + 64) * R.U + 2 * R.U * lse.abs()
    assert ((got_lse - lse).abs()[fin] <= lse_bound[fin]).all(), "lse"


CASES = [
    # lens, groups, heads per group, D, block, page, top-k, dtype
    ([1, 130, 700, 2049, 300], 2, 8, 128, 128, 128, 4, torch.bfloat16),
    ([0, 5, 64, 0, 333], 2, 4, 128, 128, 16, 6, torch.float16),
    ([5000], 1, 8, 128, 128, 64, 16, torch.bfloat16),
    ([900, 31], 4, 16, 128, 64, 32, 9, torch.bfloat16),
    ([700, 33], 2, 5, 128, 128, 128, 3, torch.float32),
    ([257, 1], 2, 13, 128, 128, 128, 3, torch.float32),
    ([200, 450, 32], 3, 16, 64, 64, 64, 12, torch.float32),
    ([300, 77], 1, 1, 64, 128, 16, 4, torch.bfloat16),
    ([300, 77], 2, 10, 64, 128, 16, 4, torch.float16),
    ([400, 12], 2, 8, 256, 128, 128, 4, torch.bfloat16),
    ([400, 12], 1, 12, 256, 128, 64, 4, torch.float32),
    ([260], 2, 12, 256, 128, 64, 4, torch.float16),
    ([260], 2, 2, 256, 128, 64, 4, torch.float32),
    ([340, 9], 2, 8, 192, 128, 128, 4, torch.bfloat16),
    ([340, 9], 2, 6, 96, 128, 32, 4, torch.float16),
    ([150], 1, 40, 128, 128, 128, 2, torch.bfloat16),      # more heads than one tile of rows
    ([3000], 1, 4, 128, 16, 16, 70, torch.bfloat16),       # short blocks, more ids than lanes
    ([500, 120], 2, 8, 128, 100, 48, 5, torch.bfloat16),   # blocks and pages that share no boundary
    ([90, 13], 2, 3, 80, 7, 300, 9, torch.float32),
    ([90, 13], 2, 3, 27, 16, 5, 4, torch.bfloat16),        # rows off the 16-byte alignment
    ([70, 3], 2, 2, 1, 32, 1, 2, torch.float32),
    ([130], 1, 2, 130, 64, 16, 2, torch.float16),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[1]}x{c[2]}x{c[3]}b{c[4]}p{c[5]}k{c[6]}-{c[7]}")
@pytest.mark.parametrize("head_major", [False, True])
def test_decode8_matches_fp64(case, head_major, cuda_device):
    *sizes, dtype = case
    made = make_case(*sizes, dtype, seed=sum(case[0]), head_major=head_major)
    check(made, sizes[4], run(made, sizes[4], cuda_device))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scales_far_apart(dtype, cuda_device):
    """Pages whose values differ by many powers of two, pages of zeros with the smallest scale."""
    made = make_case([900, 333], 2, 8, 128, 128, 16, 7, dtype, seed=4, spread=6.0)
    q, k, v, ks, vs, *_ = made
    k.view(torch.uint8)[::5], v.view(torch.uint8)[::5] = 0, 0
    vs[::5] = 2.0 ** -126
    ks[::7] *= 0.01
    q *= 0.05
    check(made, 128, run(made, 128, cuda_device))
    check(made, 128, run(made, 128, cuda_device, scale=-0.3), scale=-0.3)
    vs[:] = 0  # every value zero
    out, lse = run(made, 128, cuda_device)
    assert torch.count_nonzero(out) == 0 and torch.isfinite(lse).all()


def test_repeated_empty_and_future_selections(cuda_device):
    made = make_case([300, 129], 2, 8, 128, 128, 64, 40, torch.bfloat16, seed=3)
    ids = made[-1]
    ids[:] = -1
    ids[0, 0, :4] = torch.tensor([2, 2, 0, 9])
    ids[0, 0, 35:] = torch.tensor([0, 1, 2, 1, 2 ** 31 - 1])  # repeats of the first 32 ids
    ids[0, 1, 5], ids[1, 0, 39] = 5, 0
    out, lse = run(made, 128, cuda_device)
    check(made, 128, (out, lse))
    assert torch.count_nonzero(out[0, 8:]) == 0 and torch.isneginf(lse[0, 8:]).all()
    assert torch.count_nonzero(out[1, 8:]) == 0 and torch.isneginf(lse[1, 8:]).all()
    empty = tuple(x[..., :0] if i == 7 else x for i, x in enumerate(made))
    out, lse = run(empty, 128, cuda_device)
    assert torch.count_nonzero(out) == 0 and torch.isneginf(lse).all()


def test_bad_pages_and_short_tables_are_not_attended(cuda_device):
    made = list(make_case([300, 400, 50], 2, 8, 128, 128, 64, 4, torch.bfloat16, seed=5))
    made[5][0, 1], made[5][1, 0], made[5][2, 0] = -7, 10 ** 6, made[1].shape[0]
    made[5] = made[5][:, :5].contiguous()
    check(made, 128, run(made, 128, cuda_device))


def test_nan_in_attended_places_shows(cuda_device):
    made = make_case([200, 200], 2, 8, 128, 128, 64, 2, torch.bfloat16, seed=6)
    q, k, v, *_ , table, lens, ids = made
    page = int(table[0, 0])
    k.view(torch.uint8)[page, 3, 0, 7] = NAN_CODE
    v.view(torch.uint8)[page, 3, 1, 7] = NAN_CODE
    out, lse = run(made, 128, cuda_device)
    assert torch.isnan(out[0, :8]).all() and torch.isnan(lse[0, :8]).all()
    bad = torch.isnan(out[0, 8:])
    assert bad[:, 7].all() and int(bad.sum()) == 8 and torch.isfinite(lse[0, 8:]).all()
    assert torch.isfinite(out[1].float()).all()


def test_views_streams_and_repeats(cuda_device):
    """Strided q, ids, lengths and block tables; another stream; the same bits every time."""
    dev = cuda_device
    made = make_case([700, 1000, 64], 2, 8, 128, 128, 64, 6, torch.bfloat16, seed=7)
    q, k, v, ks, vs, table, lens, ids = (x.to(dev) for x in made)
    want = run(made, 128, dev)
    wide = torch.zeros(3, 16, 200, dtype=torch.bfloat16, device=dev)
    wide[..., 8:136] = q
    args = (wide[..., 8:136], k, v, torch.stack((table, table), 2)[..., 1], torch.stack((lens, lens), 1)[:, 1],
            torch.stack((ids, ids), 3)[..., 0])
    got = m3_sparse_decode(*args, block_size=128, return_lse=True, k_scale=ks, v_scale=vs)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = run(made, 128, dev)
    torch.cuda.current_stream(dev).wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_memory_at_odd_addresses(cuda_device):
    """Dense tensors that begin off the 16-byte alignment: q, the caches, or both."""
    dev = cuda_device
    made = make_case([500, 40], 2, 8, 128, 128, 64, 3, torch.bfloat16, seed=13)
    q, k, v, ks, vs, table, lens, ids = (x.to(dev) for x in made)

    def shifted(x, by):
        base = torch.empty(x.numel() + by, dtype=torch.uint8 if x.dtype == FP8 else x.dtype, device=dev)
        y = base[by:].view(x.dtype) if x.dtype == FP8 else base[by:]
        y = y.view(x.shape)
        (y.view(torch.uint8) if x.dtype == FP8 else y).copy_(x.view(torch.uint8) if x.dtype == FP8 else x)
        return y

    for dq, dk, dv in ((1, 0, 0), (0, 4, 0), (0, 0, 1), (3, 8, 5)):
        got = m3_sparse_decode(shifted(q, dq), shifted(k, dk), shifted(v, dv), table, lens, ids, return_lse=True,
                               k_scale=ks, v_scale=vs)
        check(made, 128, got)


def test_two_captured_steps_share_nothing(cuda_device):
    """Two captured graphs replayed on two streams at once, lengths and selections changed in between."""
    dev = cuda_device
    cases = [make_case([2000, 900, 3], 4, 8, 128, 128, 64, 16, torch.bfloat16, seed=s) for s in (8, 9)]
    graphs, held, inputs = [], [], []
    for case in cases:
        q, k, v, ks, vs, table, lens, ids = (x.to(dev) for x in case)
        inputs.append((lens, ids))
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            m3_sparse_decode(q, k, v, table, lens, ids, k_scale=ks, v_scale=vs)
        torch.cuda.current_stream(dev).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append((q, k, v, table, ks, vs, m3_sparse_decode(q, k, v, table, lens, ids, return_lse=True,
                                                                  k_scale=ks, v_scale=vs)))
        graphs.append(graph)
    for case, (lens, ids) in zip(cases, inputs):
        case[6][:] = torch.tensor([1500, 0, 2])
        case[7][:] = torch.where(case[7] < 12, case[7], -1)
        lens.copy_(case[6])
        ids.copy_(case[7])
    streams = [torch.cuda.Stream(dev) for _ in graphs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(dev))
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for case, h in zip(cases, held):
        check(case, 128, h[-1])


def test_cache_past_32_bits(cuda_device):
    """A cache of more than 2^32 bytes, the request's pages at its end, appended and read."""
    dev = cuda_device
    gen = torch.Generator().manual_seed(11)
    heads, dim, size = 8, 128, 128
    pages = 2 ** 32 // (heads * dim * size) + 40
    k_cache = torch.zeros(pages, size, heads, dim, dtype=FP8, device=dev)
    scale = [torch.ones(pages, heads, device=dev) for _ in range(2)]
    v_cache = torch.zeros_like(k_cache)
    n = 900
    k, v = (torch.randn(n, heads, dim, generator=gen).bfloat16() for _ in range(2))
    table = torch.arange(pages - 1, pages - 9, -1, dtype=torch.int32).view(1, 8)
    lens, cu = torch.tensor([n], dtype=torch.int32), torch.tensor([0, n], dtype=torch.int32)
    m3_cache_append(k.to(dev), v.to(dev), k_cache, v_cache, table.to(dev), lens.to(dev), cu_seqlens=cu.to(dev),
                    k_scale=scale[0], v_scale=scale[1])
    q = torch.randn(1, 64, dim, generator=gen).bfloat16()
    ids = torch.tensor([7, 0, 3, -1], dtype=torch.int32).expand(1, heads, 4).contiguous()
    got = m3_sparse_decode(q.to(dev), k_cache, v_cache, table.to(dev), lens.to(dev), ids.to(dev), return_lse=True,
                           k_scale=scale[0], v_scale=scale[1])
    at = table[0].long().to(dev)
    small = [torch.stack([x[int(i)] for i in at]).cpu() for x in (k_cache, v_cache, *scale)]
    case = (q, *small, torch.arange(8, dtype=torch.int32).view(1, 8), lens, ids)
    check(case, 128, got)


@pytest.mark.parametrize("batch,heads,ratio,dim,dtype", [
    (148, 3, 8, 128, torch.bfloat16), (149, 3, 8, 128, torch.bfloat16), (150, 3, 4, 128, torch.float16),
    (151, 3, 8, 128, torch.bfloat16), (225, 3, 8, 128, torch.bfloat16), (60, 4, 20, 128, torch.float16),
    (83, 5, 8, 256, torch.bfloat16), (61, 5, 12, 256, torch.float32), (101, 7, 8, 64, torch.float16)])
def test_more_requests_than_run_at_once(batch, heads, ratio, dim, dtype, cuda_device):
    """Around whole waves of blocks and behind them, where the first items are shared between blocks and the others
    have one each; every tenth request is empty."""
    gen = torch.Generator().manual_seed(batch)
    lens = torch.randint(1, 600, (batch,), generator=gen)
    lens[::10] = 0
    case = make_case(lens.tolist(), heads, ratio, dim, 128, 64, 4, dtype, seed=batch)
    check(case, 128, run(case, 128, cuda_device))
