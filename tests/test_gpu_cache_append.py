"""m3_cache_append against a token-by-token restatement on the CPU.

The definition fixes every float32 rounding (each product and sum of the rotation by itself, one
rounding to the cache's type), so caches and scales have to be equal, bit for bit where they are
finite. The values a cache stands for are checked against float64 as well: 16-bit caches within half
a step of their type plus the rotation's three roundings (3 * 2^-24 on its terms); e4m3 within half a
step, 2^-4 of a normal value or 2^-10 of the scale below those, once more 2^-10 of the final scale for
each time a page moved to a larger one."""

import pytest
import torch

from msa_triton_b200 import m3_cache_append, m3_rope_table
from msa_triton_b200._lib import MsaError
from tests import cache_oracle as C
from tests import rope_oracle as R

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def same(name, got, want):
    got, want = got.cpu().float(), want.float()
    both_nan = torch.isnan(got) & torch.isnan(want)
    assert torch.equal(torch.where(both_nan, 0.0, got), torch.where(both_nan, 0.0, want)), name


class Pool:
    """A paged cache on the CPU and its copy on the device, for requests of at most `longest` tokens."""

    def __init__(self, requests, longest, size, heads, dim, dtype, gen, head_major=False, with_v=True):
        per = (longest + size - 1) // size
        pages = requests * per + 2
        self.table = torch.randperm(pages, generator=gen)[:requests * per].view(requests, per).to(torch.int32)

        def cache():
            x = torch.randn(pages, size, heads, dim, generator=gen).to(dtype)
            return x.float().transpose(1, 2).contiguous().to(dtype).transpose(1, 2) if head_major else x

        self.k, self.v = cache(), cache() if with_v else None
        fp8 = dtype == FP8
        self.ks = 2.0 ** torch.randint(-12, -2, (pages, heads), generator=gen).float() if fp8 else None
        self.vs = self.ks.flip(0).contiguous() if fp8 and with_v else None

    def to(self, dev):
        def move(x):
            if x is None:
                return None
            if x.is_contiguous():
                return x.to(dev)
            return x.transpose(1, 2).contiguous().to(dev).transpose(1, 2)  # head-major storage stays so
        return [move(x) for x in (self.k, self.v, self.ks, self.vs)]

    def check(self, device):
        for name, a, b in zip(("k", "v", "k_scale", "v_scale"), device, (self.k, self.v, self.ks, self.vs)):
            if b is not None:
                same(name, a, b)


CASES = [
    # heads, D, R, interleaved, page size, cache, dtype, head-major
    (8, 128, 64, False, 128, "same", torch.bfloat16, False),
    (8, 128, 64, False, 128, "fp8", torch.bfloat16, False),
    (4, 128, 128, True, 64, "fp8", torch.float16, True),
    (2, 64, 32, False, 16, "fp8", torch.float32, False),
    (3, 192, 48, True, 32, "same", torch.float32, True),
    (1, 96, 24, False, 16, "fp8", torch.bfloat16, False),
    (2, 256, 256, False, 300, "fp8", torch.bfloat16, False),   # pages longer than the registers hold
    (2, 32, 0, False, 200, "fp8", torch.float16, False),
    (5, 64, 32, False, 1, "fp8", torch.bfloat16, False),       # a scale to every token; 5 heads: 4 and 1 to a block
    (2, 27, 10, True, 5, "fp8", torch.bfloat16, False),        # off the vector layout
    (2, 40, 20, False, 7, "fp8", torch.float32, True),
    (3, 20, 12, False, 1, "same", torch.float16, False),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}x{c[1]}r{c[2]}{'i' if c[3] else 'h'}p{c[4]}-{c[5]}-{c[6]}")
def test_chunks_then_tokens_match_the_definition(case, cuda_device):
    heads, dim, rotary, inter, size, kind, dtype, major = case
    gen = torch.Generator().manual_seed(heads * dim + size)
    lens = [3, 0, 2 * size + 5, size, 141]
    pool = Pool(5, max(lens) + 40, size, heads, dim, FP8 if kind == "fp8" else dtype, gen, major)
    dev = cuda_device
    on = pool.to(dev)
    table = m3_rope_table(600 + 2 * size, rotary, base=50.0) if rotary else None
    table_dev = None if table is None else table.to(dev)
    held = torch.zeros(5, dtype=torch.int32)
    grows = 1.0
    # a prompt, a second chunk that goes on inside pages, then single tokens; values grow now and then,
    # so that pages have to move to larger scales
    for step, new in enumerate((lens, [9, 1, 0, 17, 2], [1] * 5, [1] * 5, [1] * 5)):
        n = sum(new)
        k, v = (grows * torch.randn(n, heads, dim, generator=gen).to(dtype) for _ in range(2))
        v *= 3
        held += torch.tensor(new, dtype=torch.int32)
        cu = torch.tensor([0] + new).cumsum(0).to(torch.int32) if step < 2 else None
        args = (k, v, pool.k, pool.v, pool.table, held, cu, table, inter, pool.ks, pool.vs)
        C.append(*args)
        m3_cache_append(k.to(dev), v.to(dev), on[0], on[1], pool.table.to(dev), held.to(dev),
                        cu_seqlens=None if cu is None else cu.to(dev), rope_table=table_dev, interleaved=inter,
                        k_scale=on[2], v_scale=on[3])
        pool.check(on)
        grows *= 1.0 if step % 2 else 3.0


@pytest.mark.parametrize("kind,dtype", [("fp8", torch.bfloat16), ("same", torch.bfloat16), ("same", torch.float16)])
def test_stored_values_match_fp64(kind, dtype, cuda_device):
    gen = torch.Generator().manual_seed(2)
    heads, dim, size, lens = 4, 128, 64, [200, 77]
    pool = Pool(2, 300, size, heads, dim, FP8 if kind == "fp8" else dtype, gen)
    dev = cuda_device
    on = pool.to(dev)
    table = m3_rope_table(400, 64)
    parts = [torch.randn(n, heads, dim, generator=gen).to(dtype) * (1 + 5 * (torch.arange(n) % 50 == 49))[:, None, None]
             for n in lens]
    cuts, held = [[150, 30], [50, 47]], [0, 0]
    for new in cuts:
        k = torch.cat([p[h:h + n] for p, h, n in zip(parts, held, new)])
        held = [h + n for h, n in zip(held, new)]
        m3_cache_append(k.to(dev), k.to(dev), on[0], on[1], pool.table.to(dev),
                        torch.tensor(held, dtype=torch.int32, device=dev),
                        cu_seqlens=torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32),
                        rope_table=table.to(dev), k_scale=on[2], v_scale=on[3])
    for b, part in enumerate(parts):
        n = held[b]
        cos, sin = table.double()[:n].split(32, -1)
        x = part[:n].double()
        for cache, scale, y, terms in ((on[0], on[2], R.rotate(x, cos, sin, False), R.rotate_abs(x, cos, sin, False)),
                                       (on[1], on[3], x, x.abs())):
            pages = pool.table[b].long()[torch.arange(n) // size]
            got = cache.cpu()[pages, torch.arange(n) % size].float().double()
            if kind == "fp8":
                s = scale.cpu().double()[pages][:, :, None]
                bound = y.abs() * 2.0 ** -4 + 2 * s * 2.0 ** -10
                got = got * s
            else:
                bound = y.abs() * R.half_step(dtype) * (1 + 2 ** -6) + 2.0 ** -25
            assert ((got - y).abs() <= bound + 3 * R.U * terms).all()


def test_padded_batches_and_bad_pages_write_nothing(cuda_device):
    gen = torch.Generator().manual_seed(4)
    dev = cuda_device
    for kind in (FP8, torch.bfloat16):
        for dim in (128, 27):
            pool = Pool(4, 100, 16, 2, dim, kind, gen)
            pool.table[1, 0], pool.table[2, :] = -1, 10 ** 6
            on = pool.to(dev)
            table = m3_rope_table(50, 8)
            # 4 requests, the last without tokens, and three rows behind the last one
            new, held = [5, 20, 18, 0], torch.tensor([5, 20, 18, 0], dtype=torch.int32)
            k, v = (torch.randn(46, 2, dim, generator=gen).bfloat16() for _ in range(2))
            cu = torch.tensor([0] + new).cumsum(0).to(torch.int32)
            C.append(k, v, pool.k, pool.v, pool.table, held, cu, table, False, pool.ks, pool.vs)
            m3_cache_append(k.to(dev), v.to(dev), on[0], on[1], pool.table.to(dev), held.to(dev), cu_seqlens=cu.to(dev),
                            rope_table=table.to(dev), k_scale=on[2], v_scale=on[3])
            pool.check(on)
            # a decode step: an idle request, one past its block table, one past the rotation table
            held = torch.tensor([0, 21, 19, 51], dtype=torch.int32)
            pool.table[3, 3] = pool.table[0, 0]
            narrow = pool.table[:, :4].contiguous()
            held[1] = 65
            C.append(k[:4], v[:4], pool.k, pool.v, narrow, held, None, table, False, pool.ks, pool.vs)
            m3_cache_append(k[:4].to(dev), v[:4].to(dev), on[0], on[1], narrow.to(dev), held.to(dev),
                            rope_table=table.to(dev), k_scale=on[2], v_scale=on[3])
            pool.check(on)
            assert torch.isnan(on[0][int(pool.table[3, 3]), 2].float()).all()  # its key has no angle


@pytest.mark.parametrize("inter", [False, True])
def test_chunks_and_single_tokens_store_the_same_bits(inter, cuda_device):
    """The same tokens in one packed call and one at a time, the largest of a page first (so that no page moves
    to a larger scale): 4 million values, enough for a product and a sum rounded as one to show."""
    dev = cuda_device
    gen = torch.Generator(device=dev).manual_seed(12)
    pages, size, heads, dim = 256, 16, 8, 128  # a page to a request
    k = torch.randn(pages, size, heads, dim, generator=gen, device=dev).bfloat16()
    k[:, 0] = 10
    table = m3_rope_table(size, dim, device=dev) * 0.7
    table[0] = torch.cat((torch.ones(dim // 2), torch.zeros(dim // 2))).to(dev)
    own = torch.randperm(pages, generator=gen, device=dev).to(torch.int32).view(-1, 1)

    def cache():
        return torch.zeros(pages, size, heads, dim, dtype=FP8, device=dev), torch.zeros(pages, heads, device=dev)

    (chunk, chunk_scale), (token, token_scale) = cache(), cache()
    m3_cache_append(k.flatten(0, 1), None, chunk, None, own, torch.full((pages,), size, dtype=torch.int32, device=dev),
                    cu_seqlens=torch.arange(0, pages * size + 1, size, dtype=torch.int32, device=dev), rope_table=table,
                    interleaved=inter, k_scale=chunk_scale)
    for row in range(size):
        m3_cache_append(k[:, row], None, token, None, own, torch.full((pages,), row + 1, dtype=torch.int32, device=dev),
                        rope_table=table, interleaved=inter, k_scale=token_scale)
    assert torch.equal(chunk_scale, token_scale)
    assert torch.equal(chunk.view(torch.uint8), token.view(torch.uint8))


def test_empty_calls_do_nothing(cuda_device):
    """No tokens, no requests, no pages: nothing to store, and no error."""
    dev = cuda_device
    for kind in (FP8, torch.bfloat16):
        cache = [torch.zeros(3, 16, 2, 64, device=dev).to(kind) for _ in range(2)]
        scale = [torch.ones(3, 2, device=dev) if kind == FP8 else None for _ in range(2)]
        lens = torch.zeros(2, dtype=torch.int32, device=dev)
        pages, cu = torch.zeros(2, 1, dtype=torch.int32, device=dev), torch.zeros(3, dtype=torch.int32, device=dev)
        none = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=dev)
        m3_cache_append(none, none, *cache, pages, lens, cu_seqlens=cu, k_scale=scale[0], v_scale=scale[1])
        m3_cache_append(none, none, *cache, pages[:0], lens[:0], k_scale=scale[0], v_scale=scale[1])
        one = torch.ones(2, 2, 64, dtype=torch.bfloat16, device=dev)
        m3_cache_append(one, one, *cache, pages[:, :0], lens + 1, k_scale=scale[0], v_scale=scale[1])
        empty = [c[:0] for c in cache]
        m3_cache_append(one, one, *empty, pages, lens + 1, k_scale=None if kind != FP8 else scale[0][:0],
                        v_scale=None if kind != FP8 else scale[1][:0])
        assert all(torch.count_nonzero(c.float()) == 0 for c in cache)


def test_more_new_rows_than_tokens_stores_the_last(cuda_device):
    gen = torch.Generator().manual_seed(5)
    dev = cuda_device
    pool = Pool(2, 64, 16, 2, 64, FP8, gen)
    on = pool.to(dev)
    held, cu = torch.tensor([3, 9], dtype=torch.int32), torch.tensor([0, 7, 12], dtype=torch.int32)
    k, v = (torch.randn(12, 2, 64, generator=gen).bfloat16() for _ in range(2))
    C.append(k, v, pool.k, pool.v, pool.table, held, cu, None, False, pool.ks, pool.vs)
    m3_cache_append(k.to(dev), v.to(dev), on[0], on[1], pool.table.to(dev), held.to(dev), cu_seqlens=cu.to(dev),
                    k_scale=on[2], v_scale=on[3])
    pool.check(on)


@pytest.mark.parametrize("dim", [128, 27])
def test_extreme_values(dim, cuda_device):
    """Zeros, subnormals, the largest floats, infinities and NaN: the scale counts finite values only."""
    gen = torch.Generator().manual_seed(6)
    dev = cuda_device
    pool = Pool(1, 80, 16, 6, dim, FP8, gen)
    on = pool.to(dev)
    k = torch.randn(33, 6, dim, generator=gen).bfloat16()
    k[:, 0] = 0
    k[:, 1] = 2.0 ** -133
    k[:, 2] *= 2.0 ** 120
    k[3, 3, 5], k[20, 3, 7], k[21, 3, 8] = float("inf"), float("-inf"), float("nan")
    k[:, 4] = float("inf")
    k[:, 5] = 448 * 2.0 ** -9  # exactly at the end of a scale
    cu = torch.tensor([0, 33], dtype=torch.int32)
    held = torch.tensor([33], dtype=torch.int32)
    C.append(k, k, pool.k, pool.v, pool.table, held, cu, None, False, pool.ks, pool.vs)
    m3_cache_append(k.to(dev), k.to(dev), on[0], on[1], pool.table.to(dev), held.to(dev), cu_seqlens=cu.to(dev),
                    k_scale=on[2], v_scale=on[3])
    pool.check(on)
    first = int(pool.table[0, 0])
    assert float(on[2][first, 0]) == 2.0 ** -126 and float(on[2][first, 5]) == 2.0 ** -9
    assert torch.isnan(on[0][first, :, 4].float()).all()
    # a page of zeros takes the next token's scale
    held += 1
    k1 = torch.ones(1, 6, dim).bfloat16()
    C.append(k1, k1, pool.k, pool.v, pool.table, held, None, None, False, pool.ks, pool.vs)
    m3_cache_append(k1.to(dev), k1.to(dev), on[0], on[1], pool.table.to(dev), held.to(dev), k_scale=on[2], v_scale=on[3])
    pool.check(on)


def test_keys_alone_and_strided_inputs(cuda_device):
    """The indexer's keys (one head, no v) out of a wider projection, into a 16-bit cache."""
    gen = torch.Generator().manual_seed(7)
    dev = cuda_device
    pool = Pool(2, 50, 16, 1, 64, torch.bfloat16, gen, with_v=False)
    on = pool.to(dev)
    wide = torch.randn(40, 200, generator=gen).bfloat16()
    held, cu = torch.tensor([25, 15], dtype=torch.int32), torch.tensor([0, 25, 40], dtype=torch.int32)
    table = m3_rope_table(64, 64)
    for offset in (64, 3):  # on and off the vector alignment
        k = wide[:, offset:offset + 64].unsqueeze(1)
        C.append(k, None, pool.k, None, pool.table, held, cu, table, False, None, None)
        m3_cache_append(wide.to(dev)[:, offset:offset + 64].unsqueeze(1), None, on[0], None, pool.table.to(dev),
                        held.to(dev), cu_seqlens=cu.to(dev), rope_table=table.to(dev))
        pool.check(on)
    # block table, lengths and boundaries as strided views
    both = torch.stack((pool.table, pool.table.flip(0)), dim=2).to(dev)
    m3_cache_append(k.to(dev), None, on[0], None, both[:, :, 0], torch.stack((held, held), 1).to(dev)[:, 0],
                    cu_seqlens=torch.stack((cu, cu), 1).to(dev)[:, 0], rope_table=table.to(dev))
    pool.check(on)


def test_captured_append_follows_lengths(cuda_device):
    """A captured decode step replayed as the requests grow over page ends."""
    gen = torch.Generator().manual_seed(8)
    dev = cuda_device
    pool = Pool(3, 64, 4, 2, 64, FP8, gen)
    on = pool.to(dev)
    table = m3_rope_table(64, 32)
    held = torch.tensor([0, 3, 10], dtype=torch.int32)
    static = [torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    held_dev, pages, angles = held.to(dev), pool.table.to(dev), table.to(dev)

    def step():
        m3_cache_append(*static, on[0], on[1], pages, held_dev, rope_table=angles, k_scale=on[2], v_scale=on[3])

    held_dev.zero_()  # the warm-up stores nothing
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(9):
        held += 1
        k, v = ((1 + i) * torch.randn(3, 2, 64, generator=gen).bfloat16() for _ in range(2))
        static[0].copy_(k)
        static[1].copy_(v)
        held_dev.copy_(held)
        graph.replay()
        C.append(k, v, pool.k, pool.v, pool.table, held, None, table, False, pool.ks, pool.vs)
    pool.check(on)


def test_offsets_past_32_bits(cuda_device):
    """A cache of more than 2^31 elements: the last pages, first and last heads."""
    dev = cuda_device
    gen = torch.Generator().manual_seed(9)
    pages, size, heads, dim = 2 ** 31 // (128 * 8 * 128) + 9, 128, 8, 128
    cache = torch.zeros(pages, size, heads, dim, dtype=FP8, device=dev)
    scale = torch.ones(pages, heads, device=dev)
    k = torch.randn(140, heads, dim, generator=gen).bfloat16()
    table = torch.tensor([[pages - 1, pages - 5]], dtype=torch.int32)
    held, cu = torch.tensor([140], dtype=torch.int32), torch.tensor([0, 140], dtype=torch.int32)
    m3_cache_append(k.to(dev), None, cache, None, table.to(dev), held.to(dev), cu_seqlens=cu.to(dev), k_scale=scale)
    small, small_scale = torch.zeros(2, size, heads, dim).to(FP8), torch.ones(2, heads)
    C.append(k, None, small, None, torch.tensor([[1, 0]], dtype=torch.int32), held, cu, None, False, small_scale, None)
    same("codes", torch.stack((cache[pages - 5], cache[pages - 1])), small)
    same("scales", scale[[pages - 5, pages - 1]], small_scale)
    assert torch.count_nonzero(cache[:pages - 9].view(torch.uint8)) == 0


@pytest.mark.parametrize("kind", [FP8, torch.bfloat16], ids=str)
def test_pages_past_32_bits(kind, cuda_device):
    """The last token of a page of 2^31 elements; off the vector layout, where elements are counted in 32 bits, such
    a page is refused."""
    dev = cuda_device
    for dim, size in ((128, 2 ** 24), (100, 2 ** 31 // 100 + 1)):
        cache = torch.zeros(1, size, 1, dim, dtype=kind, device=dev)
        scale = torch.ones(1, 1, device=dev) if kind == FP8 else None
        held = torch.tensor([size], dtype=torch.int32, device=dev)
        k = torch.randint(-8, 9, (1, 1, dim), device=dev).bfloat16()
        if dim == 100:
            with pytest.raises(MsaError, match="too large"):
                m3_cache_append(k, None, cache, None, held[:, None] * 0, held, k_scale=scale)
            continue
        m3_cache_append(k, None, cache, None, held[:, None] * 0, held, k_scale=scale)
        assert torch.equal(cache[0, -1].float(), k[0].float())
        assert not cache[0, -3:-1].float().any() and not cache[0, :2].float().any()
