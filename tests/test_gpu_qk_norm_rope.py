"""m3_qk_norm_rope (forward, backward, compiled, captured) against a float64 definition.

Tolerance of a value y stored in type t: half a step of t on y, plus K * 2^-24 on the absolute
terms behind y. K counts the float32 roundings on the way to an element, each at most 2^-24
relative: forward, the mean of squares (8 terms a lane or 16 units, 5 shuffle steps, the scale: 22),
halved by the square root, rsqrtf's 2 ulp (4), two products and the rotation's three: below 24.
Backward: the same 22 for the dot product (not halved), r twice, the rotation and the products:
below 64. A weight's gradient adds one rounding per row of its running sum."""

import pytest
import torch

from msa_triton_b200 import m3_qk_norm_rope, m3_rope_table, prepare_batch
from tests import rope_oracle as R
from tests.helpers import cu_of

pytestmark = pytest.mark.gpu

FWD, BWD = 24 * R.U, 64 * R.U
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def close(name, got, want, size, factor, dtype):
    got, want = got.detach().cpu().double(), want
    assert got.shape == want.shape, name
    bound = R.half_step(dtype) * want.abs() * (1 + 2 ** -6) + factor * size * (1 + R.half_step(dtype)) + TINY[dtype]
    over = (got - want).abs() / bound
    assert not torch.isnan(over).any() and float(over.max()) <= 1, f"{name}: {float(over.max())} of the bound"


def make(lens, hq, hk, dim, rotary, dtype, w_dtype, seed=0, fused=False):
    gen = torch.Generator().manual_seed(seed)
    t = sum(lens)
    row = torch.randn(t, (hq + 2 * hk) * dim, generator=gen) * (0.5 * torch.randn(t, 1, generator=gen)).exp()
    row = row.to(dtype)
    q, k = row[:, :hq * dim].view(t, hq, dim), row[:, hq * dim:(hq + hk) * dim].view(t, hk, dim)
    if not fused:
        q, k = q.clone(), k.clone()
    wq, wk = ((1 + 0.3 * torch.randn(dim, generator=gen)).to(w_dtype) for _ in range(2))
    gq, gk = torch.randn(t, hq, dim, generator=gen).to(dtype), torch.randn(t, hk, dim, generator=gen).to(dtype)
    return q, k, wq, wk, gq, gk, m3_rope_table(max(lens + [1]) + 5, rotary, base=100.0)


def on(dev, *xs):
    """Copies on the device that keep the strides (a fused projection's views stay views)."""
    out = []
    for x in xs:
        if x.is_contiguous():
            out.append(x.to(dev))
        else:
            base = torch.empty(x.shape[0], x.stride(0), dtype=x.dtype, device=dev)
            y = base[:, :x.shape[1] * x.shape[2]].view(x.shape)
            y.copy_(x)
            out.append(y)
    return out


CASES = [
    # lens, Hq, Hk, D, R, interleaved, dtype, weights, fused
    ([1], 64, 8, 128, 64, False, torch.bfloat16, torch.bfloat16, False),
    ([70, 1, 0, 129], 16, 4, 128, 128, False, torch.bfloat16, torch.float32, True),
    ([33, 40], 8, 1, 64, 32, True, torch.float32, torch.float32, True),
    ([5, 260], 32, 8, 128, 64, True, torch.float16, torch.float16, True),
    ([37], 3, 5, 96, 24, False, torch.bfloat16, torch.bfloat16, True),
    ([37], 5, 2, 192, 96, True, torch.float16, torch.float32, False),
    ([9, 8], 2, 1, 256, 256, False, torch.float32, torch.float32, False),
    ([19], 7, 3, 32, 8, False, torch.bfloat16, torch.bfloat16, False),
    ([19], 7, 3, 8, 8, True, torch.bfloat16, torch.bfloat16, False),
    ([23], 4, 2, 128, 0, False, torch.bfloat16, torch.bfloat16, False),
    # off the vector layout: odd widths, a wide head, rows at odd addresses
    ([21, 4], 3, 2, 24, 20, False, torch.float32, torch.float32, False),
    ([21, 4], 3, 2, 27, 10, True, torch.bfloat16, torch.bfloat16, True),
    ([11], 2, 1, 512, 128, False, torch.float16, torch.float16, False),
    ([11], 1, 1, 1, 0, False, torch.float32, torch.float32, False),
    ([50], 2, 2, 300, 300, True, torch.float32, torch.float32, False),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[1]}x{c[2]}x{c[3]}r{c[4]}{'i' if c[5] else 'h'}-{c[6]}")
def test_forward_and_backward_match_fp64(case, cuda_device):
    lens, hq, hk, dim, rotary, inter, dtype, w_dtype, fused = case
    q, k, wq, wk, gq, gk, table = make(lens, hq, hk, dim, rotary, dtype, w_dtype, fused=fused)
    dev = cuda_device
    leaves = [x.requires_grad_() for x in on(dev, q, k, wq, wk)]
    cu = cu_of(lens, dev)
    out = m3_qk_norm_rope(*leaves, table.to(dev), cu, interleaved=inter, eps=1e-5, prepared=prepare_batch(cu))
    grads = torch.autograd.grad(out, leaves, (gq.to(dev), gk.to(dev)))
    cos, sin = table.double()[R.positions_of(lens)].split(rotary // 2, -1) if rotary else [torch.zeros(sum(lens), 0)] * 2
    rows = sum(lens)
    for i, (x, w, g, heads) in enumerate(((q, wq, gq, hq), (k, wk, gk, hk))):
        args = (x.double(), w.double())
        y, size = R.norm_rope(*args, cos, sin, 1e-5, inter)
        close(f"out {i}", out[i], y, size, FWD, dtype)
        assert out[i].is_contiguous()
        dx, dw, dx_size, dw_size = R.norm_rope_backward(*args, g.double(), cos, sin, 1e-5, inter)
        close(f"dx {i}", grads[i], dx, dx_size, BWD, dtype)
        close(f"dw {i}", grads[2 + i], dw, dw_size, BWD + rows * heads * R.U, w_dtype)


def test_gradients_match_differences(cuda_device):
    """Directional derivatives by central differences of the float64 definition: with step h the
    differences are off by O(h^2) of the third derivative, far below the 1e-6 allowed here."""
    lens, hq, hk, dim, rotary, eps = [13, 6], 4, 2, 64, 32, 1e-6
    q, k, wq, wk, gq, gk, table = make(lens, hq, hk, dim, rotary, torch.float32, torch.float32, seed=3)
    dev = cuda_device
    leaves = [x.to(dev).requires_grad_() for x in (q, k, wq, wk)]
    out = m3_qk_norm_rope(*leaves, table.to(dev), cu_of(lens, dev), eps=eps)
    grads = [g.cpu().double() for g in torch.autograd.grad(out, leaves, (gq.to(dev), gk.to(dev)))]
    cos, sin = table.double()[R.positions_of(lens)].split(rotary // 2, -1)

    def loss(values):
        a, b, c, d = values
        return float((R.norm_rope(a, c, cos, sin, eps, False)[0] * gq.double()).sum()
                     + (R.norm_rope(b, d, cos, sin, eps, False)[0] * gk.double()).sum())

    gen = torch.Generator().manual_seed(9)
    at = [x.double() for x in (q, k, wq, wk)]
    for i in range(4):
        step = torch.randn(at[i].shape, generator=gen, dtype=torch.float64)
        h = 1e-5
        up = loss([x + h * step if j == i else x for j, x in enumerate(at)])
        down = loss([x - h * step if j == i else x for j, x in enumerate(at)])
        size = float((grads[i].abs() * step.abs()).sum())
        # the kernel's float32 error over all elements (BWD, and its sums') and the differences' own
        assert abs((up - down) / (2 * h) - float((grads[i] * step).sum())) <= (1e-6 + 16 * BWD) * size


@pytest.mark.parametrize("need", [(1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 1, 0, 0), (0, 0, 1, 1)])
def test_each_input_can_need_its_gradient_alone(need, cuda_device):
    lens = [40, 3]
    q, k, wq, wk, gq, gk, table = make(lens, 8, 2, 128, 64, torch.bfloat16, torch.bfloat16)
    dev = cuda_device
    full = [x.to(dev).requires_grad_() for x in (q, k, wq, wk)]
    g = (gq.to(dev), gk.to(dev))
    want = torch.autograd.grad(m3_qk_norm_rope(*full, table.to(dev), cu_of(lens, dev)), full, g)
    some = [x.to(dev).requires_grad_(bool(n)) for x, n in zip((q, k, wq, wk), need)]
    torch.autograd.backward(m3_qk_norm_rope(*some, table.to(dev), cu_of(lens, dev)), g)
    for x, w, n in zip(some, want, need):
        assert (x.grad is None) == (not n)
        if n:
            assert torch.equal(x.grad, w)  # fixed-order sums: the same bits


def test_broadcast_and_strided_gradients(cuda_device):
    lens = [25]
    q, k, wq, wk, gq, gk, table = make(lens, 8, 2, 128, 64, torch.bfloat16, torch.bfloat16)
    dev = cuda_device
    leaves = [x.to(dev).requires_grad_() for x in (q, k, wq, wk)]
    row = gq[:1, :1].to(dev)
    for a, b in ((row.expand(25, 8, 128), gk.to(dev).transpose(0, 1).contiguous().transpose(0, 1)),
                 (torch.ones((), dtype=torch.bfloat16, device=dev).expand(25, 8, 128), gk.to(dev))):
        out = m3_qk_norm_rope(*leaves, table.to(dev), cu_of(lens, dev))
        got = torch.autograd.grad(out, leaves, (a, b))
        out = m3_qk_norm_rope(*leaves, table.to(dev), cu_of(lens, dev))
        want = torch.autograd.grad(out, leaves, (a.clone(memory_format=torch.contiguous_format), b.contiguous()))
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_positions_inside_and_outside_the_table(cuda_device):
    dev = cuda_device
    q, k, wq, wk, _, _, _ = make([6], 8, 2, 128, 64, torch.bfloat16, torch.bfloat16)
    table = m3_rope_table(1000, 64, device=dev)
    pos = torch.tensor([0, 999, 1000, -1, 2 ** 31 - 1, 17], dtype=torch.int32)
    out = m3_qk_norm_rope(*(x.to(dev) for x in (q, k, wq, wk)), table, positions=pos.to(dev))
    bad = torch.tensor([False, False, True, True, True, False])
    cos, sin = table.cpu().double()[torch.where(bad, 0, pos).long()].split(32, -1)
    for got, x, w in zip(out, (q, k), (wq, wk)):
        assert torch.isnan(got[bad.to(dev)]).all()
        y, size = R.norm_rope(x.double(), w.double(), cos, sin, 1e-6, False)
        close("inside", got[(~bad).to(dev)], y[~bad], size[~bad], FWD, torch.bfloat16)
    # the scalar path answers the same way
    odd = m3_qk_norm_rope(*(x[..., :27].contiguous().to(dev) for x in (q, k, wq, wk)), table[:, :10].contiguous(),
                          positions=pos.to(dev))
    assert torch.isnan(odd[0][bad.to(dev)]).all() and not torch.isnan(odd[0][(~bad).to(dev)]).any()


def test_table_is_exact_at_far_positions(cuda_device):
    table = m3_rope_table(300001, 16, base=5e6, device=cuda_device)
    angle = 300000 * 5e6 ** (-torch.arange(0, 16, 2, dtype=torch.float64) / 16)
    want = torch.cat((angle.cos(), angle.sin()))
    # float32's half step on values up to 1, and float64's error of an angle near 3e5 (2^-34)
    assert (table[300000].cpu().double() - want).abs().max() <= 2.0 ** -25 + 2.0 ** -33


def test_nonfinite_rows_stay_apart_and_zero_rows_are_zero(cuda_device):
    dev = cuda_device
    q, k, wq, wk, gq, gk, table = make([8], 8, 2, 128, 64, torch.bfloat16, torch.bfloat16)
    q[2, 3, 5], q[4, 1, 100], k[5, 1] = float("inf"), float("nan"), 0
    leaves = [x.to(dev).requires_grad_() for x in (q, k, wq, wk)]
    out = m3_qk_norm_rope(*leaves, table.to(dev), cu_of([8], dev))
    finite = torch.isfinite(out[0]).all(-1).cpu()
    want = torch.ones(8, 8, dtype=torch.bool)
    want[2, 3] = want[4, 1] = False
    assert torch.equal(finite, want)
    assert torch.count_nonzero(out[1][5, 1]) == 0 and torch.isfinite(out[1]).all()
    dq, dk = torch.autograd.grad(out, leaves[:2], (gq.to(dev), gk.to(dev)))
    assert torch.equal(torch.isfinite(dq).all(-1).cpu(), want) and torch.isfinite(dk).all()


def test_empty_batch(cuda_device):
    dev = cuda_device
    q, k, wq, wk, gq, gk, table = make([0], 4, 2, 64, 32, torch.bfloat16, torch.bfloat16)
    leaves = [x.to(dev).requires_grad_() for x in (q, k, wq, wk)]
    out = m3_qk_norm_rope(*leaves, table.to(dev), cu_of([0, 0], dev))
    grads = torch.autograd.grad(out, leaves, (gq.to(dev), gk.to(dev)))
    assert out[0].shape == (0, 4, 64) and torch.count_nonzero(grads[2]) == 0 and torch.count_nonzero(grads[3]) == 0


def test_runs_are_bit_identical_and_streams_are_honoured(cuda_device):
    dev = cuda_device
    lens = [3000, 1200]
    q, k, wq, wk, gq, gk, table = make(lens, 32, 8, 128, 128, torch.bfloat16, torch.float32)
    table, cu = table.to(dev), cu_of(lens, dev)
    leaves = [x.to(dev).requires_grad_() for x in (q, k, wq, wk)]

    def step():
        out = m3_qk_norm_rope(*leaves, table, cu)
        return [x.detach() for x in out] + list(torch.autograd.grad(out, leaves, (gq.to(dev), gk.to(dev))))

    first = step()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream(dev).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_captured_step_follows_its_inputs(cuda_device):
    dev = cuda_device
    q, k, wq, wk, gq, gk, table = make([64], 8, 2, 128, 64, torch.bfloat16, torch.bfloat16)
    q, k, wq, wk, gq, gk, table = (x.to(dev) for x in (q, k, wq, wk, gq, gk, table))
    pos = torch.arange(64, dtype=torch.int32, device=dev)

    def step():
        leaves = [x.detach().requires_grad_() for x in (q, k, wq, wk)]
        out = m3_qk_norm_rope(*leaves, table, positions=pos)
        return [x.detach() for x in out] + list(torch.autograd.grad(out, leaves, (gq, gk)))

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    gen = torch.Generator(device=dev).manual_seed(5)
    q.normal_(generator=gen)
    pos.copy_(pos.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, step()))


def test_compiled_call_matches_eager(cuda_device):
    dev = cuda_device
    lens = [40, 9]
    q, k, wq, wk, gq, gk, table = make(lens, 8, 2, 128, 64, torch.bfloat16, torch.bfloat16)
    leaves = [x.to(dev).requires_grad_() for x in (q, k, wq, wk)]
    table, cu = table.to(dev), cu_of(lens, dev)
    prep = prepare_batch(cu)

    def layer(a, b, c, d):
        x, y = m3_qk_norm_rope(a * 2, b, c, d, table, prep.cu_seqlens, prepared=prep)
        return x + 1, y

    want = layer(*leaves)
    got = torch.compile(layer, fullgraph=True)(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = (gq.to(dev), gk.to(dev))
    for a, b in zip(torch.autograd.grad(got, leaves, g), torch.autograd.grad(want, leaves, g)):
        assert torch.equal(a, b)


def test_registered_operator_passes_opcheck(cuda_device):
    import msa_triton_b200.library  # noqa: F401  (registers the operators)

    dev = cuda_device
    lens = [9, 4]
    q, k, wq, wk, _, _, table = make(lens, 4, 2, 64, 32, torch.float32, torch.float32)
    leaves = [x.to(dev).requires_grad_() for x in (q, k, wq, wk)]
    args = (*leaves, table.to(dev), None, cu_of(lens, dev), 1e-6, False)
    torch.library.opcheck(torch.ops.msa_b200.qk_norm_rope.default, args)


def test_rows_past_32_bit_offsets(cuda_device):
    """Queries of more than 2^31 elements: rows at both ends, forward and backward, match a short call on them."""
    dev = cuda_device
    heads, dim, short = 64, 128, 5
    total = 2 ** 31 // (heads * dim) + short
    gen = torch.Generator(device=dev).manual_seed(21)
    ends = torch.cat((torch.arange(short), torch.arange(total - short, total))).to(dev)
    q = torch.zeros(total, heads, dim, dtype=torch.bfloat16, device=dev)
    q[ends] = torch.randn(2 * short, heads, dim, generator=gen, device=dev).bfloat16()
    k = torch.zeros(total, 1, dim, dtype=torch.bfloat16, device=dev)
    k[ends] = torch.randn(2 * short, 1, dim, generator=gen, device=dev).bfloat16()
    wq, wk = ((1 + 0.3 * torch.randn(dim, generator=gen, device=dev)).requires_grad_() for _ in range(2))
    table = m3_rope_table(64, dim, device=dev)
    positions = (torch.arange(total, device=dev) % 64).to(torch.int32)

    def run(q, k, positions):
        q, k = q.requires_grad_(), k.requires_grad_()
        yq, yk = m3_qk_norm_rope(q, k, wq, wk, table, positions=positions)
        return yq, yk, *torch.autograd.grad((yq, yk), (q, k, wq, wk), (q.detach(), k.detach()))

    # zero rows add nothing to the weights' gradients
    want = run(q[ends].clone(), k[ends].clone(), positions[ends])
    got = run(q, k, positions)
    for a, b in zip(got[:4], want[:4]):
        assert torch.equal(a[ends], b)
        assert torch.count_nonzero(a[short:-short]) == 0
    for a, b, rows in zip(got[4:], want[4:], (2 * short * heads, 2 * short)):
        # the same rows in another order: a float32 rounding per row on each side, of |g'| |x'| <= 3 * 6 * 6
        assert (a - b).abs().max() <= 2 * rows * 2.0 ** -24 * 108 * rows
