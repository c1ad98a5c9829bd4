"""The softmax weights of the 8-bit decode: inputs whose logits are so small that their errors say little, so
that the bound is what the weights and the values' scales leave.

Tolerance (u = 2^-24, sizes from the oracle; the bound of test_gpu_decode8.py without a rounding of the weights
to 16 bits): a logit's error (D + 32) u of its absolute terms, twice; exp2's 2 ulp (2^-21 with the argument's); a weight
as the sum of two fp16 numbers, 2^-22; one u per key and 64 for the merges; the output's own rounding, half a
step. ``cut``: what a weight loses at most below fp16's normal range, of its row's largest weight times scale."""

import pytest
import torch

from tests import cache_oracle as C
from tests import rope_oracle as R
from tests.test_gpu_decode8 import make_case, run

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def check(case, block, got, cut, scale=None):
    q, k, v, ks, vs, table, lens, ids = case
    dim, dtype = q.shape[2], q.dtype
    eff = dim ** -0.5 if scale is None else scale
    out, _, size_s, size_o, size_w, keys = C.attend(q, k, v, ks, vs, table, lens, ids, block, eff)
    weight = 2 * (dim + 32) * R.U * size_s + 2.0 ** -21 + 2.0 ** -22 + (keys + 64) * R.U
    bound = (R.half_step(dtype) * out.abs() * (1 + 2.0 ** -6) + weight[..., None] * size_o + cut * size_w[..., None]
             + 2.0 ** -25 * (dtype == torch.float16))
    got_out = got[0].cpu().double()
    assert not torch.isnan(got_out).any()
    off = (got_out - out).abs()
    assert float((off - bound).max()) <= 0, f"{float((off / bound.clamp(min=1e-300)).max())} of the bound"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ratio,dim", [(8, 128), (16, 128), (4, 64), (3, 27), (8, 256)])
def test_weights_keep_float32(ratio, dim, dtype, cuda_device):
    """Few keys with weights close to one another: a weight rounded to the output's bits would show."""
    made = make_case([3, 5, 9, 17, 40, 70], 2, ratio, dim, 128, 16, 4, dtype, seed=dim + ratio)
    made[0].mul_(0.02)
    check(made, 128, run(made, 128, cuda_device), 2.0 ** -25)


# Half of fp16's smallest step, 2^-25, over a largest weight of 2^13 or more.
CUT = 2.0 ** -38


@pytest.mark.parametrize("dtype", TYPES)
def test_many_small_weights_beside_a_few_large_ones(dtype, cuda_device):
    """In every 32 keys one that outweighs the others by e^17.5 and whose value is zero in the odd dims, where the
    others' values have one sign: what is left of them there is their sum alone."""
    made = make_case([1100], 1, 4, 64, 128, 128, 9, dtype, seed=1)
    q, k, v, ks, vs, table, lens, ids = made
    gen = torch.Generator().manual_seed(2)
    kc, vc = torch.zeros(k.shape), torch.randint(4, 400, v.shape, generator=gen).float()
    kc[:, ::32, :, 0] = 7
    vc[:, ::32, :, 1::2] = 0
    k.copy_(kc.to(FP8))
    v.copy_(vc.to(FP8))
    ks.fill_(1.0)
    q.zero_()
    q[..., 0] = 20
    check(made, 128, run(made, 128, cuda_device), CUT)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("far", [12, 20])
def test_pages_with_a_large_value_scale(far, dtype, cuda_device):
    """Every second page has a value scale 2^far times the others' and zeros in the odd dims."""
    made = make_case([180, 60], 2, 8, 64, 128, 16, 2, dtype, seed=far)
    q, k, v, ks, vs, table, lens, ids = made
    large = torch.zeros(k.shape[0], dtype=torch.bool)
    large[table[:, ::2].flatten().clamp(min=0).long()] = True
    bits = v.view(torch.uint8)
    codes = bits[large]
    codes[..., 1::2] = 0
    bits[large] = codes
    vs.copy_(torch.where(large[:, None], 2.0 ** (far - 8), 2.0 ** -8))
    q.mul_(0.01)
    if dtype == torch.float16:
        vs.mul_(2.0 ** (8 - far))  # within fp16's range
    check(made, 128, run(made, 128, cuda_device), CUT)


@pytest.mark.parametrize("dtype", TYPES)
def test_no_value_scale_left_far_below_zero(dtype, cuda_device):
    """Pages of scale 0 stand for zeros: also where every logit is far below zero."""
    made = make_case([300, 40, 1], 2, 8, 128, 128, 64, 3, dtype, seed=9)
    q, k, v, ks, vs, *_ = made
    k.copy_(k.float().abs().to(FP8))
    q.copy_(-3 * q.abs())
    vs[:] = 0
    out, lse = run(made, 128, cuda_device)
    assert (lse < -100).any() and torch.isfinite(lse).all()
    assert torch.count_nonzero(out) == 0


@pytest.mark.parametrize("scale", [1.3 * 2.0 ** -6, 1.7 * 2.0 ** -100, 1.1 * 2.0 ** 60, 2.0 ** 118])
@pytest.mark.parametrize("size", [0.1, 60.0, 1e4, 1e7])
def test_equal_logits_average_the_values(size, scale, cuda_device):
    """One key to a request, or several with the same codes: whatever the logits and the value scales are, the weights
    are equal, and the output is the mean of the values: 2^-21 for the weights' two terms and the powers of two, u a key
    and 64 of the values' sizes."""
    made = make_case([1, 1, 2, 70, 130], 2, 8, 64, 128, 16, 2, torch.float32, seed=5)
    q, k, v, ks, vs, table, lens, ids = made
    k.copy_(torch.randn(1, 1, 2, 64, generator=torch.Generator().manual_seed(3)).to(FP8).expand(k.shape))
    ks.fill_(float(ks[0, 0]))
    gen = torch.Generator().manual_seed(1)
    vs.copy_(scale * (1 + torch.rand(vs.shape, generator=gen)))
    q.mul_(size)
    out, _ = run(made, 128, cuda_device)
    out = out.cpu().double()
    for b, n in enumerate(lens.tolist()):
        at = torch.arange(n)
        page = table[b, at // 16].long()
        x = v[page, at % 16].float().double() * vs[page].double()[..., None]
        want, sizes = (y.mean(0).repeat_interleave(8, 0) for y in (x, x.abs()))
        off = (out[b] - want).abs()
        bound = (2.0 ** -21 + (n + 64) * R.U) * sizes + R.U * want.abs()
        assert float((off - bound).max()) <= 0, f"{n} keys: {float((off / bound.clamp(min=1e-300)).max())} of the bound"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("power", [-133, -126, -118, 125, 126, 127])
def test_queries_at_the_ends_of_the_range(power, dtype, cuda_device):
    """Queries around 2^power with key scales and a factor that bring their logits back to ordinary size."""
    made = make_case([90, 200], 2, 8, 64, 128, 16, 2, dtype, seed=17)
    q, k, v, ks, vs, *_ = made
    signs = torch.randn(q.shape, generator=torch.Generator().manual_seed(4))
    q.copy_((signs.sign() * (1 + signs.abs().clamp(max=0.9))).double().mul(2.0 ** power).to(dtype))
    scale = 2.0 ** -20 if power > 0 else 2.0 ** 20
    ks.copy_((ks.double() * (2.0 ** -power / scale / 8)).float())
    assert torch.isfinite(q.float()).all() and (ks >= torch.finfo(torch.float32).tiny).all() and torch.isfinite(ks).all()
    check(made, 128, run(made, 128, cuda_device, scale=scale), CUT, scale=scale)


def test_logits_across_the_range(cuda_device):
    """Logits near both ends of float32: one key outweighs whatever came before it."""
    made = make_case([256], 1, 4, 64, 32, 32, 8, torch.float32, seed=18)
    q, k, v, ks, vs, table, lens, ids = made
    q.zero_()
    q[..., 0] = 1.0
    k.zero_()
    for i in range(8):
        k[int(table[0, i]), :, 0, 0] = torch.tensor(-448.0 if i < 4 else 448.0).to(FP8)
    k[int(table[0, 6]), 5:, 0, 0] = 0
    ks.fill_(2.0 ** 119)
    ids.copy_(torch.arange(8, dtype=torch.int32))
    out, lse = run(made, 32, cuda_device, scale=0.5)
    keys = torch.tensor([i * 32 + j for i in range(4, 8) for j in range(32) if i != 6 or j < 5])
    page = table[0][keys // 32].long()
    x = v[page, keys % 32, 0].float().double() * vs[page, 0].double()[:, None]
    off = (out[0].cpu().double() - x.mean(0)).abs()
    assert float((off - (2.0 ** -21 + (len(keys) + 64) * R.U) * x.abs().mean(0)).max()) <= 0
    assert torch.isfinite(lse).all()
