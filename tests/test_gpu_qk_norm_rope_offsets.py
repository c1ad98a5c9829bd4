"""Weight gradients over more than 2^31 query elements against the float64 definition on the rows that are not
zero (zero rows add nothing, and no rounding). Tolerance as in test_gpu_qk_norm_rope.py: 64 roundings behind a
term and one per row of the running sum, of the terms' absolute sum, hundredths where a row's share is about one: a
row that is left out or counted twice shows."""

import pytest
import torch

from msa_triton_b200 import m3_qk_norm_rope, m3_rope_table
from tests import rope_oracle as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [128, 120])
def test_weight_gradients_past_32_bit_offsets(dim, cuda_device):
    dev = cuda_device
    heads = 64
    total = 2 ** 31 // (heads * dim) + 40
    gen = torch.Generator().manual_seed(dim)
    rows = torch.cat((torch.arange(3), torch.randint(3, total - 3, (6,), generator=gen), torch.arange(total - 3, total)))
    rows = torch.unique(rows)
    n = len(rows)
    few = [torch.randn(n, h, dim, generator=gen).bfloat16() for h in (heads, 1, heads, 1)]

    def spread(x):
        y = torch.zeros(total, *x.shape[1:], dtype=x.dtype, device=dev)
        y[rows.to(dev)] = x.to(dev)
        return y

    q, k, gq, gk = (spread(x) for x in few)
    wq, wk = (1 + 0.3 * torch.randn(dim, generator=gen) for _ in range(2))
    leaves = [wq.to(dev).requires_grad_(), wk.to(dev).requires_grad_()]
    table = m3_rope_table(64, dim)
    positions = (torch.arange(total) % 64).to(torch.int32)
    out = m3_qk_norm_rope(q, k, *leaves, table.to(dev), positions=positions.to(dev))
    grads = torch.autograd.grad(out, leaves, (gq, gk))
    cos, sin = table.double()[positions[rows].long()].split(dim // 2, -1)
    for x, g, w, got in ((few[0], few[2], wq, grads[0]), (few[1], few[3], wk, grads[1])):
        _, dw, _, size = R.norm_rope_backward(x.double(), w.double(), g.double(), cos, sin, 1e-6, False)
        bound = (R.half_step(torch.float32) * dw.abs() + (64 + n * x.shape[1]) * R.U * size)
        assert float(bound.max()) < 0.1
        assert ((got.cpu().double() - dw).abs() <= bound).all()
