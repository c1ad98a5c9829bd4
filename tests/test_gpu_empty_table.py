"""Rotation tables without rows: every position lies outside them, so rotated heads are NaN, whatever the
layout. (An empty tensor has no address: nothing may be read through it.)"""

import pytest
import torch

from msa_triton_b200 import m3_qk_norm_rope

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(128, 64), (64, 64), (100, 50), (27, 4), (512, 512), (300, 2), (64, 6)])
def test_norm_gives_nan(dim, rotary, interleaved, dtype, cuda_device):
    dev = cuda_device
    gen = torch.Generator().manual_seed(dim)
    q, k = (torch.randn(5, h, dim, generator=gen).to(dtype).to(dev).requires_grad_() for h in (3, 1))
    wq, wk = (torch.ones(dim, dtype=dtype, device=dev).requires_grad_() for _ in range(2))
    table = torch.empty(0, rotary, device=dev)
    positions = torch.tensor([0, 1, -1, 7, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    out = m3_qk_norm_rope(q, k, wq, wk, table, positions=positions, interleaved=interleaved)
    assert all(torch.isnan(x).all() for x in out)
    grads = torch.autograd.grad(out, (q, k, wq, wk), [torch.ones_like(x) for x in out])
    assert all(torch.isnan(x).all() for x in grads)
