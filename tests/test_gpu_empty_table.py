"""Rotation tables without rows: every position lies outside them, so rotated heads are NaN, whatever the
layout. (An empty tensor has no address: nothing may be read through it.)"""

import pytest
import torch

from msa_triton_b200 import m3_cache_append, m3_qk_norm_rope

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


@pytest.mark.parametrize("form", ["token", "chunk"])
@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("heads,dim,rotary", [(4, 64, 32), (1, 64, 64), (2, 27, 4)])
def test_append_stores_nan_keys(heads, dim, rotary, eight_bit, form, cuda_device):
    dev = cuda_device
    gen = torch.Generator().manual_seed(dim)
    n = 3 if form == "token" else 7
    k, v = (torch.randn(n, heads, dim, generator=gen).bfloat16().to(dev) for _ in range(2))
    kind = torch.float8_e4m3fn if eight_bit else torch.bfloat16
    kc, vc = (torch.zeros(4, 16, heads, dim, device=dev).to(kind) for _ in range(2))
    scales = {f"{x}_scale": torch.ones(4, heads, device=dev) for x in "kv"} if eight_bit else {}
    block_table = torch.tensor([[2], [0], [3]], dtype=torch.int32, device=dev)
    lens = torch.tensor([1, 1, 1] if form == "token" else [3, 0, 4], dtype=torch.int32, device=dev)
    cu = None if form == "token" else torch.tensor([0, 3, 3, 7], dtype=torch.int32, device=dev)
    m3_cache_append(k, v, kc, vc, block_table, lens, cu_seqlens=cu, rope_table=torch.empty(0, rotary, device=dev), **scales)
    at = 0
    for b, count in enumerate(lens.tolist()):
        page = int(block_table[b])
        keys, values = kc[page].float(), vc[page].float()
        if eight_bit:
            values = values * scales["v_scale"][page][:, None]
        assert torch.isnan(keys[:count]).all() and torch.count_nonzero(keys[count:]) == 0
        # e4m3: half a step, or of the smallest step 2^-9 of a scale of at most 2^-6 (448 * 2^-6 = 7)
        want = v[at:at + count].float()
        assert want.numel() == 0 or float(want.abs().max()) <= 7
        assert ((values[:count] - want).abs() <= (2.0 ** -4 * want.abs() + 2.0 ** -16 if eight_bit else 0)).all()
        at += count
