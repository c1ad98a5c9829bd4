"""The 16-bit decode calls on views: strided queries, lengths, block tables and selections give what
their contiguous copies give, bit for bit."""

import torch

import pytest

from msa_triton_b200 import m3_index_score_decode, m3_sparse_decode

pytestmark = pytest.mark.gpu


def test_strided_arguments(cuda_device):
    dev = cuda_device
    gen = torch.Generator(device=dev).manual_seed(0)
    lens = torch.tensor([300, 129, 700], dtype=torch.int32, device=dev)
    table = torch.randperm(36, generator=gen, device=dev).to(torch.int32).view(3, 12)
    k, v = (torch.randn(36, 64, 2, 128, generator=gen, device=dev).bfloat16() for _ in range(2))
    ik = torch.randn(36, 64, 1, 64, generator=gen, device=dev).bfloat16()
    q = torch.randn(16, 3, 128, generator=gen, device=dev).bfloat16().transpose(0, 1)  # dense, in another order
    iq = torch.randn(3, 2, 64, generator=gen, device=dev).bfloat16()
    ids = torch.tensor([[2, 0], [1, 0], [5, 3]], dtype=torch.int32, device=dev)[:, None].expand(3, 2, 2).contiguous()
    two = lambda x: torch.stack((x, x.flip(0)), -1)[..., 0]  # noqa: E731
    want = m3_sparse_decode(q.contiguous(), k, v, table, lens, ids, return_lse=True)
    got = m3_sparse_decode(q, k, v, two(table), two(lens), two(ids), return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(m3_index_score_decode(iq, ik, two(table), two(lens), 700),
                       m3_index_score_decode(iq, ik, table, lens, 700))
