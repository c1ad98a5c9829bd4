"""Argument checks of m3_qk_norm_rope, m3_cache_append and m3_sparse_decode over 8-bit caches: they run on
the host before any device work, so these run on the CPU."""

import pytest
import torch

from msa_triton_b200 import m3_cache_append, m3_qk_norm_rope, m3_rope_table, m3_sparse_decode, prepare_batch
from tests import rope_oracle as R
from tests.helpers import cu_of

FP8 = torch.float8_e4m3fn


def norm_args(**kw):
    a = dict(q=torch.ones(3, 4, 8), k=torch.ones(3, 2, 8), q_weight=torch.ones(8), k_weight=torch.ones(8),
             rope_table=m3_rope_table(10, 4), cu_seqlens=cu_of([1, 2]))
    a.update(kw)
    return a


@pytest.mark.parametrize("error,match,change", [
    (ValueError, "matching T", dict(k=torch.ones(2, 2, 8))),
    (ValueError, "matching T", dict(k=torch.ones(3, 2, 4))),
    (ValueError, "matching T", dict(q=torch.ones(3, 32))),
    (ValueError, "head dimension", dict(q=torch.ones(3, 1, 520), k=torch.ones(3, 1, 520))),
    (ValueError, "at least one head", dict(k=torch.ones(3, 0, 8))),
    (TypeError, "BF16", dict(q=torch.ones(3, 4, 8).double(), k=torch.ones(3, 2, 8).double())),
    (TypeError, "BF16", dict(k=torch.ones(3, 2, 8).half())),
    (ValueError, "shape", dict(k_weight=torch.ones(4))),
    (TypeError, "weights", dict(q_weight=torch.ones(8).half(), k_weight=torch.ones(8).half())),
    (TypeError, "weights", dict(k_weight=torch.ones(8).double())),
    (ValueError, "float32", dict(rope_table=torch.ones(10, 4).half())),
    (ValueError, "even and at most", dict(rope_table=torch.ones(10, 3))),
    (ValueError, "even and at most", dict(rope_table=torch.ones(10, 10))),
    (ValueError, "either", dict(positions=torch.zeros(3, dtype=torch.int32))),
    (ValueError, "either", dict(cu_seqlens=None)),
    (ValueError, "positions must be int32", dict(cu_seqlens=None, positions=torch.zeros(3))),
    (ValueError, "positions must be int32", dict(cu_seqlens=None, positions=torch.zeros(2, dtype=torch.int32))),
    (ValueError, "end at total_tokens", dict(cu_seqlens=cu_of([1, 1]))),
    (ValueError, "nondecreasing", dict(cu_seqlens=torch.tensor([0, 4, 3], dtype=torch.int32))),
    (ValueError, "fewer rows", dict(rope_table=m3_rope_table(1, 4))),
    (ValueError, "eps", dict(eps=-1.0)),
    (ValueError, "eps", dict(eps=float("nan"))),
    (ValueError, "same device", dict(k=torch.ones(3, 2, 8, device="meta"))),
    (ValueError, "same device", dict(rope_table=torch.ones(10, 4, device="meta"))),
    (ValueError, "different cu_seqlens", dict(prepared=prepare_batch(cu_of([3])))),
    (RuntimeError, "CUDA", dict()),
    (RuntimeError, "CUDA", dict(cu_seqlens=None, positions=torch.zeros(3, dtype=torch.int32))),
])
def test_norm_rope_refuses(error, match, change):
    a = norm_args(**change)
    with pytest.raises(error, match=match):
        m3_qk_norm_rope(a.pop("q"), a.pop("k"), a.pop("q_weight"), a.pop("k_weight"), a.pop("rope_table"),
                        a.pop("cu_seqlens"), **a)


def test_rope_table():
    table = m3_rope_table(50, 6, base=100.0)
    angle = torch.arange(50, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(0, 6, 2, dtype=torch.float64) / 6)
    assert table.dtype == torch.float32 and torch.equal(table, torch.cat((angle.cos(), angle.sin()), -1).float())
    assert m3_rope_table(5, 0).shape == (5, 0)
    for bad in (dict(max_position=0, rotary_dim=4), dict(max_position=4, rotary_dim=3),
                dict(max_position=4, rotary_dim=4, base=0.0), dict(max_position=4, rotary_dim=4, base=float("inf"))):
        with pytest.raises(ValueError):
            m3_rope_table(**bad)


ONE_CACHE, ONE_SCALE = torch.zeros(4, 8, 2, 16), torch.ones(4, 2)


def append_args(**kw):
    a = dict(k=torch.ones(2, 2, 16), v=torch.ones(2, 2, 16), k_cache=torch.zeros(4, 8, 2, 16),
             v_cache=torch.zeros(4, 8, 2, 16), block_table=torch.zeros(2, 2, dtype=torch.int32),
             seq_lens=torch.ones(2, dtype=torch.int32))
    a.update(kw)
    return a


def eight(**kw):
    return dict(k_cache=torch.zeros(4, 8, 2, 16).to(FP8), v_cache=torch.zeros(4, 8, 2, 16).to(FP8),
                **{**dict(k_scale=torch.ones(4, 2), v_scale=torch.ones(4, 2)), **kw})


@pytest.mark.parametrize("error,match,change", [
    (ValueError, "matching v", dict(v=torch.ones(2, 2, 8))),
    (ValueError, "go together", dict(v=None)),
    (ValueError, "go together", dict(v_cache=None)),
    (TypeError, "BF16", dict(k=torch.ones(2, 2, 16).double(), v=torch.ones(2, 2, 16).double())),
    (ValueError, "at least one head", dict(k=torch.ones(2, 0, 16), v=torch.ones(2, 0, 16))),
    (ValueError, "P,S,G,D", dict(k_cache=torch.zeros(4, 8, 1, 16))),
    (ValueError, "P,S,G,D", dict(v_cache=torch.zeros(4, 2, 16))),
    (ValueError, "share their pages", dict(v_cache=torch.zeros(5, 8, 2, 16))),
    (ValueError, "at least one token", dict(k_cache=torch.zeros(4, 0, 2, 16))),
    (TypeError, "inputs' dtype", dict(k_cache=torch.zeros(4, 8, 2, 16).half())),
    (ValueError, "dense head rows", dict(k_cache=torch.zeros(4, 8, 16, 2).transpose(2, 3))),
    (ValueError, "overlap", dict(k_cache=torch.zeros(1, 8, 2, 16).expand(4, 8, 2, 16))),
    (ValueError, "overlap", dict(k_cache=torch.zeros(1000).as_strided((4, 8, 2, 16), (128, 32, 8, 1)))),
    (ValueError, "k_scale belongs", dict(k_scale=torch.ones(4, 2))),
    (ValueError, "k_scale must be", eight(k_scale=None)),
    (ValueError, "v_scale must be", eight(v_scale=torch.ones(4, 1))),
    (ValueError, "k_scale must be", eight(k_scale=torch.ones(4, 2).double())),
    (ValueError, "k_scale must be contiguous", eight(k_scale=torch.ones(2, 4).t())),
    (ValueError, "v_scale belongs", dict(v=None, v_cache=None, v_scale=torch.ones(4, 2))),
    (ValueError, "of their own", dict(k_cache=ONE_CACHE, v_cache=ONE_CACHE)),
    (ValueError, "of their own", eight(k_scale=ONE_SCALE, v_scale=ONE_SCALE)),
    (ValueError, "seq_lens", dict(seq_lens=torch.ones(2))),
    (ValueError, "seq_lens", dict(seq_lens=torch.ones(2, 1, dtype=torch.int32))),
    (ValueError, "block_table", dict(block_table=torch.zeros(3, 2, dtype=torch.int32))),
    (ValueError, "block_table", dict(block_table=torch.zeros(2, 2))),
    (ValueError, "one token per request", dict(k=torch.ones(3, 2, 16), v=torch.ones(3, 2, 16))),
    (ValueError, r"int32 \[B \+ 1\]", dict(cu_seqlens=torch.zeros(2, dtype=torch.int32))),
    (ValueError, r"int32 \[B \+ 1\]", dict(cu_seqlens=torch.zeros(3))),
    (ValueError, "even and at most", dict(rope_table=torch.ones(5, 18))),
    (ValueError, "same device", dict(v=torch.ones(2, 2, 16, device="meta"))),
    (ValueError, "same device", dict(k_cache=torch.ones(4, 8, 2, 16, device="meta"))),
    (ValueError, "same device", dict(seq_lens=torch.ones(2, dtype=torch.int32, device="meta"))),
    (RuntimeError, "CUDA", dict()),
    (RuntimeError, "CUDA", eight()),
])
def test_append_refuses(error, match, change):
    a = append_args(**change)
    with pytest.raises(error, match=match):
        m3_cache_append(a.pop("k"), a.pop("v"), a.pop("k_cache"), a.pop("v_cache"), a.pop("block_table"),
                        a.pop("seq_lens"), **a)


@pytest.mark.parametrize("error,match,change", [
    (ValueError, "k_scale must be", dict(k_scale=None)),
    (ValueError, "v_scale must be", dict(v_scale=torch.ones(2, 4))),
    (ValueError, "v_scale must be contiguous", dict(v_scale=torch.ones(2, 4).t())),
    (TypeError, "BF16", dict(v_cache=torch.zeros(4, 8, 2, 16))),
    (TypeError, "BF16", dict(q=torch.ones(2, 4, 16).double())),
    (ValueError, "8-bit cache", dict(k_cache=torch.zeros(4, 8, 2, 16), v_cache=torch.zeros(4, 8, 2, 16))),
    (ValueError, "indices", dict(indices=torch.zeros(2, 4, 1, dtype=torch.int32))),
    (ValueError, "block_size", dict(block_size=0)),
    (ValueError, "finite", dict(scale=float("inf"))),
    (ValueError, "multiple of G", dict(q=torch.ones(2, 3, 16))),
    (ValueError, "same device", dict(indices=torch.zeros(2, 2, 1, dtype=torch.int32, device="meta"))),
    (RuntimeError, "CUDA", dict()),
])
def test_decode8_refuses(error, match, change):
    a = dict(q=torch.ones(2, 4, 16), block_table=torch.zeros(2, 2, dtype=torch.int32),
             seq_lens=torch.ones(2, dtype=torch.int32), indices=torch.zeros(2, 2, 1, dtype=torch.int32), **eight())
    a.update(change)
    with pytest.raises(error, match=match):
        m3_sparse_decode(a.pop("q"), a.pop("k_cache"), a.pop("v_cache"), a.pop("block_table"), a.pop("seq_lens"),
                         a.pop("indices"), **a)


def test_library_checks_its_arguments():
    """The C entry points answer bad arguments with a status, before any CUDA call."""
    from msa_triton_b200 import _lib

    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    n = None
    with pytest.raises(_lib.MsaError, match="head_dim"):
        _lib.call("msa_qk_norm_rope_fwd", n, n, 2, n, n, 2, n, 0, 0, 0, n, n, 0, 1, 1, 1, 513, 0, 0, 0, 0, 1e-6, n, n, n)
    with pytest.raises(_lib.MsaError, match="positions or cu_seqlens"):
        _lib.call("msa_qk_norm_rope_fwd", n, n, 2, n, n, 2, n, 0, 0, 0, n, n, 0, 1, 1, 1, 64, 0, 0, 0, 0, 1e-6, n, n, n)
    with pytest.raises(_lib.MsaError, match="bad dtype"):
        _lib.call("msa_cache_append", n, n, 3, 0, 0, 0, 0, n, 0, 0, 0, n, n, n, 0, 0, 1, 1, 1, 0, 0, n, n, 3, 0, 0, 0, 0,
                  0, 0, n, n, n)
    some = 16  # never read: the checks come first
    with pytest.raises(_lib.MsaError, match="needs its scales"):
        _lib.call("msa_cache_append", some, n, 2, 0, 0, 0, 0, n, 0, 0, 0, n, some, some, 1, 1, 1, 1, 1, 1, 1, some, n, 3,
                  0, 0, 0, 0, 0, 0, n, n, n)
    with pytest.raises(_lib.MsaError, match="missing pointers"):
        _lib.call("msa_cache_append", some, some, 2, 0, 0, 0, 0, n, 0, 0, 0, n, some, some, 1, 1, 1, 1, 1, 1, 1, some, n,
                  2, 0, 0, 0, 0, 0, 0, n, n, n)
    # nothing to do: no pointer is needed
    _lib.call("msa_cache_append", n, n, 2, 0, 0, 0, 0, n, 0, 0, 0, n, n, n, 0, 0, 1, 1, 1, 0, 0, n, n, 3, 0, 0, 0, 0, 0, 0,
              n, n, n)
    with pytest.raises(_lib.MsaError, match="head_dim"):
        _lib.call("msa_decode_attn_e4m3", n, 2, n, n, 0, 0, 0, 0, 0, 0, n, n, n, n, n, 1, 4, 2, 300, 16, 1, 1, 1, 16, 1.0,
                  n, n, n)


def test_oracle_gradients_match_autograd():
    """The float64 formulas that the kernels are held to, against autograd of the forward."""
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(5, 3, 12, generator=gen, dtype=torch.float64, requires_grad=True)
    w = torch.randn(12, generator=gen, dtype=torch.float64, requires_grad=True)
    g = torch.randn(5, 3, 12, generator=gen, dtype=torch.float64)
    cos, sin = m3_rope_table(5, 8).double().split(4, -1)
    for interleaved in (False, True):
        y, _ = R.norm_rope(x, w, cos, sin, 1e-3, interleaved)
        dx, dw = torch.autograd.grad(y, (x, w), g)
        fx, fw, _, _ = R.norm_rope_backward(x.detach(), w.detach(), g, cos, sin, 1e-3, interleaved)
        torch.testing.assert_close(fx, dx, rtol=1e-11, atol=1e-11)
        torch.testing.assert_close(fw, dw, rtol=1e-11, atol=1e-11)


def test_fake_kernels_give_output_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import msa_triton_b200.library  # noqa: F401  (registers the operators)

    ops = torch.ops.msa_b200
    with FakeTensorMode():
        row = torch.empty(7, 40 * 128, dtype=torch.bfloat16, device="cuda")
        q, k = row[:, :32 * 128].view(7, 32, 128), row[:, 32 * 128:].view(7, 8, 128)
        w = torch.empty(128, dtype=torch.float32, device="cuda")
        table = torch.empty(9, 64, dtype=torch.float32, device="cuda")
        cu = torch.empty(2, dtype=torch.int32, device="cuda")
        out = ops.qk_norm_rope(q, k, w, w, table, None, cu, 1e-6, False)
        assert [x.shape for x in out] == [q.shape, k.shape] and all(x.is_contiguous() for x in out)
        grads = ops.qk_norm_rope_backward(q, k, w, w, table, None, cu, 1e-6, False, *out, [True, False, True, False])
        assert grads[0].shape == q.shape and grads[1].numel() == 0 and grads[2].shape == w.shape
        assert grads[2].dtype == torch.float32 and grads[3].numel() == 0
