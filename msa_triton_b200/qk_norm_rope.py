"""Per-head RMS norm of queries and keys with the position rotation, in one pass.

The operators of this package take normalised, rotated heads (the reference's
inputs, docs/msa_training_flow.md); this is the step that makes them from a
layer's projections, for the attention heads and, with ``index_q`` / ``index_k``
in the places of ``q`` / ``k``, for the indexer's:

    table = m3_rope_table(max_position, rotary_dim, base=5e6, device=q.device)
    q, k  = m3_qk_norm_rope(q, k, q_weight, k_weight, table, cu_seqlens)             # packed batch, differentiable
    q, k  = m3_qk_norm_rope(q, k, q_weight, k_weight, table, positions=seq_lens - 1)  # decode

    y = R(p) (weight * x * r),   r = (mean(x^2) + eps)^(-1/2) over the head's elements

All arithmetic is float32 with one rounding to the inputs' dtype at the end.
``q`` and ``k`` may be strided views of a fused projection (rows of a head
dense); the outputs are contiguous. CUDA tensors only.
"""

from __future__ import annotations

import math

import torch

from . import _lib
from ._lib import DTYPE_CODE, call, device_of, ptr, stream_of
from .decode import dense_rows
from .layout import sequence_lengths

MAX_HEAD_DIM = 512


def m3_rope_table(max_position: int, rotary_dim: int, *, base: float = 10000.0, device=None) -> torch.Tensor:
    """float32 ``[max_position, rotary_dim]``: the cosines, then the sines, of
    ``position * base^(-2i / rotary_dim)``. The angles are taken in float64, so far
    positions lose nothing; any table of this layout (scaled frequencies, say) can
    take its place."""
    if not isinstance(max_position, int) or max_position <= 0:
        raise ValueError("max_position must be a positive integer")
    if not isinstance(rotary_dim, int) or rotary_dim < 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be an even nonnegative integer")
    if not (math.isfinite(base) and base > 0):
        raise ValueError("base must be positive and finite")
    step = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    inv = base ** (-step / max(rotary_dim, 1))
    angle = torch.arange(max_position, dtype=torch.float64, device=device)[:, None] * inv
    return torch.cat((angle.cos(), angle.sin()), dim=-1).float()


def check_table(rope_table, head_dim, device):
    """The table's checks, shared with the cache append."""
    if rope_table.ndim != 2 or rope_table.dtype != torch.float32:
        raise ValueError("rope_table must be float32 [max_position, rotary_dim]")
    if rope_table.shape[1] % 2 or rope_table.shape[1] > head_dim:
        raise ValueError("rope_table's rotary_dim must be even and at most the head dimension")
    if rope_table.device != device:
        raise ValueError("All inputs must reside on the same device.")


def _common(q, k, q_weight, k_weight, table, positions, cu, interleaved):
    """The arguments that both launchers pass between the tensors and the gradients' strides."""
    dtype, (total, q_heads, dim), q_strides, k_strides = q.dtype, q.shape, q.stride(), k.stride()
    return (DTYPE_CODE[dtype], q_weight.data_ptr(), k_weight.data_ptr(), DTYPE_CODE[q_weight.dtype],
            table.data_ptr(), *table.shape, interleaved, ptr(positions), ptr(cu), 0 if cu is None else cu.shape[0] - 1,
            total, q_heads, k.shape[1], dim, q_strides[0], q_strides[1], k_strides[0], k_strides[1])


def _laid_out(q, k, q_weight, k_weight, table, positions, cu):
    return (dense_rows(q), dense_rows(k), q_weight.contiguous(), k_weight.contiguous(), table.contiguous(),
            None if positions is None else positions.contiguous(), None if cu is None else cu.contiguous())


def norm_rope_forward(q, k, q_weight, k_weight, table, positions, cu, eps, interleaved):
    """(q_out, k_out); shared by the autograd Function and the torch.library operator."""
    q, k, q_weight, k_weight, table, positions, cu = _laid_out(q, k, q_weight, k_weight, table, positions, cu)
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    with device_of(q):
        call("msa_qk_norm_rope_fwd", q.data_ptr(), k.data_ptr(), *_common(q, k, q_weight, k_weight, table, positions, cu,
                                                              interleaved),
             eps, q_out.data_ptr(), k_out.data_ptr(), stream_of(q))
    return q_out, k_out


def norm_rope_backward(q, k, q_weight, k_weight, table, positions, cu, eps, interleaved, grad_q, grad_k, need):
    """(dq, dk, dq_weight, dk_weight); `need`: which of the four to compute (the others are None)."""
    if not any(need):
        return None, None, None, None
    q, k, q_weight, k_weight, table, positions, cu = _laid_out(q, k, q_weight, k_weight, table, positions, cu)
    gq, gk = dense_rows(grad_q.to(q.dtype)), dense_rows(grad_k.to(k.dtype))
    dq, dk, dwq, dwk = (torch.empty_like(x, memory_format=torch.contiguous_format) if n else None
                        for x, n in zip((q, k, q_weight, k_weight), need))
    ws_bytes = _lib.load().msa_qk_norm_rope_bwd_workspace_size(q.shape[2]) if need[2] or need[3] else 0
    workspace = q.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
    with device_of(q):
        call("msa_qk_norm_rope_bwd", q.data_ptr(), k.data_ptr(), gq.data_ptr(), gk.data_ptr(),
             *_common(q, k, q_weight, k_weight, table, positions, cu, interleaved), *gq.stride()[:2],
             *gk.stride()[:2], eps, ptr(dq), ptr(dk), ptr(dwq), ptr(dwk), ptr(workspace), ws_bytes,
             stream_of(q))
    return dq, dk, dwq, dwk


class _QKNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, table, positions, cu, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, table, positions, cu)
        ctx.meta = (eps, interleaved)
        return norm_rope_forward(q, k, q_weight, k_weight, table, positions, cu, eps, interleaved)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_q, grad_k):
        eps, interleaved = ctx.meta
        grads = norm_rope_backward(*ctx.saved_tensors, eps, interleaved, grad_q, grad_k, ctx.needs_input_grad[:4])
        return (*grads, None, None, None, None, None)


def m3_qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    rope_table: torch.Tensor,
    cu_seqlens: torch.Tensor | None = None,
    *,
    positions: torch.Tensor | None = None,
    eps: float = 1e-6,
    interleaved: bool = False,
    prepared=None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every head of ``q[T,Hq,D]`` and ``k[T,Hk,D]``, then the rotation of its
    first ``rotary_dim`` elements by its token's position.

    ``q_weight[D]``, ``k_weight[D]``: the norms' weights (the inputs' dtype or float32).
    ``rope_table[max_position, rotary_dim]``: as ``m3_rope_table`` makes it; a width below
    ``D`` leaves the other elements unrotated. Positions count from the start of each packed
    sequence of ``cu_seqlens``, or are given as ``positions`` (int32 ``[T]``); a row whose
    position lies outside the table comes out as NaN. ``interleaved`` pairs neighbouring
    elements ``(2i, 2i + 1)`` instead of ``(i, i + rotary_dim / 2)``. Differentiable in ``q``,
    ``k`` and the weights (once). ``prepared`` as for ``m3_sparse_attention``.
    """
    if q.ndim != 3 or k.ndim != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError("expected q[T,Hq,D] and k[T,Hk,D] with matching T and D")
    (total, heads, dim), dtype, device = q.shape, q.dtype, q.device
    if heads <= 0 or k.shape[1] <= 0 or not 0 < dim <= MAX_HEAD_DIM:
        raise ValueError(f"expected at least one head and a head dimension in [1, {MAX_HEAD_DIM}]")
    if dtype not in DTYPE_CODE or k.dtype != dtype:
        raise TypeError("q/k must share a BF16, FP16, or FP32 dtype.")
    if q_weight.shape != (dim,) or k_weight.shape != (dim,):
        raise ValueError("q_weight and k_weight must have shape [D]")
    if q_weight.dtype not in (dtype, torch.float32) or k_weight.dtype != q_weight.dtype:
        raise TypeError("the weights must share the inputs' dtype or FP32")
    check_table(rope_table, dim, device)
    if (cu_seqlens is None) == (positions is None):
        raise ValueError("give either cu_seqlens or positions")
    if k.device != device or q_weight.device != device or k_weight.device != device:
        raise ValueError("All inputs must reside on the same device.")
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError("eps must be finite and nonnegative")
    if positions is not None:
        if positions.shape != (total,) or positions.dtype != torch.int32:
            raise ValueError("positions must be int32 [T]")
        if positions.device != device:
            raise ValueError("All inputs must reside on the same device.")
    else:
        if cu_seqlens.device != device:
            raise ValueError("All inputs must reside on the same device.")
        if max(sequence_lengths(cu_seqlens, total, prepared)) > rope_table.shape[0]:
            raise ValueError("rope_table has fewer rows than the longest sequence")
    _lib.require_cuda(q)
    if torch.compiler.is_compiling():  # traced by torch.compile: the registered operator
        from . import library

        return library.qk_norm_rope(q, k, q_weight, k_weight, rope_table, positions, cu_seqlens, eps, interleaved)
    if not (torch.is_grad_enabled()
            and (q.requires_grad or k.requires_grad or q_weight.requires_grad or k_weight.requires_grad)):
        return norm_rope_forward(q, k, q_weight, k_weight, rope_table, positions, cu_seqlens, eps, interleaved)
    return _QKNormRope.apply(q, k, q_weight, k_weight, rope_table, positions, cu_seqlens, eps, bool(interleaved))
