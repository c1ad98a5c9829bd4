"""New keys and values into a paged KV cache, in the inputs' type or in 8 bits.

The caches are those the decode operators read (``decode.py``): ``[P, S, G, D]``,
P physical pages of S tokens, addressed through a block table. One call per cache
stores the newest tokens of every request, rotating the keys on the way:

    m3_cache_append(k, v, k_cache, v_cache, block_table, seq_lens, rope_table=table)      # one token per request
    m3_cache_append(k, v, k_cache, v_cache, block_table, seq_lens, cu_seqlens=cu)         # packed chunks
    m3_cache_append(index_k, None, index_k_cache, None, block_table, seq_lens)            # the indexer's keys

(``m3_index_score_decode`` reads the indexer's cache in the type of its queries only: keep that one in 16 or
32 bits.)

8-bit caches are ``torch.float8_e4m3fn`` with float32 scales ``[P, G]``, one per page and
head: a code ``c`` stands for ``c * scale``. The append chooses powers of two, the smallest
with every value at most ``448 * scale`` (e4m3 is a floating format, so that costs no
precision); a page that already holds tokens keeps its scale unless the new ones need a
larger one, and then its earlier codes move to it, exactly as long as they stay normal
numbers. ``m3_sparse_decode`` reads such a cache with ``k_scale=`` / ``v_scale=``.
Inference only (no autograd). CUDA tensors only.
"""

from __future__ import annotations

import torch

from . import _lib
from ._lib import DTYPE_CODE, E4M3_CODE, call, device_of, ptr, stream_of
from .decode import CACHE_8BIT, _check_paged, check_scale, dense_rows
from .qk_norm_rope import check_table


CACHE_CODE = {**DTYPE_CODE, CACHE_8BIT: E4M3_CODE}


def _check_cache(name, heads, dim, dtype, device, cache, scale):
    shape = cache.shape
    if len(shape) != 4 or shape[2] != heads or shape[3] != dim:
        raise ValueError(f"expected {name}_cache[P,S,G,D] with {name}'s G and D")
    if cache.device != device:
        raise ValueError("All inputs must reside on the same device.")
    if shape[1] < 1:
        raise ValueError("pages must hold at least one token")
    kind = cache.dtype
    if kind == CACHE_8BIT:
        check_scale(f"{name}_scale", scale, shape[0], heads, device)
    elif kind != dtype:
        raise TypeError("a cache must have the inputs' dtype or float8_e4m3fn")
    elif scale is not None:
        raise ValueError(f"{name}_scale belongs to an 8-bit cache")
    # written in place: head rows must be dense, and no two elements may share memory
    if cache.is_contiguous():
        return
    if dim > 1 and cache.stride(3) != 1:
        raise ValueError(f"{name}_cache must have dense head rows")
    span = 1
    for stride, size in sorted((cache.stride(i), shape[i]) for i in range(4) if shape[i] > 1):
        if stride < span:
            raise ValueError(f"{name}_cache must not overlap itself")
        span = stride * size


def m3_cache_append(
    k: torch.Tensor,
    v: torch.Tensor | None,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor | None,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    *,
    cu_seqlens: torch.Tensor | None = None,
    rope_table: torch.Tensor | None = None,
    interleaved: bool = False,
    k_scale: torch.Tensor | None = None,
    v_scale: torch.Tensor | None = None,
) -> None:
    """Store the newest tokens ``k[T,G,D]`` (and ``v``, or None) of B requests in their pages.

    ``seq_lens[B]`` (int32) counts each request's tokens with the new ones; request b's new
    rows are ``cu_seqlens[b] .. cu_seqlens[b+1] - 1`` (int32 ``[B + 1]``, on the device, not read
    by the host), or row b without ``cu_seqlens`` (``T = B``), and take its last positions.
    ``rope_table`` rotates the keys as ``m3_qk_norm_rope`` does (NaN where a position lies outside
    it); without it, or with one of width 0, they are stored as they are. Caches ``[P,S,G,D]`` are
    written in place; ``k_scale`` / ``v_scale`` (positive) come with 8-bit ones, whose values that are
    not finite are stored as NaN. Skipped, with nothing written: rows behind ``cu_seqlens[B]``,
    requests of length 0 (a padded batch), pages past the block table's width or outside the cache.
    A page that receives tokens must belong to one request. Pages of 2^31 elements a head are refused where
    head rows are not whole aligned vectors, of 2^34 in 8 bits.
    """
    if k.ndim != 3 or (v is not None and v.shape != k.shape):
        raise ValueError("expected k[T,G,D] and a matching v")
    if (v is None) != (v_cache is None):
        raise ValueError("v and v_cache go together")
    dtype, device = k.dtype, k.device
    if dtype not in DTYPE_CODE or (v is not None and v.dtype != dtype):
        raise TypeError("k/v must share a BF16, FP16, or FP32 dtype.")
    total, heads, dim = k.shape
    if heads <= 0 or dim <= 0:
        raise ValueError("expected at least one head and a positive head dimension")
    _check_cache("k", heads, dim, dtype, device, k_cache, k_scale)
    if v is not None:
        if v.device != device:
            raise ValueError("All inputs must reside on the same device.")
        _check_cache("v", heads, dim, dtype, device, v_cache, v_scale)
        if v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype:
            raise ValueError("k_cache and v_cache must share their pages and dtype")
        if k_cache.data_ptr() == v_cache.data_ptr() and k_cache.numel() or (
                v_scale is not None and k_scale.data_ptr() == v_scale.data_ptr() and k_scale.numel()):
            raise ValueError("k and v need caches and scales of their own")
    elif v_scale is not None:
        raise ValueError("v_scale belongs to an 8-bit cache")
    if seq_lens.ndim != 1:
        raise ValueError("seq_lens must be int32 [B]")
    batch = seq_lens.shape[0]
    _check_paged(block_table, seq_lens, batch, device)
    if cu_seqlens is None:
        if total != batch:
            raise ValueError("without cu_seqlens, k holds one token per request")
    elif cu_seqlens.shape != (batch + 1,) or cu_seqlens.dtype != torch.int32:
        raise ValueError("cu_seqlens must be int32 [B + 1]")
    elif cu_seqlens.device != device:
        raise ValueError("All inputs must reside on the same device.")
    if rope_table is not None:
        check_table(rope_table, dim, device)
    _lib.require_cuda(k)
    # every copy is held by name until the launch: a temporary's memory would be handed to the next one
    k = dense_rows(k)
    v_ptr = v_cache_ptr = None
    v_strides, v_cache_strides = (0, 0, 0), (0, 0, 0, 0)
    if v is not None:
        v = dense_rows(v)
        v_ptr, v_cache_ptr, v_strides, v_cache_strides = v.data_ptr(), v_cache.data_ptr(), v.stride(), v_cache.stride()
    rows = rotary = 0
    if rope_table is not None:
        rope_table = rope_table.contiguous()
        rows, rotary = rope_table.shape
    if cu_seqlens is not None:
        cu_seqlens = cu_seqlens.contiguous()
    block_table, seq_lens = block_table.contiguous(), seq_lens.contiguous()
    pages, page_size, _, _ = k_cache.shape
    k_strides, k_cache_strides = k.stride(), k_cache.stride()
    with device_of(k):
        call("msa_cache_append", k.data_ptr(), v_ptr, DTYPE_CODE[dtype], k_strides[0], k_strides[1], v_strides[0],
             v_strides[1], ptr(rope_table), rows, rotary, interleaved, ptr(cu_seqlens), block_table.data_ptr(),
             seq_lens.data_ptr(), batch, total, heads, dim, page_size, block_table.shape[1], pages,
             k_cache.data_ptr(), v_cache_ptr, CACHE_CODE[k_cache.dtype], k_cache_strides[0], k_cache_strides[1],
             k_cache_strides[2], v_cache_strides[0], v_cache_strides[1], v_cache_strides[2], ptr(k_scale),
             ptr(v_scale), stream_of(k))
