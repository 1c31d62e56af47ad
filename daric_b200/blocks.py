"""Selection of cache pages by a cheap score, for sparse attention.

A page's keys are summed up by their smallest and largest value per dimension
(``page_bounds``, kept by the caller and refreshed for the pages that change);
``select_pages`` bounds each query's logits over a page from them and lists the
pages of highest bound, which :func:`daric_b200.attend.sparse_attention` reads.
Batches are described as in :mod:`daric_b200.attend`.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib
from ._lib import check
from .attend import check_batch, check_rows, layer_tensor, on_stream, _ptr, _raw_stream
from .cache_ops import CacheCopier, kv_dtype_code

__all__ = ["new_bounds", "page_bounds", "select_pages"]


def _dims(kv: torch.Tensor, page_first: bool) -> tuple[int, int, int]:
    """(blocks, KV heads, head_dim) of a layer tensor."""
    if kv.dim() == 5:
        return kv.shape[0 if page_first else 1], kv.shape[3], kv.shape[4]
    if kv.dim() == 4:
        return kv.shape[0], kv.shape[1], kv.shape[3] // 2
    raise RuntimeError(f"KV cache must be 5-D or packed 4-D to hold K and V rows, got {kv.dim()}-D")


def new_bounds(copier: CacheCopier, layer_name: str) -> torch.Tensor:
    """Room for a layer's page bounds: [blocks, KV heads, 2, head_dim] in the
    cache's dtype (index 0 of the third dimension: minima, 1: maxima)."""
    kv = layer_tensor(copier, layer_name)
    nb, heads, dim = _dims(kv, copier._page_first[layer_name])
    return torch.zeros((nb, heads, 2, dim), dtype=kv.dtype, device=kv.device)


def page_bounds(copier: CacheCopier, layer_name: str, block_table: torch.Tensor, seq_lens: torch.Tensor,
                bounds: Optional[torch.Tensor] = None, *, start: Optional[torch.Tensor] = None,
                stream: int = 0) -> torch.Tensor:
    """Writes the bounds of every page of every sequence that holds a position
    in [start[b], seq_lens[b]) (``start``: int32 [sequences], default 0; a
    decode step passes the position it wrote). Only tokens below ``seq_lens``
    count; a NaN key makes its dimension's bounds NaN. ``bounds`` is indexed by
    block id and may be shared by all sequences; sequences that share a partly
    filled block must have the same length in it."""
    kv = layer_tensor(copier, layer_name)
    dev = kv.device
    n = check_batch(dev, block_table, seq_lens, None)
    if start is not None and (start.device != dev or start.dtype != torch.int32 or start.shape != (n,)
                              or not start.is_contiguous()):
        raise RuntimeError("start must be a contiguous int32 vector, one entry per sequence, on the cache's device")
    nb, heads, dim = _dims(kv, copier._page_first[layer_name])
    if bounds is not None and (bounds.device != dev or bounds.dtype != kv.dtype
                               or bounds.shape != (nb, heads, 2, dim) or not bounds.is_contiguous()):
        raise RuntimeError(f"bounds must be a contiguous {kv.dtype} [{nb}, {heads}, 2, {dim}] tensor on {dev}")
    if stream:
        with on_stream(stream, dev, block_table, seq_lens, bounds, start):
            return page_bounds(copier, layer_name, block_table, seq_lens, bounds, start=start)
    if bounds is None:
        bounds = new_bounds(copier, layer_name)
    if n and block_table.shape[1]:
        check(_lib.load().daric_copier_page_bounds(
            copier._h, layer_name.encode(), kv_dtype_code(kv.dtype), block_table.data_ptr(), block_table.stride(0), n,
            block_table.shape[1], seq_lens.data_ptr(), _ptr(start), bounds.data_ptr(), dev.index,
            _raw_stream(dev.index)))
    return bounds


def select_pages(q: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, k: int,
                 block_size: int, *, cu_q: Optional[torch.Tensor] = None, first: int = 1, last: int = 1,
                 out: Optional[torch.Tensor] = None, stream: int = 0) -> torch.Tensor:
    """Pages for each query row and KV head: int32 [rows, KV heads, k],
    ascending, padded with -1.

    A row sees the pages up to the one of its own position. The first ``first``
    and the last ``last`` (at least 1) of them are always listed; the others by
    ``max over the group's query heads of sum_d max(q_d min_d, q_d max_d)``,
    highest first, ties to the lower page. The order is that of the score
    summed up in 64 bits, whatever the rounding of the fast pass. NaN (0 times
    an infinite bound among them) ranks highest. Rows outside every sequence are not written."""
    dev = q.device
    if not q.is_cuda:
        raise RuntimeError("q must be a CUDA tensor")
    check_rows(q, dev, q.dtype)
    n = check_batch(dev, block_table, seq_lens, cu_q)
    if bounds.device != dev or bounds.dtype != q.dtype or bounds.dim() != 4 or bounds.shape[2] != 2 or \
            bounds.shape[3] != q.shape[2] or not bounds.is_contiguous():
        raise RuntimeError("bounds must be a contiguous [blocks, KV heads, 2, head_dim] tensor of q's dtype and device")
    rows, heads, dim = q.shape
    nb, kv_heads = bounds.shape[:2]
    k = int(k)
    if out is not None and (out.device != dev or out.dtype != torch.int32 or out.shape != (rows, kv_heads, k)
                            or not out.is_contiguous()):
        raise RuntimeError(f"out must be a contiguous int32 [{rows}, {kv_heads}, {k}] tensor on {dev}")
    if stream:
        with on_stream(stream, dev, q, bounds, block_table, seq_lens, cu_q, out):
            return select_pages(q, bounds, block_table, seq_lens, k, block_size, cu_q=cu_q, first=first, last=last, out=out)
    if out is None:
        out = q.new_empty((rows, kv_heads, max(k, 0)), dtype=torch.int32)
    if n == 0 or rows == 0:
        return out
    cols = block_table.shape[1]
    size = C.c_int64(0)
    check(_lib.load().daric_select_pages_workspace(rows, kv_heads, cols, C.byref(size)))
    ws = q.new_empty(size.value, dtype=torch.uint8)
    check(_lib.load().daric_select_pages(
        q.data_ptr(), kv_dtype_code(q.dtype), q.stride(0), q.stride(1), rows, heads, dim, bounds.data_ptr(), nb,
        kv_heads, block_table.data_ptr(), block_table.stride(0), n, cols, seq_lens.data_ptr(), _ptr(cu_q),
        int(block_size), k, int(first), int(last), out.data_ptr(), ws.data_ptr(), size.value, dev.index,
        _raw_stream(dev.index)))
    return out
