"""Eviction from the paged KV cache by accumulated attention weight.

``attention_scores`` adds up the attention weight every cached token receives,
per KV head, into score rows that :func:`daric_b200.select.score_select` reads;
``compact`` moves the tokens of such a selection to the front of their block
tables (with their keys re-rotated to the new positions, where the cache's
positions are renumbered), which frees the blocks behind them. Batches are
described as in :mod:`daric_b200.attend`.
"""
from __future__ import annotations

import ctypes as C
import math
from collections.abc import Sequence
from typing import Optional

import numpy as np
import torch

from . import _lib
from ._lib import check, i64, names_array
from .attend import (check_batch, check_lse, check_mask, check_rows, kv_heads_of, layer_tensor, on_stream, _ptr,
                     _raw_stream)
from .cache_ops import CacheCopier, kv_dtype_code, mode_code
from .select import Selection

__all__ = ["attention_scores", "compact"]


def attention_scores(copier: CacheCopier, layer_name: str, q: torch.Tensor, block_table: torch.Tensor,
                     seq_lens: torch.Tensor, scores: torch.Tensor, col_off: torch.Tensor, *,
                     cu_q: Optional[torch.Tensor] = None, tree_mask: Optional[torch.Tensor] = None,
                     lse: Optional[torch.Tensor] = None, scale: Optional[float] = None, accumulate: bool = True,
                     stream: int = 0) -> torch.Tensor:
    """Attention weight of every cached token: for KV head h and position p of
    sequence b, ``scores[h, col_off[b] + p]`` gets (``accumulate``: is
    increased by) the sum of ``exp(scale q.k_p - lse)`` over the sequence's
    query rows that see p and the query heads of h.

    ``scores`` is float32 [KV heads, columns] with unit column stride,
    ``col_off`` int64 [sequences] on the device (the ``seg_col_off`` of
    ``score_select``); the columns of two sequences must not overlap. ``lse`` is what :func:`daric_b200.attend.tree_attention`
    returned for the same rows and mask; without it the log-sums are computed
    here. Rows with lse -inf add nothing. The sums have one fixed order.
    Returns ``scores``."""
    kv = layer_tensor(copier, layer_name)
    dev = kv.device
    check_rows(q, dev, kv.dtype)
    n = check_batch(dev, block_table, seq_lens, cu_q)
    rows, heads, dim = q.shape
    words = check_mask(tree_mask, rows, dev)
    if lse is not None:
        check_lse(lse, q)
    kv_heads = kv_heads_of(kv)
    if scores.device != dev or scores.dtype != torch.float32 or scores.dim() != 2 or scores.shape[0] != kv_heads or \
            (scores.shape[1] > 1 and scores.stride(1) != 1):
        raise RuntimeError(f"scores must be a float32 [{kv_heads}, columns] matrix with unit column stride on {dev}")
    if col_off.device != dev or col_off.dtype != torch.int64 or col_off.shape != (n,) or not col_off.is_contiguous():
        raise RuntimeError("col_off must be a contiguous int64 vector, one entry per sequence, on the cache's device")
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    cols = block_table.shape[1]
    if stream:
        with on_stream(stream, dev, q, block_table, seq_lens, scores, col_off, cu_q, tree_mask, lse):
            return attention_scores(copier, layer_name, q, block_table, seq_lens, scores, col_off, cu_q=cu_q,
                                    tree_mask=tree_mask, lse=lse, scale=scale, accumulate=accumulate)
    if n == 0 or cols == 0:
        return scores
    ws, ws_bytes = None, 0
    if lse is None and rows:
        size = C.c_int64(0)
        check(_lib.load().daric_scores_workspace(rows, heads, cols, kv.shape[2], C.byref(size)))
        ws_bytes = size.value
        ws = q.new_empty(ws_bytes, dtype=torch.uint8)
    check(_lib.load().daric_copier_attention_scores(
        copier._h, layer_name.encode(), kv_dtype_code(kv.dtype), q.data_ptr(), q.stride(0), q.stride(1), rows,
        heads, dim, block_table.data_ptr(), block_table.stride(0), n, cols, seq_lens.data_ptr(), _ptr(cu_q),
        _ptr(tree_mask), words, _ptr(lse), 0 if lse is None else lse.stride(0), scale, scores.data_ptr(),
        scores.stride(0), scores.shape[1], col_off.data_ptr(), 1 if accumulate else 0, _ptr(ws), ws_bytes, dev.index,
        _raw_stream(dev.index)))
    return scores


def compact(copier: CacheCopier, layer_names: Sequence[str], keep: Selection, block_table: torch.Tensor, *,
            per_head: bool = False, seg_blk_off: Optional[Sequence[int]] = None,
            dst_start: Optional[Sequence[int]] = None, mode="none", stream: int = 0) -> None:
    """Moves the kept tokens of every segment to positions ``dst_start[s]``,
    ``dst_start[s] + 1``, ... of its block table, K and V, in place, all layers
    per launch. Tokens that are not overwritten stay as they are. A block that
    is written must belong to one segment only (shared blocks are copied
    first, or left in front of ``dst_start``).

    ``keep`` is a :class:`daric_b200.select.Selection` (or one like it) whose
    ``idx`` rows hold ascending positions: one row per layer, or one row for
    all layers; with ``per_head`` one row per KV head in place of each (row
    ``layer * heads + head``). ``block_table`` is flat int32, segment s's
    blocks start at ``seg_blk_off[s]`` (default 0), as in ``score_select``.
    Token n of a segment must stand at ``dst_start[s] + n`` (default 0 + n) or
    later; one that does not, or that breaks the ascending order, is left out
    and sets a device error bit. ``mode`` "none" keeps keys as they are;
    "flexible" turns them from their old to their new position by the layers'
    rotary tables (register_rotary), in fp32, rounded once; a token that stays
    where it is is not touched. Works for every KV dtype."""
    names = list(layer_names)
    if not names or keep.idx.numel() == 0:
        return
    layers = copier._layers
    kv = layer_tensor(copier, names[0])
    dev, dtype = kv.device, kv.dtype
    for t, what in ((keep.idx, "keep.idx"), (keep.count, "keep.count")):
        if t.dtype != torch.int32 or t.dim() != 2 or t.device != dev or (t.shape[1] > 1 and t.stride(1) != 1):
            raise RuntimeError(f"{what} must be an int32 matrix with unit column stride on the cache's device")
    if block_table.dtype != torch.int32 or block_table.device != dev or not block_table.is_contiguous():
        raise RuntimeError("block_table must be a contiguous CUDA int32 tensor on the cache's device")
    if len(names) > 1 and any(name in layers and layers[name].dtype != dtype for name in names):
        raise RuntimeError("compact: layers of one call must share the KV dtype")
    lists, width = keep.idx.shape
    nseg = keep.count.shape[1]
    off, offp = i64(keep.out_off)
    if keep.count.shape[0] != lists or len(off) != nseg:
        raise RuntimeError("keep.count and keep.out_off must have one entry per row and segment")
    cap = np.empty(nseg, np.int64)  # room of each segment: up to the next one's entries
    np.subtract(off[1:], off[:-1], out=cap[:-1])
    cap[-1:] = width - off[-1:]
    blk, blkp = (None, None) if seg_blk_off is None else i64(seg_blk_off)
    dst, dstp = (None, None) if dst_start is None else i64(dst_start)
    if (blk is not None and len(blk) != nseg) or (dst is not None and len(dst) != nseg):
        raise RuntimeError("seg_blk_off and dst_start must have one entry per segment")
    if stream:
        with on_stream(stream, dev, keep.idx, keep.count, block_table):
            return compact(copier, names, keep, block_table, per_head=per_head, seg_blk_off=seg_blk_off,
                           dst_start=dst_start, mode=mode)
    check(_lib.load().daric_copier_compact(
        copier._h, len(names), names_array(names), kv_dtype_code(dtype), mode_code(mode), lists, 1 if per_head else 0,
        keep.idx.data_ptr(), keep.idx.stride(0), keep.count.data_ptr(), keep.count.stride(0), nseg, offp,
        cap.ctypes.data, blkp, dstp, block_table.data_ptr(), block_table.numel(), dev.index, _raw_stream(dev.index)))
