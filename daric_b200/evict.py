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
from .attend import check_batch, check_lse, check_mask, check_rows, layer_tensor, on_stream, _ptr
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
    ``score_select``). ``lse`` is what :func:`daric_b200.attend.tree_attention`
    returned for the same rows and mask; without it the log-sums are computed
    here. Rows with lse -inf add nothing. The sums have one fixed order.
    Returns ``scores``."""
    kv = layer_tensor(copier, layer_name)
    check_rows(q)
    dev = kv.device
    if q.device != dev or q.dtype != kv.dtype:
        raise RuntimeError(f"q must be {kv.dtype} on {dev} like the KV cache, got {q.dtype} on {q.device}")
    n = check_batch(dev, block_table, seq_lens, cu_q)
    rows, heads, dim = q.shape
    words = check_mask(tree_mask, rows, dev)
    if lse is not None:
        check_lse(lse, q)
    kv_heads = kv.shape[1] if kv.dim() == 4 else kv.shape[3] if kv.dim() == 5 else -1
    if scores.device != dev or scores.dtype != torch.float32 or scores.dim() != 2 or scores.shape[0] != kv_heads or \
            (scores.shape[1] > 1 and scores.stride(1) != 1):
        raise RuntimeError(f"scores must be a float32 [{kv_heads}, columns] matrix with unit column stride on {dev}")
    if col_off.device != dev or col_off.dtype != torch.int64 or col_off.shape != (n,) or not col_off.is_contiguous():
        raise RuntimeError("col_off must be a contiguous int64 vector, one entry per sequence, on the cache's device")
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    cols = block_table.shape[1]
    with on_stream(stream, dev, q, block_table, seq_lens, scores, col_off, cu_q, tree_mask, lse) as s:
        if n == 0 or cols == 0:
            return scores
        ws = None
        if lse is None and rows:
            block = kv.shape[2]
            splits = (cols * block + 255) // 256
            ws = torch.empty(rows * heads * (splits * 2 + 1) + 4, dtype=torch.float32, device=dev)
        check(_lib.load().daric_copier_attention_scores(
            copier._h, layer_name.encode(), kv_dtype_code(kv.dtype), q.data_ptr(), q.stride(0), q.stride(1), rows,
            heads, dim, block_table.data_ptr(), block_table.stride(0), n, cols, seq_lens.data_ptr(), _ptr(cu_q),
            _ptr(tree_mask), words, _ptr(lse), 0 if lse is None else lse.stride(0), scale, scores.data_ptr(),
            scores.stride(0), scores.shape[1], col_off.data_ptr(), int(bool(accumulate)), _ptr(ws),
            0 if ws is None else ws.numel() * 4, dev.index, s))
    return scores


def compact(copier: CacheCopier, layer_names: Sequence[str], keep: Selection, block_table: torch.Tensor, *,
            per_head: bool = False, seg_blk_off: Optional[Sequence[int]] = None,
            dst_start: Optional[Sequence[int]] = None, mode="none", stream: int = 0) -> None:
    """Moves the kept tokens of every segment to positions ``dst_start[s]``,
    ``dst_start[s] + 1``, ... of its block table, K and V, in place, all layers
    per launch. Tokens that are not overwritten stay as they are.

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
    kv = layer_tensor(copier, names[0])
    dev = kv.device
    for t, what in ((keep.idx, "keep.idx"), (keep.count, "keep.count")):
        if t.device != dev or t.dtype != torch.int32 or t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
            raise RuntimeError(f"{what} must be an int32 matrix with unit column stride on the cache's device")
    if block_table.device != dev or block_table.dtype != torch.int32 or not block_table.is_contiguous():
        raise RuntimeError("block_table must be a contiguous CUDA int32 tensor on the cache's device")
    for name in names:
        if layer_tensor(copier, name).dtype != kv.dtype:
            raise RuntimeError("compact: layers of one call must share the KV dtype")
    lists, width = keep.idx.shape
    nseg = keep.count.shape[1]
    off, offp = i64(keep.out_off)
    if keep.count.shape[0] != lists or len(off) != nseg:
        raise RuntimeError("keep.count and keep.out_off must have one entry per row and segment")
    ends = np.append(off[1:], width)
    cap, capp = i64(ends - off)
    blk, blkp = i64(seg_blk_off if seg_blk_off is not None else [0] * nseg)
    dst, dstp = i64(dst_start if dst_start is not None else [0] * nseg)
    if len(blk) != nseg or len(dst) != nseg:
        raise RuntimeError("seg_blk_off and dst_start must have one entry per segment")
    with on_stream(stream, dev, keep.idx, keep.count, block_table) as s:
        check(_lib.load().daric_copier_compact(
            copier._h, len(names), names_array(names), kv_dtype_code(kv.dtype), mode_code(mode), lists,
            int(bool(per_head)), keep.idx.data_ptr(), keep.idx.stride(0), keep.count.data_ptr(), keep.count.stride(0),
            nseg, offp, capp, blkp, dstp, block_table.data_ptr(), block_table.numel(), dev.index, s))
