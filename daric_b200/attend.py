"""Attention over the paged KV cache: full (with a tree of drafted tokens) and
over the pages that a selection lists for each query row.

The batch: sequence ``b`` has ``seq_lens[b]`` cache positions whose slots come
from ``block_table[b]``; its query rows ``q[cu_q[b]:cu_q[b + 1]]`` stand at its
last positions, so their keys and values are in the cache already (one row per
sequence: a decode step). Lengths, offsets and tables are device tensors and
nothing waits for the GPU: a call can be captured into a CUDA graph and
replayed while the tensors' values change. A block id outside the cache is
skipped like a key that does not exist, a length past the block table is cut
off, and both set a device error bit (``_lib.device_errors``).
"""
from __future__ import annotations

import ctypes as C
import math
import threading
from typing import Optional

import torch

from . import _lib
from ._lib import check
from .cache_ops import CacheCopier, kv_dtype_code

__all__ = ["tree_attention", "sparse_attention"]

class _Workspaces(threading.local):
    def __init__(self):
        self.of: dict[tuple, torch.Tensor] = {}


_workspaces = _Workspaces()
_raw_stream = torch._C._cuda_getCurrentRawStream
_capturing = torch.cuda.is_current_stream_capturing


def layer_tensor(copier: CacheCopier, layer_name: str) -> torch.Tensor:
    kv = copier._layers.get(layer_name)
    if kv is None:
        raise RuntimeError(f"layer not registered: {layer_name}")
    return kv


def kv_heads_of(kv: torch.Tensor) -> int:
    return kv.shape[3] if kv.dim() == 5 else kv.shape[1] if kv.dim() == 4 else -1


def check_rows(q: torch.Tensor, dev: torch.device, dtype: torch.dtype) -> None:
    if q.device != dev or q.dtype != dtype:
        raise RuntimeError(f"q must be {dtype} on {dev} like the KV cache, got {q.dtype} on {q.device}")
    if q.dim() != 3 or q.stride(2) != 1:
        raise RuntimeError("q must be a [rows, heads, head_dim] tensor with unit last stride")


def check_batch(dev: torch.device, block_table: torch.Tensor, seq_lens: torch.Tensor, cu_q: Optional[torch.Tensor]) -> int:
    """Checks the batch's tables; returns the number of sequences."""
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.device != dev or \
            (block_table.stride(1) != 1 and block_table.shape[1] > 1):
        raise RuntimeError("block_table must be an int32 [sequences, pages] matrix with unit column stride on the cache's device")
    n = block_table.shape[0]
    if seq_lens.dtype != torch.int32 or seq_lens.shape != (n,) or seq_lens.device != dev or not seq_lens.is_contiguous():
        raise RuntimeError("seq_lens must be a contiguous int32 vector, one entry per sequence, on the cache's device")
    if cu_q is not None and (cu_q.dtype != torch.int32 or cu_q.shape != (n + 1,) or cu_q.device != dev
                             or not cu_q.is_contiguous()):
        raise RuntimeError("cu_q must be a contiguous int32 vector of sequences + 1 entries on the cache's device")
    return n


def check_mask(tree_mask: Optional[torch.Tensor], rows: int, dev: torch.device) -> int:
    """Words per row of a tree mask (0: no mask)."""
    if tree_mask is None:
        return 0
    if tree_mask.device != dev or tree_mask.dtype != torch.int64 or tree_mask.dim() not in (1, 2) or \
            tree_mask.shape[0] != rows or not tree_mask.is_contiguous() or tree_mask.numel() == 0 < rows:
        raise RuntimeError("tree_mask must be a contiguous int64 [rows] or [rows, words] tensor on the cache's device")
    return 1 if tree_mask.dim() == 1 else tree_mask.shape[1]


def check_lse(lse: torch.Tensor, q: torch.Tensor) -> None:
    if lse.device != q.device or lse.dtype != torch.float32 or lse.shape != q.shape[:2] or \
            (lse.shape[1] > 1 and lse.stride(1) != 1):
        raise RuntimeError("lse must be a float32 [rows, heads] matrix with unit column stride on q's device")


class on_stream:
    """A call on the stream of the given handle: allocations are made on the
    stream that uses them, and the caller's tensors are kept from reuse until
    that stream is done with them."""

    def __init__(self, stream: int, dev: torch.device, *tensors):
        ext = torch.cuda.ExternalStream(stream, device=dev)
        self.ctx = torch.cuda.stream(ext)
        for t in tensors:
            if t is not None:
                t.record_stream(ext)

    def __enter__(self):
        return self.ctx.__enter__()

    def __exit__(self, *exc):
        return self.ctx.__exit__(*exc)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stays(dev: torch.device, stream: int) -> bool:
    """Whether the current stream of ``dev``, of the given handle, is one of
    torch's own, which live as long as the process (the handle of any other may
    come back as another stream), and captures nothing (which is asked of the
    current device's stream)."""
    return (stream == 0 or torch._C._cuda_getCurrentStream(dev.index)[0] != stream) and \
        torch.cuda.current_device() == dev.index and not _capturing()


def _kept(key: tuple, kept: bool, dev: torch.device, size) -> torch.Tensor:
    """Workspace of a call. The calls of one thread on one stream follow each
    other, so they share one that is kept (a call is several launches, and
    those of two threads may take turns on a stream); a captured call has its
    own, which belongs to its graph, and so has one on a stream that is not
    torch's. ``key`` starts with the device's index, head_dim and the stream;
    ``size`` fills in the bytes (39 MB for head_dim 128, 20 MB for 64 and
    256)."""
    kept = kept and _stays(dev, key[2])
    ws = _workspaces.of.get(key) if kept else None
    if ws is None:
        v = C.c_int64(0)
        check(size(C.byref(v)))
        ws = torch.empty(v.value, dtype=torch.uint8, device=dev)
        if kept:
            _workspaces.of[key] = ws
    return ws


def _attend_workspace(dev: torch.device, head_dim: int, stream: int, kept: bool) -> torch.Tensor:
    return _kept((dev.index, head_dim, stream), kept, dev,
                 lambda v: _lib.load().daric_attend_workspace(dev.index, head_dim, v))


def _outputs(q, out, lse):
    if out is None:
        out = q.new_empty(q.shape)
    elif out.device != q.device or out.dtype != q.dtype or out.shape != q.shape or out.stride(2) != 1:
        raise RuntimeError("out must be like q: same shape, dtype and device, unit last stride")
    if lse is None:
        lse = q.new_empty(q.shape[:2], dtype=torch.float32)
    else:
        check_lse(lse, q)
    return out, lse


def tree_attention(copier: CacheCopier, layer_name: str, q: torch.Tensor, block_table: torch.Tensor,
                   seq_lens: torch.Tensor, *, cu_q: Optional[torch.Tensor] = None,
                   tree_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                   out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                   stream: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """Softmax attention of every query row over its sequence's cache.

    ``q`` is [rows, query heads, head_dim] in the cache's dtype (bfloat16 or
    float16; head_dim 64, 128 or 256); query heads are a multiple of the
    layer's KV heads. Row ``j`` of a sequence of ``T`` rows and length ``s``
    sees the first ``s - T`` positions and, of the last ``T`` (the drafted
    tokens), token ``i`` where bit ``i % 64`` of ``tree_mask[row, i // 64]`` is
    set; without a mask the tokens up to its own. Without ``cu_q`` the rows
    divide evenly over the sequences. ``scale`` (positive) defaults to
    1 / sqrt(head_dim). Nothing is recorded for a backward pass.

    Returns (out [rows, heads, head_dim], lse [rows, heads] float32: natural
    log of the sum of exp of the scaled logits). A row that sees nothing gets
    out 0 and lse -inf. Rows outside every sequence are not written."""
    kv = layer_tensor(copier, layer_name)
    dev = kv.device
    check_rows(q, dev, kv.dtype)
    n = check_batch(dev, block_table, seq_lens, cu_q)
    rows, heads, dim = q.shape
    words = check_mask(tree_mask, rows, dev)
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    if stream:
        with on_stream(stream, dev, q, block_table, seq_lens, cu_q, tree_mask, out, lse):
            return _tree(copier, layer_name, kv, q, block_table, seq_lens, cu_q, tree_mask, words, n, scale, out, lse, False)
    return _tree(copier, layer_name, kv, q, block_table, seq_lens, cu_q, tree_mask, words, n, scale, out, lse, True)


def _tree(copier, layer_name, kv, q, block_table, seq_lens, cu_q, tree_mask, words, n, scale, out, lse, kept):
    out, lse = _outputs(q, out, lse)
    rows, heads, dim = q.shape
    if n == 0 or rows == 0:
        return out, lse
    dev = kv.device
    s = _raw_stream(dev.index)
    ws = _attend_workspace(dev, dim, s, kept)
    check(_lib.load().daric_copier_tree_attention(
        copier._h, layer_name.encode(), kv_dtype_code(kv.dtype), q.data_ptr(), q.stride(0), q.stride(1), rows,
        heads, dim, block_table.data_ptr(), block_table.stride(0), n, block_table.shape[1], seq_lens.data_ptr(),
        _ptr(cu_q), _ptr(tree_mask), words, scale, out.data_ptr(), out.stride(0), out.stride(1), lse.data_ptr(),
        lse.stride(0), ws.data_ptr(), ws.numel(), dev.index, s))
    return out, lse


def sparse_attention(copier: CacheCopier, layer_name: str, q: torch.Tensor, pages: torch.Tensor,
                     block_table: torch.Tensor, seq_lens: torch.Tensor, *, cu_q: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                     lse: Optional[torch.Tensor] = None, stream: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """Softmax attention of every query row over the pages listed for it.

    ``pages`` is int32 [rows, KV heads, k]: page numbers of the row's sequence
    (columns of its block table) as :func:`daric_b200.blocks.select_pages`
    returns them, ascending; negative entries are empty, an entry past the block
    table is skipped and sets a device error bit, and one that repeats the entry
    before it counts once. A row sees the listed positions up to its own. The rest is as in
    :func:`tree_attention` (without a mask)."""
    kv = layer_tensor(copier, layer_name)
    dev = kv.device
    check_rows(q, dev, kv.dtype)
    n = check_batch(dev, block_table, seq_lens, cu_q)
    rows, heads, dim = q.shape
    if pages.device != dev or pages.dtype != torch.int32 or pages.dim() != 3 or pages.shape[0] != rows or \
            (pages.shape[2] > 1 and pages.stride(2) != 1):
        raise RuntimeError("pages must be an int32 [rows, KV heads, k] tensor with unit last stride on the cache's device")
    kv_heads = kv_heads_of(kv)
    if pages.shape[1] != kv_heads:
        raise RuntimeError(f"pages must list pages for each of the {kv_heads} KV heads, got {pages.shape[1]}")
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    if stream:
        with on_stream(stream, dev, q, pages, block_table, seq_lens, cu_q, out, lse):
            return _sparse(copier, layer_name, kv, q, pages, block_table, seq_lens, cu_q, n, scale, out, lse, False)
    return _sparse(copier, layer_name, kv, q, pages, block_table, seq_lens, cu_q, n, scale, out, lse, True)


def _sparse(copier, layer_name, kv, q, pages, block_table, seq_lens, cu_q, n, scale, out, lse, kept):
    out, lse = _outputs(q, out, lse)
    rows, heads, dim = q.shape
    if n == 0 or rows == 0:
        return out, lse
    dev = kv.device
    s = _raw_stream(dev.index)
    # a shape of few rows needs what any such call does; lists of many rows
    # have sizes of their own and are not kept
    sizes = (rows, n, heads, pages.shape[1], pages.shape[2], block_table.shape[1])
    few = rows * heads < 128 * n * pages.shape[1]
    ws = _kept((dev.index, dim, s, "sparse"), kept and few, dev,
               lambda v: _lib.load().daric_sparse_workspace(dev.index, dim, *sizes, v))
    check(_lib.load().daric_copier_sparse_attention(
        copier._h, layer_name.encode(), kv_dtype_code(kv.dtype), q.data_ptr(), q.stride(0), q.stride(1), rows,
        heads, dim, pages.data_ptr(), pages.stride(0), pages.stride(1), pages.shape[2], block_table.data_ptr(),
        block_table.stride(0), n, block_table.shape[1], seq_lens.data_ptr(), _ptr(cu_q), scale, out.data_ptr(),
        out.stride(0), out.stride(1), lse.data_ptr(), lse.stride(0), ws.data_ptr(), ws.numel(), dev.index, s))
    return out, lse
