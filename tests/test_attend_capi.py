"""Refusals of the paged-cache operators' C entries: every one of them is made
before anything reaches a GPU, so the pointers here are never followed."""
import ctypes as C

import pytest
import torch

from daric_b200 import _lib

# Where a GPU is there, a call that was not refused would reach it.
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="pointers that lead nowhere")

P = C.c_void_p(0x10000)
ODD = C.c_void_p(0x10008)
BF16, F16, F32, FP8 = _lib.DTYPE_BF16, _lib.DTYPE_F16, _lib.DTYPE_F32, _lib.DTYPE_FP8_E4M3


class Calls:
    """A copier with layers l0, l1 (bf16 [2, 9, 16, 2, 128]), l2 (80-wide
    heads), l3 (fp32) and x (3-D), and each entry with arguments that pass."""

    def __init__(self):
        self.lib = _lib.load()
        self.h = C.c_void_p()
        _lib.check(self.lib.daric_copier_create(C.byref(self.h)))
        self.layer(b"l0", [2, 9, 16, 2, 128], 2, 0x100000)
        self.layer(b"l1", [2, 9, 16, 2, 128], 2, 0x900000)
        self.layer(b"l2", [2, 9, 16, 2, 80], 2, 0x100000)
        self.layer(b"l3", [2, 9, 16, 2, 128], 4, 0x100000)
        self.layer(b"l4", [2, 8, 16, 2, 128], 2, 0x100000)
        self.layer(b"x", [9, 16, 256], 2, 0x100000, page_first=1)
        self.layer(b"big", [2, 9, 1025, 2, 128], 2, 0x100000)
        self.layer(b"off", [2, 9, 16, 2, 128], 2, 0x100008)

    def layer(self, name, sizes, es, at, page_first=0):
        st = [1]
        for n in reversed(sizes[1:]):
            st.insert(0, st[0] * n)
        _, sp = _lib.i64(sizes)
        keep, tp = _lib.i64(st)
        s, sp = _lib.i64(sizes)
        _lib.check(self.lib.daric_copier_register_layer(self.h, name, C.c_void_p(at), 0, len(sizes), sp, tp, es, page_first))

    def run(self, entry, base, **kw):
        args = {**base, **kw}
        return getattr(self.lib, entry)(*args.values())

    def tree(self, **kw):
        return self.run("daric_copier_tree_attention", dict(
            h=self.h, name=b"l0", dt=BF16, q=P, q_row=1024, q_head=128, rows=2, heads=8, dim=128, table=P, ld=4, n=2, cols=4,
            lens=P, cu=None, mask=None, words=0, scale=1.0, out=P, out_row=1024, out_head=128, lse=None, lse_row=8, ws=P,
            ws_bytes=1 << 40, device=0, stream=None), **kw)

    def sparse(self, **kw):
        return self.run("daric_copier_sparse_attention", dict(
            h=self.h, name=b"l0", dt=BF16, q=P, q_row=1024, q_head=128, rows=2, heads=8, dim=128, pages=P, p_row=4, p_head=2,
            k=2, table=P, ld=4, n=2, cols=4, lens=P, cu=None, scale=1.0, out=P, out_row=1024, out_head=128, lse=None,
            lse_row=8, ws=P, ws_bytes=1 << 40, device=0, stream=None), **kw)

    def bounds(self, **kw):
        return self.run("daric_copier_page_bounds", dict(
            h=self.h, name=b"l0", dt=BF16, table=P, ld=4, n=2, cols=4, lens=P, start=None, bounds=P, device=0, stream=None),
            **kw)

    def select(self, **kw):
        return self.run("daric_select_pages", dict(
            q=P, dt=BF16, q_row=1024, q_head=128, rows=2, heads=8, dim=128, bounds=P, pages=9, kvh=2, table=P, ld=4, n=2,
            cols=4, lens=P, cu=None, bs=16, k=3, first=1, last=1, out=P, ws=P, ws_bytes=1 << 40, device=0, stream=None), **kw)

    def scores(self, **kw):
        return self.run("daric_copier_attention_scores", dict(
            h=self.h, name=b"l0", dt=BF16, q=P, q_row=1024, q_head=128, rows=2, heads=8, dim=128, table=P, ld=4, n=2, cols=4,
            lens=P, cu=None, mask=None, words=0, lse=P, lse_row=8, scale=1.0, scores=P, s_row=64, s_cols=64, off=P, acc=1,
            ws=None, ws_bytes=0, device=0, stream=None), **kw)

    def compact(self, names=(b"l0", b"l1"), off=(0, 3), cap=(3, 4), blk=(0, 4), dst=(0, 1), **kw):
        arrays = [_lib.i64(list(x)) if x is not None else (None, None) for x in (off, cap, blk, dst)]
        ptrs = [a[1] for a in arrays]
        return self.run("daric_copier_compact", dict(
            h=self.h, n=len(names), names=_lib.names_array([x.decode() for x in names]), dt=BF16, mode=_lib.ROPE_NONE, lists=2,
            per_head=0, idx=P, idx_row=8, count=P, count_row=2, segs=2, off=ptrs[0], cap=ptrs[1], blk=ptrs[2], dst=ptrs[3],
            table=P, numel=8, device=0, stream=None), **kw)


@pytest.fixture(scope="module")
def calls():
    c = Calls()
    yield c
    c.lib.daric_copier_destroy(c.h)


def refused(calls, rc, match):
    assert rc == _lib.ERR_INVALID, calls.lib.daric_last_error()
    assert match.encode() in calls.lib.daric_last_error(), calls.lib.daric_last_error()


BATCH = [  # of every call over a batch of rows
    (dict(table=None), "NULL block table"), (dict(lens=None), "NULL block table or lengths"), (dict(n=0), "positive"),
    (dict(cols=0), "positive"), (dict(n=65536, ld=4), "65535"), (dict(ld=3), "overlap"),
    (dict(cols=1 << 28, ld=1 << 28), "int32 positions"),
]
ROWS = BATCH + [
    (dict(rows=-1), "positive"), (dict(rows=3), "divide evenly"), (dict(heads=7), "multiple"), (dict(heads=1), "multiple"),
    (dict(heads=0), "multiple"), (dict(rows=1 << 30), "too many query rows"),
]
LAYER = [
    (dict(name=b"nope"), "not registered"), (dict(h=None), "copier is NULL"), (dict(device=1), "on the KV cache's device"),
    (dict(dt=F32), "bfloat16 or float16"), (dict(dt=FP8), "bfloat16 or float16"), (dict(dt=99), "bfloat16 or float16"),
    (dict(name=b"l3"), "element size"), (dict(name=b"x"), "5-D or packed 4-D"), (dict(name=b"big"), "block size"),
    (dict(name=b"off"), "16-byte aligned"),
]
SCALES = [(dict(scale=s), "scale") for s in (0.0, -1.0, float("inf"), float("nan"))]
ALIGN = [(dict(q=ODD), "query rows must be 16-byte aligned"), (dict(q_row=1028), "query rows must be 16-byte aligned"),
         (dict(q_head=132), "query rows must be 16-byte aligned"), (dict(q=None), "NULL query")]
OUT = [(dict(out=ODD), "output rows must be 16-byte aligned"), (dict(out_row=1028), "output rows must be 16-byte aligned"),
       (dict(out=None), "NULL query")]
MASK = [(dict(mask=P, words=0), "tree mask"), (dict(mask=P, words=(1 << 25) + 1), "tree mask")]


@pytest.mark.parametrize("kw,match", ROWS + LAYER + SCALES + ALIGN + OUT + MASK + [(dict(dim=64), "head dimension"),
                                                                                   (dict(name=b"l2"), "head dimension")])
def test_tree_attention(calls, kw, match):
    refused(calls, calls.tree(**kw), match)


@pytest.mark.parametrize("kw,match", ROWS + LAYER + SCALES + ALIGN + OUT + [(dict(pages=None), "page list"), (dict(k=0), "at least one"),
                                                                           (dict(k=1 << 30), "at least one")])
def test_sparse_attention(calls, kw, match):
    refused(calls, calls.sparse(**kw), match)


@pytest.mark.parametrize("kw,match", BATCH + LAYER + [(dict(bounds=None), "bounds"), (dict(bounds=ODD), "bounds")])
def test_page_bounds(calls, kw, match):
    refused(calls, calls.bounds(**kw), match)


@pytest.mark.parametrize("kw,match", ROWS + ALIGN + [
    (dict(dt=F32), "bfloat16 or float16"), (dict(dim=80), "64, 128 or 256"), (dict(kvh=0), "bounds sizes"), (dict(pages=0), "bounds sizes"),
    (dict(bs=0), "block size"), (dict(bs=1025), "block size"), (dict(k=0), "k must hold"), (dict(last=0), "k must hold"),
    (dict(first=-1), "k must hold"), (dict(first=2, last=2), "k must hold"), (dict(cols=(1 << 20) + 1, ld=1 << 21), "1048576"),
    (dict(bounds=None), "NULL"), (dict(bounds=ODD), "bounds must be"), (dict(out=None), "NULL"), (dict(ws=None), "workspace"),
    (dict(ws=ODD), "workspace"), (dict(ws_bytes=16), "too small")])
def test_select_pages(calls, kw, match):
    if kw.get("cols") == 1 << 28:
        match = "1048576"  # asked first here
    refused(calls, calls.select(**kw), match)


@pytest.mark.parametrize("kw,match", ROWS + LAYER + SCALES + ALIGN + MASK + [
    (dict(scores=None), "NULL"), (dict(off=None), "NULL"), (dict(s_row=63), "overlap"), (dict(s_cols=-1), "overlap"),
    (dict(cols=1 << 21, ld=1 << 21), "16.7M")])
def test_attention_scores(calls, kw, match):
    refused(calls, calls.scores(**kw), match)


@pytest.mark.parametrize("kw,match", [
    (dict(h=None), "copier is NULL"), (dict(mode=_lib.ROPE_DELTA), "mode"), (dict(idx=None), "NULL"), (dict(count=None), "NULL"),
    (dict(off=None), "NULL"), (dict(cap=None), "NULL"), (dict(table=None), "block_table"), (dict(dt=99), "unknown KV dtype"),
    (dict(dt=F32), "element size"), (dict(dt=FP8), "element size"), (dict(device=1), "on the KV cache's device"),
    (dict(names=(b"l0", b"nope")), "not registered"), (dict(names=(b"l0", b"l4")), "share block size"),
    (dict(names=(b"l0", b"l0")), "twice"), (dict(lists=3), "one row per layer"), (dict(per_head=1, lists=3), "one row per layer"),
    (dict(mode=_lib.ROPE_FLEXIBLE), "no rotary table")])
def test_compact(calls, kw, match):
    refused(calls, calls.compact(**kw), match)


def test_empty_calls_return_without_a_gpu(calls):
    """Nothing to do: no rows, no layers, no segments."""
    assert calls.tree(rows=0) == 0 and calls.sparse(rows=0) == 0 and calls.select(rows=0) == 0
    assert calls.compact(n=0) == 0 and calls.compact(segs=0) == 0


def test_workspace_sizes(calls):
    v = C.c_int64(0)
    lib = calls.lib
    for fn, args in ((lib.daric_select_pages_workspace, (4, 2, 100)), (lib.daric_scores_workspace, (4, 8, 100, 16))):
        _lib.check(fn(*args, C.byref(v)))
        small = v.value
        _lib.check(fn(args[0] * 2, *args[1:], C.byref(v)))
        assert 0 < small < v.value
        assert fn(*args, None) == _lib.ERR_INVALID
        assert fn(-1, *args[1:], C.byref(v)) == _lib.ERR_INVALID
    refused(calls, lib.daric_attend_workspace(0, 257, C.byref(v)), "head dimension")
    refused(calls, lib.daric_attend_workspace(0, 0, C.byref(v)), "head dimension")
    refused(calls, lib.daric_attend_workspace(0, 128, None), "out_bytes")
    refused(calls, lib.daric_sparse_workspace(0, 128, 4, 0, 8, 2, 3, 4, C.byref(v)), "positive")
    refused(calls, lib.daric_sparse_workspace(0, 128, 4, 2, 8, 2, 0, 4, C.byref(v)), "positive")
    refused(calls, lib.daric_sparse_workspace(0, 512, 4, 2, 8, 2, 3, 4, C.byref(v)), "head dimension")


BIG = (1 << 63) - 1


@pytest.mark.parametrize("entry,kw,match", [
    ("select", dict(first=1 << 62, last=1 << 62), "k must hold"), ("select", dict(first=BIG, last=BIG), "k must hold"),
    ("compact", dict(dst=(0, BIG)), "exceed int32"), ("compact", dict(dst=(0, BIG - 3)), "exceed int32"),
    ("compact", dict(off=(0, BIG)), "exceeds the selection's row"), ("compact", dict(cap=(3, BIG)), "exceeds the selection's row"),
    ("compact", dict(dst=(0, (1 << 31) - 4)), "exceed int32")])
def test_values_whose_sums_pass_64_bits(calls, entry, kw, match):
    refused(calls, getattr(calls, entry)(**kw), match)


@pytest.mark.parametrize("entry", ["tree", "sparse", "bounds", "select", "scores"])
@pytest.mark.parametrize("cols", [(1 << 27) - 1, (1 << 27) - 64, BIG // 16 + 1, BIG])
def test_tables_that_end_beside_2_to_31(calls, entry, cols):
    """Positions behind the last one are counted in 32 bits, too."""
    refused(calls, getattr(calls, entry)(cols=cols, ld=cols), "1048576" if entry == "select" else "int32 positions")


@pytest.mark.parametrize("kw,match", [(dict(k=(1 << 27) - 1), "positions"), (dict(k=BIG // 16 + 1), "positions"), (dict(k=BIG), "positions"),
                                      (dict(rows=BIG - 1), "too many query rows"), (dict(rows=1 << 61), "too many query rows")])
def test_lists_and_rows_that_pass_their_range(calls, kw, match):
    refused(calls, calls.sparse(**kw), match)
