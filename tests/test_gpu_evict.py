"""Accumulated attention weights, compaction of the paged cache, and a whole
eviction: weights, selection, compaction, attention over what is left."""
import math

import numpy as np
import pytest
import torch

from daric_b200 import _lib
from daric_b200.attend import tree_attention
from daric_b200.cache_ops import CacheCopier
from daric_b200.evict import attention_scores, compact
from daric_b200.select import Selection, score_select
from attend_util import Batch, attend64, check_attend, planes, tree_masks

pytestmark = pytest.mark.gpu


def offsets(lens, gap=3):
    off, at = [], 2
    for n in lens:
        off.append(at)
        at += n + gap
    return off, at


def scores_ref(bt, b, mask, lse):
    """Weights in 64 bits [head, position] and their tolerance."""
    k, v = bt.kv64(b)
    q = bt.q64(b)
    ok = bt.sees(b, mask).repeat(bt.group, 1)[None]
    scale = 1 / math.sqrt(bt.d)
    _, own, _, e = attend64(q, k, v, ok, scale)
    z = own if lse is None else lse[bt.cu[b]:bt.cu[b + 1]].double().view(bt.rows[b], bt.kvh, bt.group).permute(1, 2, 0).reshape(own.shape)
    x = torch.matmul(q, k.transpose(1, 2)) * scale
    live = ok & (z != -math.inf)[..., None]
    w = torch.where(live, torch.exp(x - torch.where(z == -math.inf, 0.0, z)[..., None]), 0.0)
    # a weight is off by the errors of its logit, of the lse (twice a logit's where it is computed here, and its
    # rounding) and of exp: relative; the sum over n rows by n 2^-24
    rel = 3 * e + 2.0 ** -21 * (torch.where(z == -math.inf, 0.0, z).abs() + 4)
    tol = (w * (rel[..., None] * 1.01 + q.shape[1] * 2.0 ** -24)).sum(1)
    return w.sum(1), tol


def check_scores(bt, mask=None, lse=None, accumulate=True):
    off, cols = offsets(bt.lens)
    before = torch.rand((bt.kvh, cols), device="cuda")
    scores = before.clone()
    attention_scores(bt.copier, "l", bt.q, bt.table, bt.seq_lens, scores, torch.tensor(off, device="cuda"), cu_q=bt.cu_q,
                     tree_mask=None if mask is None else mask.cuda(), lse=lse, accumulate=accumulate)
    assert _lib.device_errors(0) == 0
    untouched = torch.ones(cols, dtype=torch.bool)
    for b, n in enumerate(bt.lens):
        at = slice(off[b], off[b] + n)
        untouched[at] = False
        if n == 0:
            continue
        ref, tol = scores_ref(bt, b, mask, lse) if bt.rows[b] else (torch.zeros((bt.kvh, n), device="cuda").double(),) * 2
        ref = ref + (before[:, at].double() if accumulate else 0.0)
        bad = (scores[:, at].double() - ref).abs() > tol + 2.0 ** -23 * ref.abs()
        assert not bad.any(), (b, float(((scores[:, at].double() - ref).abs() / (tol + 2.0 ** -23 * ref.abs())).max()))
    assert torch.equal(scores[:, untouched], before[:, untouched])
    return scores


@pytest.mark.parametrize("layout,dtype,d", [("5d", "bf16", 128), ("5dpf", "f16", 64), ("4d", "bf16", 256), ("4d", "f16", 128)])
@pytest.mark.parametrize("kvh,group,t", [(2, 4, 1), (1, 7, 3), (2, 1, 32), (1, 20, 2)])
@pytest.mark.parametrize("given", [True, False])
def test_scores(layout, dtype, d, kvh, group, t, given):
    bt = Batch([t, 77 + t, 600], [t, t, t], kvh=kvh, group=group, layout=layout, dtype=dtype, d=d, seed=t)
    lse = tree_attention(bt.copier, "l", bt.q, bt.table, bt.seq_lens, cu_q=bt.cu_q)[1] if given else None
    check_scores(bt, lse=lse, accumulate=given)


@pytest.mark.parametrize("lens,rows", [([1], [1]), ([0, 31, 32, 33], [0, 1, 2, 3]), ([511, 512, 513, 5000], [1, 4, 0, 2]),
                                       ([70000], [1])])
def test_score_lengths(lens, rows):
    check_scores(Batch(lens, rows, kvh=1, group=4, d=64, seed=len(lens)))


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("rows,d,cols", [(17, 256, 8200), (17, 256, 16383), (17, 128, 16383), (1, 256, 16383)])
def test_scores_of_the_widest_tables(given, rows, d, cols):
    """Tables for up to 16.7M positions: the lengths are the GPU's to know."""
    bt = Batch([100], [rows], kvh=2, group=1, d=d, bs=1024, seed=1)
    table = torch.zeros((1, cols), dtype=torch.int32, device="cuda")
    table[:, :1] = bt.table[:, :1]
    lse = tree_attention(bt.copier, "l", bt.q, bt.table, bt.seq_lens)[1] if given else None
    off = torch.zeros(1, dtype=torch.int64, device="cuda")
    call = lambda t: attention_scores(bt.copier, "l", bt.q, t, bt.seq_lens, torch.zeros((2, 100), device="cuda"), off, lse=lse)
    assert torch.equal(call(table), call(bt.table))
    assert _lib.device_errors(0) == 0


def test_scores_of_a_tree_sum_to_its_rows():
    bt = Batch([100, 300], [9, 12], kvh=2, group=4, seed=3)
    mask = tree_masks(bt.rows, 1, torch.Generator().manual_seed(1))
    _, lse = tree_attention(bt.copier, "l", bt.q, bt.table, bt.seq_lens, cu_q=bt.cu_q, tree_mask=mask.cuda())
    check_scores(bt, mask, lse)
    got = check_scores(bt, mask, None, accumulate=False)
    off, _ = offsets(bt.lens)
    for b in range(2):
        total = got[:, off[b]:off[b] + bt.lens[b]].double().sum(1)
        # one per row and head, each weight off by a relative 2^-14 at most
        assert ((total - bt.rows[b] * bt.group).abs() < bt.rows[b] * bt.group * 2.0 ** -14).all()


def test_rows_that_see_nothing_and_poisoned_keys():
    bt = Batch([4, 40], [4, 2], seed=4)
    mask = tree_masks(bt.rows, 1, torch.Generator().manual_seed(1))
    mask[1] = 0
    blk = int(bt.table[1, 2])
    bt.k[blk, 8:] = math.nan               # behind the end
    mask[4] = 1                            # row 0 of sequence 1 sees token 0 alone
    mask[5] = 1                            # and so does row 1: token 1 is seen by nobody
    bt.k[int(bt.table[1, 39 // 16]), 39 % 16] = math.nan
    off, cols = offsets(bt.lens)
    scores = torch.zeros((bt.kvh, cols), device="cuda")
    attention_scores(bt.copier, "l", bt.q, bt.table, bt.seq_lens, scores, torch.tensor(off, device="cuda"), cu_q=bt.cu_q,
                     tree_mask=mask.cuda())
    assert torch.isfinite(scores).all() and (scores[:, off[1] + 39] == 0).all()
    assert abs(float(scores[:, off[0]:off[0] + 4].sum()) - 3 * bt.kvh * bt.group) < 1e-3


def test_score_bits_streams_graphs():
    bt = Batch([1000, 300], [1, 1], kvh=2, group=4, seed=5)
    off = torch.tensor([0, 1000], device="cuda")
    call = lambda s, o=off, **kw: attention_scores(bt.copier, "l", bt.q, bt.table, bt.seq_lens, s, o, cu_q=bt.cu_q, **kw)
    ref = call(torch.zeros((2, 1300), device="cuda"))
    assert torch.equal(ref, call(torch.zeros((2, 1300), device="cuda")))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    z = torch.zeros((2, 1300), device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    call(z, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(z, ref)
    acc = torch.zeros((2, 1300), device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(acc)
    for _ in range(3):
        g.replay()
    assert torch.allclose(acc, 3 * ref, rtol=1e-6, atol=0)
    z = torch.zeros((2, 1300), device="cuda")
    call(z, torch.tensor([0, 1001], device="cuda"))   # sequence 1 would pass the end
    assert _lib.device_errors(0) == 4 and torch.equal(z[:, :1000], ref[:, :1000]) and (z[:, 1000:] == 0).all()
    for kw in (dict(s=z.double()), dict(s=z[:1]), dict(s=z.t()), dict(o=off.int()), dict(o=off[:1]), dict(scale=0.0),
               dict(lse=torch.zeros((2, 7), device="cuda")), dict(tree_mask=torch.zeros(3, dtype=torch.int64, device="cuda"))):
        args = {"s": z, **kw}
        with pytest.raises((RuntimeError, ValueError)):
            call(**args)


@pytest.mark.parametrize("rows", [1, 9])
@pytest.mark.parametrize("col", [-1, -(1 << 63), (1 << 63) - 1, (1 << 63) - 100, 1 << 40, 701])
def test_score_columns_outside_are_left_out(rows, col):
    """Offsets whose sum with a length passes 64 bits, too; a sequence of length 0 has no columns."""
    bt = Batch([300, 600, 0], [rows, rows, 0], kvh=2, group=4, seed=rows)
    scores = torch.full((2, 1300), 5.0, device="cuda")
    off = torch.tensor([0, col, 1300], device="cuda")
    attention_scores(bt.copier, "l", bt.q, bt.table, bt.seq_lens, scores, off, cu_q=bt.cu_q, accumulate=False)
    assert _lib.device_errors(0) == 4
    assert (scores[:, 300:] == 5.0).all() and (scores[:, :300] != 5.0).all()


# ------------------------------------------------------------ compact --
KV = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "fp8": torch.uint8}


def rope(n, d, dtype=torch.float32):
    f = 1e4 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    a = torch.arange(n, dtype=torch.float64)[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).to(dtype)


def turn(rows, table, old, new, rot, neox):
    """The formula in 64 bits: rows [n, heads, d]."""
    rows, t = rows.double(), table.double()
    half = rot // 2
    oc, os, nc, ns = t[old, :half], t[old, half:], t[new, :half], t[new, half:]
    c, s = (nc * oc + ns * os)[:, None], (ns * oc - nc * os)[:, None]
    out = rows.clone()
    a, b = (rows[..., :half], rows[..., half:rot]) if neox else (rows[..., 0:rot:2], rows[..., 1:rot:2])
    x, y = a * c - b * s, b * c + a * s
    if neox:
        out[..., :half], out[..., half:rot] = x, y
    else:
        out[..., 0:rot:2], out[..., 1:rot:2] = x, y
    return out


def compact_case(layers, lens, keep, *, kvh=2, d=64, bs=16, dtype="bf16", layout="5d", per_head=False, shared=False,
                 mode="none", rot=None, neox=True, tab=torch.float32, dst=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    pages = [-(-n // bs) for n in lens]
    nb = sum(pages) + 2
    shape = {"5d": (2, nb, bs, kvh, d), "5dpf": (nb, 2, bs, kvh, d), "4d": (nb, kvh, bs, 2 * d)}[layout]
    caches = []
    for _ in range(layers):
        x = torch.randn(shape, generator=g)
        caches.append((x.to(torch.float8_e4m3fn).view(torch.uint8) if dtype == "fp8" else x.to(KV[dtype])).cuda())
    table = (torch.randperm(nb - 1, generator=g) + 1).int()
    blk_off = np.concatenate([[0], np.cumsum(pages)[:-1]]).astype(int).tolist()
    lists = (1 if shared else layers) * (kvh if per_head else 1)
    dst = dst or [0] * len(lens)
    caps = [max(0, k) for k in keep]
    idx = torch.full((lists, sum(caps) + 1), -77, dtype=torch.int32)
    at = 0
    for n, k, d0 in zip(lens, keep, dst):
        for r in range(lists):
            idx[r, at:at + k] = (torch.randperm(n - d0, generator=g)[:k].sort().values + d0).int()
        at += k
    count = torch.tensor([keep] * lists, dtype=torch.int32)
    off = np.concatenate([[0], np.cumsum(caps)[:-1]]).astype(np.int64)
    tabl = rope(max(lens) + 1, rot or d, tab)
    copier = CacheCopier()
    names = [f"l{i}" for i in range(layers)]
    for n, c in zip(names, caches):
        copier.register_layer(n, c, layout != "5d")
        if mode != "none":
            copier.register_rotary(n, tabl.cuda(), rot or d, neox)
    expect = [c.cpu().clone() for c in caches]
    back = (lambda x: x.view(torch.float8_e4m3fn).float()) if dtype == "fp8" else (lambda x: x.float())
    # e4m3 values of this size do not saturate
    to = (lambda x: x.to(torch.float8_e4m3fn).view(torch.uint8)) if dtype == "fp8" else (lambda x: x.to(KV[dtype]))
    exact = []
    for l in range(layers):
        old_k, old_v = planes(caches[l].cpu(), layout, d)
        new_k, new_v = planes(expect[l], layout, d)
        at = 0
        for s, k in enumerate(keep):
            for e in range(kvh if per_head else 1):
                r = (0 if shared else l * (kvh if per_head else 1)) + e
                src = idx[r, at:at + k].long()
                to_pos = torch.arange(k) + dst[s]
                hs = slice(e, e + 1) if per_head else slice(0, kvh)
                tb = table[blk_off[s]:].long()
                rows_k = old_k[tb[src // bs], src % bs][:, hs]
                if mode != "none":
                    turned = turn(back(rows_k), tabl, src, to_pos, rot or d, neox)
                    moved = (src != to_pos)[:, None, None].expand(rows_k.shape)
                    exact.append((l, tb[to_pos // bs], to_pos % bs, hs, moved, turned, back(rows_k)))
                    rows_k = torch.where(moved, to(turned.float()), rows_k)
                new_k[tb[to_pos // bs], to_pos % bs, hs] = rows_k
                new_v[tb[to_pos // bs], to_pos % bs, hs] = old_v[tb[src // bs], src % bs][:, hs]
            at += k
    sel = Selection(idx=idx.cuda(), slot=None, count=count.cuda(), out_off=off)
    kw = dict(per_head=per_head, seg_blk_off=blk_off, dst_start=dst, mode=mode)
    kw_check = dict(exact=exact, back=back, layout=layout, d=d, dtype=dtype)
    return copier, names, sel, table.cuda(), kw, caches, expect, kw_check


def check_moved(caches, expect, exact, back, layout, d, dtype):
    """Equal bytes, but for turned keys: those are within the rounding of the
    64-bit formula. The result is rounded once to the cache's type (half a step,
    and half the smallest step near 0); before that, fp32: two factors of two
    products (4 roundings of values up to 1 each: 2^-22), two products with them
    (3 more of |x| and |y|): in all 2^-20 of the larger of the pair."""
    got = [c.cpu() for c in caches]
    half = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24, "fp8": 2.0 ** -4}[dtype]
    tiny = {"bf16": 2.0 ** -133, "f16": 2.0 ** -25, "f32": 2.0 ** -149, "fp8": 2.0 ** -10}[dtype]
    for l, blk, tok, hs, moved, turned, rows in exact:
        k = planes(got[l], layout, d)[0]
        e = planes(expect[l], layout, d)[0]
        r = back(k[blk, tok][:, hs]).double()
        big = rows.double().abs().amax(-1, keepdim=True)
        tol = half * turned.abs() + tiny + 2.0 ** -20 * big * (1 + half)
        assert bool((((r - turned).abs() <= tol) | ~moved).all())
        view = k[blk, tok]
        view[:, hs] = torch.where(moved, e[blk, tok][:, hs], view[:, hs])
        k[blk, tok] = view
    for g, e in zip(got, expect):
        assert torch.equal(g.contiguous().view(torch.uint8), e.contiguous().view(torch.uint8))


def check_compact(*a, **k):
    copier, names, sel, table, kw, caches, expect, chk = compact_case(*a, **k)
    compact(copier, names, sel, table, **kw)
    assert _lib.device_errors(0) == 0
    check_moved(caches, expect, **chk)


@pytest.mark.parametrize("layout", ["5d", "5dpf", "4d"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32", "fp8"])
@pytest.mark.parametrize("per_head", [False, True])
def test_compact_moves(layout, dtype, per_head):
    check_compact(3, [300, 41, 1000], [120, 41, 37], layout=layout, dtype=dtype, per_head=per_head, seed=1)


@pytest.mark.parametrize("layout,dtype", [("5d", "bf16"), ("5dpf", "f16"), ("4d", "f32"), ("4d", "fp8")])
@pytest.mark.parametrize("neox,rot,tab", [(True, None, torch.float32), (False, None, torch.float32), (True, 32, torch.bfloat16),
                                          (False, 32, torch.float16)])
def test_compact_turns_keys(layout, dtype, neox, rot, tab):
    check_compact(2, [500, 33], [250, 20], layout=layout, dtype=dtype, mode="flexible", neox=neox, rot=rot, tab=tab, seed=2)


@pytest.mark.parametrize("dtype,d,rot,tab", [("bf16", 64, 24, torch.float32), ("bf16", 128, 8, torch.float32), ("f16", 128, 40, torch.float32),
                                             ("fp8", 64, 16, torch.bfloat16), ("fp8", 128, 48, torch.float16),
                                             ("f32", 64, 8, torch.float32), ("f32", 64, 24, torch.float32)])
@pytest.mark.parametrize("per_head", [False, True])
def test_compact_turns_an_odd_number_of_vectors(dtype, d, rot, tab, per_head):
    """GPT-J style: the turned part is whole 16-byte vectors, its half need not be."""
    check_compact(2, [500, 33], [250, 20], kvh=3, d=d, dtype=dtype, mode="flexible", neox=False, rot=rot, tab=tab,
                  per_head=per_head, seed=2)


@pytest.mark.parametrize("lens,keep", [([1], [1]), ([1], [0]), ([17, 16, 15], [17, 0, 1]), ([5000], [4900]), ([5000], [3]),
                                       ([700] * 40, [333] * 40)])
def test_compact_lengths(lens, keep):
    check_compact(1, lens, keep, seed=3, mode="flexible" if len(lens) == 3 else "none")


@pytest.mark.parametrize("bs,d", [(1, 64), (5, 128), (24, 256), (16, 80), (64, 8)])
def test_compact_shapes(bs, d):
    check_compact(2, [200, 77], [100, 50], bs=bs, d=d, kvh=3, seed=bs)


def test_compact_shared_lists_and_offsets():
    check_compact(4, [300, 90], [100, 30], shared=True, seed=4, dst=[16, 3], mode="flexible")
    check_compact(4, [300, 90], [100, 30], shared=True, per_head=True, seed=5, dst=[16, 3])
    check_compact(2, [300, 90], [284, 87], seed=6, dst=[16, 3])     # everything stays


def test_compact_many_layers_and_segments():
    check_compact(100, [20], [9], kvh=1, d=8, seed=7)
    check_compact(1, [20] * 300, [7] * 300, kvh=1, d=8, seed=8)


def test_compact_counts_bound_the_lists_and_bad_entries_are_left_out():
    copier, names, sel, table, kw, caches, _, _ = compact_case(1, [100], [10], seed=9)
    before = caches[0].clone()
    sel.count[:] = 0
    compact(copier, names, sel, table, **kw)
    assert torch.equal(caches[0], before)
    k = planes(caches[0], "5d", 64)[0]
    for bad, bit in (([5, 3, 50], 4), ([0, 0, 50], 4), ([0, 1, 10_000], 4), ([-4, 1, 50], 4)):
        caches[0].copy_(before)
        sel.idx[0, :3] = torch.tensor(bad)
        sel.count[:] = 3
        compact(copier, names, sel, table, **kw)
        assert _lib.device_errors(0) == bit, bad
    caches[0].copy_(before)
    sel.idx[0, :3] = torch.tensor([0, 1, 50])
    t2 = table.clone()
    t2[3] = 10_000  # the block of position 50
    compact(copier, names, sel, t2, **kw)
    assert _lib.device_errors(0) == 1 and torch.equal(caches[0], before)
    sel.count[:] = 1_000_000     # more than the list holds: cut to its room, whose last entry is the pad
    sel.idx[0] = torch.arange(sel.idx.shape[1])
    compact(copier, names, sel, table, **kw)
    assert _lib.device_errors(0) == 0 and torch.equal(caches[0], before)
    assert k is not None


@pytest.mark.parametrize("off", [13, 14, 1 << 40, (1 << 63) - 1])
def test_compact_tables_that_start_behind_the_end(off):
    """A segment whose block table lies outside moves nothing, the others do."""
    copier, names, sel, table, kw, caches, expect, chk = compact_case(1, [100, 60], [30, 20], seed=15)
    assert table.numel() == 12
    table = torch.cat([table, table[:1]])
    start = caches[0].clone()
    part = dict(kw, seg_blk_off=[kw["seg_blk_off"][0], off])
    compact(copier, names, sel, table, **part)
    assert _lib.device_errors(0) == 4
    own = table[kw["seg_blk_off"][1]:12].long()
    assert torch.equal(caches[0][:, own], start[:, own])
    rest = torch.ones(caches[0].shape[1], dtype=torch.bool)
    rest[own.cpu()] = False
    assert torch.equal(caches[0].cpu()[:, rest], expect[0][:, rest])


def test_compact_in_a_graph_and_on_a_stream():
    copier, names, sel, table, kw, caches, expect, chk = compact_case(2, [300], [100], seed=10, mode="flexible")
    start = [c.clone() for c in caches]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    compact(copier, names, sel, table, stream=side.cuda_stream, **kw)
    side.synchronize()
    check_moved(caches, expect, **chk)
    for c, s in zip(caches, start):
        c.copy_(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        compact(copier, names, sel, table, **kw)
    # other calls in between do not disturb what was captured
    other = compact_case(3, [90, 20], [30, 10], seed=11)
    compact(other[0], other[1], other[2], other[3], **other[4])
    g.replay()
    check_moved(caches, expect, **chk)


def test_compact_refusals():
    copier, names, sel, table, kw, caches, _, _ = compact_case(3, [100], [10], seed=12)
    bad = [dict(mode="delta"), dict(mode="flexible"), dict(per_head=True), dict(seg_blk_off=[0, 0]), dict(seg_blk_off=[-1]),
           dict(dst_start=[-2]), dict(dst_start=[0, 0])]
    for b in bad:
        with pytest.raises((RuntimeError, ValueError)):
            compact(copier, names, sel, table, **{**kw, **b})
    with pytest.raises(RuntimeError):
        compact(copier, names + ["nope"], sel, table, **kw)
    with pytest.raises(RuntimeError, match="twice"):
        compact(copier, [names[0], names[0]], sel, table, **kw)
    with pytest.raises(RuntimeError):
        compact(copier, names, sel, table.long(), **kw)
    with pytest.raises(RuntimeError):
        compact(copier, names, Selection(idx=sel.idx[:, ::2], slot=None, count=sel.count, out_off=sel.out_off), table, **kw)
    copier.register_layer("odd", torch.zeros((2, 9, 16, 2, 128), dtype=torch.bfloat16, device="cuda"), False)
    with pytest.raises(RuntimeError, match="share"):
        compact(copier, [names[0], "odd"], sel, table, **kw)
    assert _lib.device_errors(0) == 0


def test_a_whole_eviction():
    """A window of rows scores the cache, the best tokens are selected and moved
    to the front, and attention over the shorter cache is attention over them."""
    bt = Batch([700, 413], [8, 8], kvh=2, group=4, seed=20)
    lens, bs = bt.lens, bt.bs
    off = [0, lens[0]]
    scores = torch.zeros((bt.kvh, sum(lens)), device="cuda")
    _, lse = tree_attention(bt.copier, "l", bt.q, bt.table, bt.seq_lens, cu_q=bt.cu_q)
    attention_scores(bt.copier, "l", bt.q, bt.table, bt.seq_lens, scores, torch.tensor(off, device="cuda"), cu_q=bt.cu_q, lse=lse)
    cols = bt.table.shape[1]
    flat = bt.table.reshape(-1).contiguous()
    sel = score_select(scores.sum(0, keepdim=True), flat, bs, seg_len=lens, seg_col_off=off, seg_blk_off=[0, cols], ratio=0.5)
    kept = [sel.get(0, s)[0].cpu().long() for s in range(2)]
    before = [bt.kv64(b) for b in range(2)]
    compact(bt.copier, ["l"], sel, flat, seg_blk_off=[0, cols])
    short = torch.tensor([len(x) for x in kept], dtype=torch.int32, device="cuda")
    # one decode row per sequence, standing behind what is left (its own key is the last kept one)
    q = bt.q[[7, 15]].contiguous()
    out, z = tree_attention(bt.copier, "l", q, bt.table, short)
    assert _lib.device_errors(0) == 0
    bt.q, bt.rows, bt.cu, bt.n = q, [1, 1], [0, 1, 2], 2
    for b in range(2):
        k, v = (x[:, kept[b].cuda()] for x in before[b])
        bt.lens = [len(x) for x in kept]
        ok = torch.ones((1, 1, len(kept[b])), dtype=torch.bool, device="cuda")
        check_attend(bt, out, z, b, *attend64(bt.q64(b), k, v, ok, 1 / math.sqrt(bt.d)))
