"""Page bounds and page selection against exact references (equal, not close)."""
import math

import pytest
import torch

from daric_b200 import _lib
from daric_b200.blocks import new_bounds, page_bounds, select_pages
from attend_util import Batch

pytestmark = pytest.mark.gpu


def bounds_ref(bt, b, start=0):
    """{block: [head, 2, dim]} of the pages of sequence b from position start."""
    found = {}
    for pg in range(start // bt.bs, -(-bt.lens[b] // bt.bs)):
        blk = int(bt.table[b, pg])
        part = bt.k[blk, :min(bt.bs, bt.lens[b] - pg * bt.bs)].float()
        found[blk] = torch.stack([part.amin(0), part.amax(0)], 1)
    return found


@pytest.mark.parametrize("layout,dtype,d,bs", [("5d", "bf16", 128, 16), ("5dpf", "f16", 64, 16), ("4d", "bf16", 256, 8),
                                               ("5d", "f16", 128, 1), ("4d", "bf16", 128, 33), ("5d", "bf16", 64, 128)])
def test_bounds(layout, dtype, d, bs):
    bt = Batch([1, 200, bs, 3 * bs + 1, 0], [0] * 5, layout=layout, dtype=dtype, d=d, bs=bs, kvh=3, seed=bs)
    last = int(bt.table[1, -(-200 // bs) - 1])
    if 200 % bs:
        bt.k[last, 200 % bs:] = math.nan  # tokens that do not exist
    got = page_bounds(bt.copier, "l", bt.table, bt.seq_lens)
    assert _lib.device_errors(0) == 0
    touched = set()
    for b in range(5):
        for blk, ref in bounds_ref(bt, b).items():
            assert torch.equal(got[blk].float(), ref)
            touched.add(blk)
    rest = [i for i in range(bt.nb) if i not in touched]
    assert (got[rest] == 0).all()


def test_bounds_from_a_position_and_nan():
    bt = Batch([100, 47], [0, 0], seed=2)
    bt.k[int(bt.table[0, 3]), 2, 1, 5] = math.nan
    bt.k[int(bt.table[0, 5]), 2, 1, 5] = math.inf
    b = torch.full_like(new_bounds(bt.copier, "l"), 7.0)
    start = torch.tensor([53, 46], dtype=torch.int32, device="cuda")
    page_bounds(bt.copier, "l", bt.table, bt.seq_lens, b, start=start)
    for s, first in ((0, 53), (1, 46)):
        for blk, ref in bounds_ref(bt, s, first).items():
            assert torch.equal(torch.nan_to_num(b[blk].float(), 123.0), torch.nan_to_num(ref, 123.0))
    assert torch.isnan(b[int(bt.table[0, 3]), 1, :, 5]).all()
    assert (b[int(bt.table[0, 2])] == 7).all() and (b[int(bt.table[1, 1])] == 7).all()
    # a start at or behind the end touches nothing
    b.fill_(7.0)
    page_bounds(bt.copier, "l", bt.table, bt.seq_lens, b, start=torch.tensor([112, 1000], dtype=torch.int32, device="cuda"))
    assert (b == 7).all() and _lib.device_errors(0) == 0


@pytest.mark.parametrize("start,touched", [((99, 46), True), ((100, 47), False), ((111, 48), False), ((1 << 31) - 1, False),
                                           (-5, True)])
def test_bounds_from_the_end_on(start, touched):
    """A start at the length or behind it, inside the last page, too, changes nothing."""
    bt = Batch([100, 47], [0, 0], seed=2)
    b = torch.full_like(new_bounds(bt.copier, "l"), 7.0)
    start = torch.tensor(start if isinstance(start, tuple) else (start, start), dtype=torch.int32, device="cuda")
    page_bounds(bt.copier, "l", bt.table, bt.seq_lens, b, start=start)
    last = [int(bt.table[0, 6]), int(bt.table[1, 2])]
    assert ((b[last] != 7).any() if touched else (b == 7).all()) and _lib.device_errors(0) == 0


def select_ref(bt, bounds, k, first=1, last=1):
    out = torch.full((bt.n, bt.kvh, k), -1, dtype=torch.int32)
    for b, t in enumerate(bt.rows):
        near = bounds[bt.table[b].long()].double()  # [page, head, 2, d]
        for j in range(t):
            n, pos = bt.cu[b] + j, bt.lens[b] - t + j
            have = 0 if pos < 0 else pos // bt.bs + 1
            q = bt.q[n].double().view(bt.kvh, bt.group, 1, bt.d)
            part = near[:have].transpose(0, 1)[:, None]
            u = (q.clamp(min=0) * part[:, :, :, 1] + q.clamp(max=0) * part[:, :, :, 0]).sum(-1)
            for h in range(bt.kvh):
                if have <= k:
                    best = list(range(have))
                else:
                    score = [max((math.inf, 1) if math.isnan(x) else (x, 0) for x in col) for col in u[h].t().tolist()]
                    free = sorted(range(first, have - last), key=lambda p: ((-score[p][0], -score[p][1]), p))
                    free.sort(key=lambda p: (-score[p][1], -score[p][0], p))
                    best = sorted(list(range(first)) + list(range(have - last, have)) + free[:k - first - last])
                out[n, h, :len(best)] = torch.tensor(best, dtype=torch.int32)
    return out


def check_select(bt, bounds, k, **kw):
    got = select_pages(bt.q, bounds, bt.table, bt.seq_lens, k, bt.bs, cu_q=bt.cu_q, **kw)
    assert _lib.device_errors(0) == 0
    assert torch.equal(got.cpu(), select_ref(bt, bounds.cpu() if False else bounds, k, **kw))
    return got


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f16", 64), ("bf16", 256)])
@pytest.mark.parametrize("kvh,group", [(2, 4), (1, 7), (1, 20), (2, 1)])
def test_select(dtype, d, kvh, group):
    bt = Batch([1000, 33, 1, 16 * 40], [1, 2, 1, 3], kvh=kvh, group=group, d=d, dtype=dtype, seed=d + group)
    check_select(bt, page_bounds(bt.copier, "l", bt.table, bt.seq_lens), 12)


@pytest.mark.parametrize("k,first,last", [(2, 1, 1), (1, 0, 1), (5, 0, 1), (9, 4, 3), (7, 3, 4), (40, 1, 1), (64, 2, 2)])
def test_forced_pages(k, first, last):
    bt = Batch([1000, 200, 900], [1, 1, 2], seed=k)
    check_select(bt, page_bounds(bt.copier, "l", bt.table, bt.seq_lens), k, first=first, last=last)


def test_long_sequences():
    """Several score chunks, and more keys than a thread holds."""
    bt = Batch([9000, 30001], [1, 1], kvh=1, group=4, d=64, bs=8, seed=3)
    check_select(bt, page_bounds(bt.copier, "l", bt.table, bt.seq_lens), 100)


@pytest.mark.parametrize("bs,n,d", [(8, 66001, 128), (1, 41500, 64), (8, 66001, 256)])
def test_very_long_sequences(bs, n, d):
    """The widest selection CTAs, and more pages than their keys fit in shared memory."""
    bt = Batch([n, 5], [1, 1], kvh=1, group=2, d=d, bs=bs, seed=31)
    check_select(bt, page_bounds(bt.copier, "l", bt.table, bt.seq_lens), 64)


def test_ties_go_to_the_lower_page():
    """All pages alike, and few different scores: thousands of candidates at the border."""
    bt = Batch([6000, 5000], [1, 1], kvh=2, group=3, d=64, seed=4)
    b = torch.zeros_like(new_bounds(bt.copier, "l"))
    check_select(bt, b, 20)
    b[:, :, 0], b[:, :, 1] = -1.0, 1.0
    check_select(bt, b, 20)
    g = torch.Generator().manual_seed(1)
    steps = torch.randint(0, 3, (bt.nb,), generator=g).cuda()
    b[:, :, 1] = (1.0 + steps[:, None, None].float() / 64).to(b.dtype)
    check_select(bt, b, 50)


@pytest.mark.parametrize("rows", [1, 40])
def test_alike_pages_of_long_tables(rows):
    """The widest CTAs with more pages in the bin of the k-th score than are
    ranked at once: all alike, and one page far above that leaves the others in
    a few bins. Again and again: the answer does not depend on timing."""
    bt = Batch([8 * 9000] * 2, [1] * 2, kvh=1, group=2, d=64, bs=8, seed=9)
    q = bt.q[:1].expand(2 * rows, -1, -1).contiguous()
    b = torch.zeros_like(new_bounds(bt.copier, "l"))
    b[:, :, 0], b[:, :, 1] = -1.0, 1.0
    cu = torch.tensor([0, rows, 2 * rows], dtype=torch.int32, device="cuda")
    far = 5000
    for first in (list(range(19)), sorted([*range(18), far])):  # of sequence 0
        if far in first:
            b[bt.table[0, far].long(), :, 1] = 2.0 ** 40
            b[bt.table[0, far].long(), :, 0] = -2.0 ** 40
        expect = torch.tensor([[*(first if s == 0 else range(19)), (8 * 9000 - rows + j) // 8]
                               for s in range(2) for j in range(rows)], dtype=torch.int32)
        for _ in range(25):
            got = select_pages(q, b, bt.table, bt.seq_lens, 20, bt.bs, cu_q=cu)
            assert torch.equal(got[:, 0].cpu(), expect)
    assert _lib.device_errors(0) == 0


def test_scores_closer_than_fp32_tells():
    """Pages whose scores differ by less than an fp32 sum resolves."""
    bt = Batch([16 * 300], [1], kvh=1, group=1, d=128, seed=5)
    bt.q.fill_(1.0)
    b = torch.zeros_like(new_bounds(bt.copier, "l"))
    b[:, :, 1] = 1.0
    b[:, :, 1, 0] = 2.0 ** 20
    g = torch.Generator().manual_seed(2)
    order = torch.randperm(bt.nb, generator=g).cuda()
    b[:, 0, 1, 1] = (2.0 ** -10 * (1 + (order % 128).float() / 128)).to(b.dtype)
    check_select(bt, b, 30)


def test_nan_and_infinite_bounds_rank_first():
    bt = Batch([16 * 200], [1], kvh=2, group=2, d=64, seed=6)
    b = page_bounds(bt.copier, "l", bt.table, bt.seq_lens)
    b[int(bt.table[0, 77]), 0, 1, 3] = math.nan
    b[int(bt.table[0, 99]), 1, :, 3] = math.inf
    got = check_select(bt, b, 10)
    assert 77 in got[0, 0].tolist()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("low,high", [(-math.inf, 0.5), (-0.5, math.inf), (-math.inf, math.inf), (math.inf, math.inf),
                                      (-math.inf, -math.inf), (math.nan, 0.5)])
def test_infinite_bounds_by_the_definition(dtype, low, high):
    """max(q min, q max) of a dimension whose bounds are infinite, where q is
    positive, negative and 0: 0 times infinity is NaN, which ranks highest."""
    bt = Batch([16 * 200], [1], kvh=2, group=3, d=64, dtype=dtype, seed=6)
    b = page_bounds(bt.copier, "l", bt.table, bt.seq_lens)
    b[int(bt.table[0, 99]), :, 0, 3], b[int(bt.table[0, 99]), :, 1, 3] = low, high
    b[int(bt.table[0, 55]), 1, 0, 9], b[int(bt.table[0, 55]), 1, 1, 9] = low, high
    for sign in (1.0, -1.0, 0.0):
        bt.q[..., 3] = bt.q[..., 3].abs() * sign
        bt.q[:, :3, 9] = bt.q[:, :3, 9].abs() * sign
        got = select_pages(bt.q, b, bt.table, bt.seq_lens, 10, bt.bs)
        near = b[bt.table[0, :200].long()].double()
        for h in range(2):
            q = bt.q[0].double().view(2, 3, 1, 64)[h]
            u = torch.maximum(q * near[:, h, 0], q * near[:, h, 1]).sum(-1)  # [group, page]
            nan = torch.isnan(u).any(0)
            score = torch.where(nan, 0.0, u.nan_to_num(0.0, math.inf, -math.inf).amax(0)).tolist()
            rest = sorted(range(1, 199), key=lambda i: (-int(nan[i]), -score[i], i))
            assert got[0, h].tolist() == sorted([0, 199, *rest[:8]]), (sign, h)
    assert _lib.device_errors(0) == 0


def test_strides_padding_streams_and_graphs():
    bt = Batch([800, 700], [1, 1], kvh=2, group=4, seed=7)
    b = page_bounds(bt.copier, "l", bt.table, bt.seq_lens)
    ref = select_pages(bt.q, b, bt.table, bt.seq_lens, 8, 16)
    wide = torch.cat([bt.q, bt.q], 1)[:, :bt.q.shape[1]]
    out = torch.full((2, 2, 8), 55, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 1, 1], dtype=torch.int32, device="cuda")  # row 1 belongs to nobody
    select_pages(wide, b, bt.table, bt.seq_lens, 8, 16, cu_q=cu, out=out)
    assert torch.equal(out[0], ref[0]) and (out[1] == 55).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    again = select_pages(bt.q, b, bt.table, bt.seq_lens, 8, 16, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(again, ref)
    lens = bt.seq_lens.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        page_bounds(bt.copier, "l", bt.table, lens, b)
        o = select_pages(bt.q, b, bt.table, lens, 8, 16)
    lens -= 100
    g.replay()
    fresh = page_bounds(bt.copier, "l", bt.table, lens, b.clone())
    assert torch.equal(o, select_pages(bt.q, fresh, bt.table, lens, 8, 16))


def test_bad_blocks_and_refusals():
    bt = Batch([800, 700], [1, 1], kvh=2, group=4, seed=8)
    b = page_bounds(bt.copier, "l", bt.table, bt.seq_lens)
    table = bt.table.clone()
    table[0, 3], table[1, 4] = -5, bt.nb
    page_bounds(bt.copier, "l", table, bt.seq_lens, b)
    assert _lib.device_errors(0) == 1
    got = select_pages(bt.q, b, table, bt.seq_lens, 8, 16)
    assert _lib.device_errors(0) == 1 and (got >= 0).all()
    ok = dict(q=bt.q, bounds=b, block_table=bt.table, seq_lens=bt.seq_lens, k=8, block_size=16)
    for kw in (dict(k=1), dict(k=0), dict(k=3, first=2, last=2), dict(last=0), dict(first=-1), dict(block_size=0),
               dict(q=bt.q.float()), dict(q=bt.q[:, :3]), dict(bounds=b[..., :64]), dict(bounds=b.half()),
               dict(block_table=bt.table.long()), dict(seq_lens=bt.seq_lens.cpu()),
               dict(out=torch.zeros((2, 2, 7), dtype=torch.int32, device="cuda"))):
        with pytest.raises((RuntimeError, ValueError)):
            select_pages(**{**ok, **kw})
    for kw in (dict(bounds=b.half()), dict(bounds=b[1:]), dict(start=bt.seq_lens.long()), dict(start=bt.seq_lens[:1])):
        with pytest.raises((RuntimeError, ValueError)):
            page_bounds(bt.copier, "l", bt.table, bt.seq_lens, **kw)
    assert _lib.device_errors(0) == 0
