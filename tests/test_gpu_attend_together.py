"""The paged-cache operators as they are used together, and calls at once."""
import math
import threading

import pytest
import torch

from daric_b200 import _lib
from daric_b200 import attend
from daric_b200.attend import sparse_attention, tree_attention
from daric_b200.blocks import new_bounds, page_bounds, select_pages
from daric_b200.evict import attention_scores
from attend_util import Batch, attend64, check_attend
from test_gpu_attend import check_sparse, check_tree, random_pages, run_tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kvh,group,t,bs", [(1, 40, 1, 16), (1, 160, 1, 16), (2, 150, 2, 256), (1, 300, 3, 1024)])
def test_large_groups_and_blocks(kvh, group, t, bs):
    bt = Batch([1500, 33], [t, t], kvh=kvh, group=group, bs=bs, seed=group)
    check_tree(bt, *run_tree(bt))
    pages = random_pages(bt, 2, torch.Generator().manual_seed(group)).cuda()
    out, lse = sparse_attention(bt.copier, "l", bt.q, pages, bt.table, bt.seq_lens, cu_q=bt.cu_q)
    assert _lib.device_errors(0) == 0
    check_sparse(bt, pages.cpu(), out, lse)


@pytest.mark.parametrize("dtype,layout,t", [("bf16", "5d", 40), ("f16", "4d", 3)])
def test_prompt_rows_then_decode_steps(dtype, layout, t):
    """The last rows of two prompts select and read pages, then decode steps
    refresh the bounds of the page they wrote and do the same."""
    bt = Batch([900 + t, 333 + t], [t, t], kvh=2, group=4, layout=layout, dtype=dtype, seed=t)
    k = 9
    lens = bt.seq_lens.clone()
    bounds = page_bounds(bt.copier, "l", bt.table, lens)

    def step(start=None):
        page_bounds(bt.copier, "l", bt.table, lens, bounds, start=start)
        pages = select_pages(bt.q, bounds, bt.table, lens, k, bt.bs, cu_q=bt.cu_q)
        out, lse = sparse_attention(bt.copier, "l", bt.q, pages, bt.table, lens, cu_q=bt.cu_q)
        assert _lib.device_errors(0) == 0
        check_sparse(bt, pages.cpu(), out, lse)
        # every row lists its own page, the first one, and as many as there are up to k
        for b in range(2):
            for j in range(bt.rows[b]):
                own = (bt.lens[b] - bt.rows[b] + j) // bt.bs
                for h in range(bt.kvh):
                    row = pages[bt.cu[b] + j, h].tolist()
                    have = [x for x in row if x >= 0]
                    assert have == sorted(set(have)) and have[0] == 0 and have[-1] == own
                    assert len(have) == min(k, own + 1) and row[len(have):] == [-1] * (k - len(have))
        return pages

    step()
    bt.rows, bt.cu, bt.n, bt.cu_q = [1, 1], [0, 1, 2], 2, None
    gen = torch.Generator().manual_seed(1)
    for _ in range(3):  # tables have room for one more page each
        start = lens.clone()
        lens += 1
        bt.lens = [n + 1 for n in bt.lens]
        pos = start.long()
        for b in range(2):
            if bt.lens[b] % bt.bs == 1:  # a new page, the one block that is free (of one sequence at most)
                bt.table[b, int(pos[b]) // bt.bs] = 0
        blk = bt.table.long()[torch.arange(2), pos // bt.bs]
        new = torch.randn((2, bt.kvh, bt.d), generator=gen).to(bt.cache.dtype).cuda()
        bt.k[blk, pos % bt.bs] = new
        bt.v[blk, pos % bt.bs] = -new
        bt.q = torch.randn((2, bt.kvh * bt.group, bt.d), generator=gen).to(bt.cache.dtype).cuda()
        step(start)
    fresh = new_bounds(bt.copier, "l")
    page_bounds(bt.copier, "l", bt.table, lens, fresh)
    for b in range(2):
        ids = bt.table[b, :-(-bt.lens[b] // bt.bs)].long()
        assert torch.equal(bounds[ids], fresh[ids])


def test_two_threads_on_one_stream():
    """Calls of two threads take turns on the default stream: neither's parts
    are joined into the other's rows."""
    bts = [Batch([6000, 1200], [2, 2], kvh=2, group=4, seed=50), Batch([3500, 4400], [30, 30], kvh=2, group=4, seed=51)]
    pages = [random_pages(b, 40, torch.Generator().manual_seed(3)).cuda() for b in bts]

    def once(i):
        b = bts[i]
        a = tree_attention(b.copier, "l", b.q, b.table, b.seq_lens, cu_q=b.cu_q)
        s = sparse_attention(b.copier, "l", b.q, pages[i], b.table, b.seq_lens, cu_q=b.cu_q)
        return (*a, *s)

    expect = [once(i) for i in range(2)]
    torch.cuda.synchronize()
    wrong = []

    def many(i):
        got = [once(i) for _ in range(60)]
        torch.cuda.synchronize()
        wrong.extend(i for g in got if not all(torch.equal(x, y) for x, y in zip(g, expect[i])))

    threads = [threading.Thread(target=many, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and _lib.device_errors(0) == 0


def test_two_streams_at_once():
    bt = Batch([5000, 700], [2, 2], kvh=2, group=4, seed=52)
    expect = run_tree(bt)
    scores = torch.zeros((2, 5700), device="cuda")
    off = torch.tensor([0, 5000], device="cuda")
    attention_scores(bt.copier, "l", bt.q, bt.table, bt.seq_lens, scores, off, cu_q=bt.cu_q)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                o, z = tree_attention(bt.copier, "l", bt.q, bt.table, bt.seq_lens, cu_q=bt.cu_q)
                w = attention_scores(bt.copier, "l", bt.q, bt.table, bt.seq_lens, torch.zeros_like(scores), off, cu_q=bt.cu_q)
                got.append((o, z, w))
    torch.cuda.synchronize()
    assert all(torch.equal(o, expect[0]) and torch.equal(z, expect[1]) and torch.equal(w, scores) for o, z, w in got)


def test_lists_longer_than_any_table():
    """A list of more entries than the many-row form takes goes row by row."""
    bt = Batch([130], [40], kvh=1, group=4, seed=53)
    few = random_pages(bt, 4, torch.Generator().manual_seed(4), holes=False).cuda()
    long = torch.full((40, 1, 50000), -1, dtype=torch.int32, device="cuda")
    long[:, :, 49996:] = few
    out, lse = sparse_attention(bt.copier, "l", bt.q, long, bt.table, bt.seq_lens, cu_q=bt.cu_q)
    assert _lib.device_errors(0) == 0
    check_sparse(bt, few.cpu(), out, lse)


FORMS = [(1, 4, 1), (1, 4, 5), (2, 4, 16), (1, 8, 33)]  # KV heads, group, rows: each form of the kernels


@pytest.mark.parametrize("kvh,group,t", FORMS)
@pytest.mark.parametrize("bs", [16, 24, 128])
@pytest.mark.parametrize("layout", ["5d", "4d"])
def test_slots_behind_the_length_do_not_matter(kvh, group, t, bs, layout):
    """Whatever stands in the rest of the last page and in other blocks, NaN too."""
    bt = Batch([300, 77, 129], [t, t, t], kvh=kvh, group=group, bs=bs, layout=layout, seed=t)
    pages = random_pages(bt, 2, torch.Generator().manual_seed(t)).cuda()

    def both():
        return (*run_tree(bt), *sparse_attention(bt.copier, "l", bt.q, pages, bt.table, bt.seq_lens, cu_q=bt.cu_q))

    used = torch.zeros((bt.nb, bs), dtype=torch.bool, device="cuda")
    for b, n in enumerate(bt.lens):
        pos = torch.arange(n, device="cuda")
        used[bt.table[b].long()[pos // bs], pos % bs] = True
    expect = both()
    for x in (bt.k, bt.v):
        x[~used] = math.nan
    assert all(torch.equal(a, b) for a, b in zip(both(), expect))
    assert _lib.device_errors(0) == 0


@pytest.mark.parametrize("kvh,group,t", FORMS)
@pytest.mark.parametrize("bs", [16, 24])
def test_bad_blocks_in_every_form(kvh, group, t, bs):
    """Keys of a block that is not there are keys that do not exist."""
    bt = Batch([400, 200], [t, t], kvh=kvh, group=group, bs=bs, seed=t + bs)
    clean = bt.table.clone()
    bt.table[0, 2] = -5
    bt.table[1, 4] = 1 << 30
    out, lse = tree_attention(bt.copier, "l", bt.q, bt.table, bt.seq_lens, cu_q=bt.cu_q)
    assert _lib.device_errors(0) == 1
    bt.table = clean
    for b, page in ((0, 2), (1, 4)):
        k, v = bt.kv64(b)
        ok = bt.sees(b) & (torch.arange(bt.lens[b], device="cuda") // bs != page)
        check_attend(bt, out, lse, b, *attend64(bt.q64(b), k, v, ok.repeat(group, 1)[None], 1 / math.sqrt(bt.d)))


@pytest.mark.parametrize("seqs,length", [(12, 2048), (60, 150), (100, 61)])
@pytest.mark.parametrize("t", [16, 40])
@pytest.mark.parametrize("d", [64, 128])
def test_many_segments_on_a_block(seqs, length, t, d):
    """A block of the many-row forms goes through several whole and cut segments."""
    lens = [length + 3 * (b % 7) for b in range(seqs)]
    bt = Batch(lens, [t] * seqs, kvh=8, group=4, d=d, seed=seqs + t)
    first = run_tree(bt)
    check_tree(bt, *first)
    pages = random_pages(bt, 3 if length < 1000 else 40, torch.Generator().manual_seed(t)).cuda()
    out, lse = sparse_attention(bt.copier, "l", bt.q, pages, bt.table, bt.seq_lens, cu_q=bt.cu_q)
    check_sparse(bt, pages.cpu(), out, lse)
    for _ in range(10):
        again = run_tree(bt)
        o, z = sparse_attention(bt.copier, "l", bt.q, pages, bt.table, bt.seq_lens, cu_q=bt.cu_q)
        assert all(torch.equal(x, y) for x, y in zip((*first, out, lse), (*again, o, z)))
    assert _lib.device_errors(0) == 0


@pytest.mark.parametrize("cu,kept", [([0, 1, 99], [True, False, False]), ([0, 3, 1], [True] * 3), ([0, 2, 99], [True, True, False]),
                                     ([-1, 1, 2], [False, True, False])])
def test_sequences_with_bad_offsets_have_no_rows(cu, kept):
    """Every call leaves their rows as they were and sets the error bit (a call
    that goes from rows to sequences sees only the sequences that rows lead to)."""
    bt = Batch([270, 233], [2, 1], kvh=2, group=4, seed=54)
    bounds = page_bounds(bt.copier, "l", bt.table, bt.seq_lens)
    cu_q = torch.tensor(cu, dtype=torch.int32, device="cuda")
    pages = torch.zeros((3, bt.kvh, 1), dtype=torch.int32, device="cuda")
    for call in (tree_attention, lambda c, n, q, *a, **k: sparse_attention(c, n, q, pages, *a, **k)):
        out, lse = torch.full_like(bt.q, 55.0), torch.full(bt.q.shape[:2], 55.0, device="cuda")
        call(bt.copier, "l", bt.q, bt.table, bt.seq_lens, cu_q=cu_q, out=out, lse=lse)
        assert _lib.device_errors(0) == (4 if call is tree_attention or cu != [0, 3, 1] else 0)
        for r in range(3):
            assert (out[r] != 55).any().item() == (lse[r] != 55).any().item() == kept[r]
    got = torch.full((3, bt.kvh, 5), 55, dtype=torch.int32, device="cuda")
    select_pages(bt.q, bounds, bt.table, bt.seq_lens, 5, bt.bs, cu_q=cu_q, out=got)
    assert _lib.device_errors(0) == (4 if cu != [0, 3, 1] else 0)
    assert [(got[r] != 55).any().item() for r in range(3)] == kept


def test_workspaces_are_kept_for_torchs_streams_only(monkeypatch):
    """Not where the handle of a stream may come back as another one, where the
    call is captured, or where that cannot be told."""
    bt = Batch([5000, 700], [2, 2], kvh=2, group=4, seed=55)
    pages = random_pages(bt, 40, torch.Generator().manual_seed(3)).cuda()
    kept = attend._workspaces.of

    def both():
        return (*tree_attention(bt.copier, "l", bt.q, bt.table, bt.seq_lens, cu_q=bt.cu_q),
                *sparse_attention(bt.copier, "l", bt.q, pages, bt.table, bt.seq_lens, cu_q=bt.cu_q))

    kept.clear()
    expect = both()
    assert len(kept) == 2
    both()
    assert len(kept) == 2
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream, more in ((torch.cuda.ExternalStream(side.cuda_stream), 0), (side, 2)):
        kept.clear()
        with torch.cuda.stream(stream):
            got = both()
        side.synchronize()
        assert len(kept) == more and all(torch.equal(a, b) for a, b in zip(got, expect))
    kept.clear()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = both()
    g.replay()
    assert not kept and all(torch.equal(a, b) for a, b in zip(got, expect))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    got = both()
    assert not kept and all(torch.equal(a, b) for a, b in zip(got, expect))

