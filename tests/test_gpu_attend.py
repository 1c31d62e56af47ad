"""Attention over the paged cache against 64-bit references: trees of drafted
tokens, listed pages, lengths, layouts, empty rows and non-finite values."""
import math

import pytest
import torch

from daric_b200 import _lib
from daric_b200.attend import sparse_attention, tree_attention
from attend_util import Batch, attend64, check_attend, tree_masks

pytestmark = pytest.mark.gpu


def run_tree(bt, mask=None, **kw):
    out, lse = tree_attention(bt.copier, "l", bt.q, bt.table, bt.seq_lens, cu_q=bt.cu_q,
                              tree_mask=None if mask is None else mask.cuda(), **kw)
    assert _lib.device_errors(0) == 0
    return out, lse


def check_tree(bt, out, lse, mask=None, scale=None):
    scale = 1 / math.sqrt(bt.d) if scale is None else scale
    for b in range(len(bt.lens)):
        if bt.rows[b] == 0:
            continue
        k, v = bt.kv64(b)
        ok = bt.sees(b, mask).repeat(bt.group, 1)[None]
        check_attend(bt, out, lse, b, *attend64(bt.q64(b), k, v, ok, scale))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("layout", ["5d", "5dpf", "4d"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_layouts_types_dims(dtype, layout, d):
    bt = Batch([1, 77, 300, 16], [1, 3, 5, 2], d=d, dtype=dtype, layout=layout, seed=d)
    check_tree(bt, *run_tree(bt))


@pytest.mark.parametrize("kvh,group", [(8, 4), (4, 7), (1, 8), (1, 16), (2, 1), (3, 5), (2, 20)])
@pytest.mark.parametrize("t", [1, 4, 13])
def test_heads_and_rows(kvh, group, t):
    bt = Batch([513, 64 + t, 129], [t, t, t], kvh=kvh, group=group, seed=group * 31 + t, uniform_rows=t == 4)
    mask = tree_masks(bt.rows, 1, torch.Generator().manual_seed(t)) if t > 1 else None
    check_tree(bt, *run_tree(bt, mask), mask)


@pytest.mark.parametrize("bs", [1, 5, 8, 16, 24, 64, 128])
def test_block_sizes(bs):
    bt = Batch([3, 130, 257], [2, 2, 2], bs=bs, seed=bs)
    check_tree(bt, *run_tree(bt))


@pytest.mark.parametrize("lens", [[1], [2, 1, 31], [32, 33, 127, 128, 129, 4097], [20001]])
def test_lengths(lens):
    bt = Batch(lens, [1] * len(lens), seed=len(lens))
    check_tree(bt, *run_tree(bt))


@pytest.mark.parametrize("t,words", [(64, 1), (65, 2), (100, 2), (130, 3), (100, 1)])
def test_wide_trees(t, words):
    """More drafted tokens than a word of the mask, or than the mask holds."""
    bt = Batch([t + 40, t, 700], [t, t, 9], group=2, seed=t)
    mask = tree_masks(bt.rows, words, torch.Generator().manual_seed(t))
    check_tree(bt, *run_tree(bt, mask), mask)


@pytest.mark.parametrize("dtype,layout,d", [("bf16", "5d", 128), ("f16", "4d", 128), ("bf16", "5dpf", 64), ("f16", "5d", 64),
                                            ("bf16", "4d", 256)])
@pytest.mark.parametrize("kvh,group,t", [(2, 4, 16), (1, 8, 17), (2, 7, 37), (1, 8, 64)])
def test_many_rows(dtype, layout, d, kvh, group, t):
    """64 to 512 (row, head) pairs of a KV head, ragged, trees and chains, one and several CTAs per segment."""
    bt = Batch([t + 1, 900, 128 + t, 5000], [t, t - 3, 1, t], kvh=kvh, group=group, d=d, dtype=dtype, layout=layout, seed=t)
    check_tree(bt, *run_tree(bt))
    mask = tree_masks(bt.rows, 1, torch.Generator().manual_seed(t))
    check_tree(bt, *run_tree(bt, mask), mask)


def test_growing_logits_move_the_maximum():
    """Keys whose logits rise along the sequence by far more than 2^8 each tile:
    what was summed up so far is rescaled, often to nothing."""
    bt = Batch([1500, 700], [16, 16], kvh=1, group=4, seed=41)
    for b in range(2):
        pos = torch.arange(bt.lens[b], device="cuda")
        blk = bt.table[b].long()[pos // bt.bs]
        bt.k[blk, pos % bt.bs, 0, 0] = (pos.float() / 20).to(bt.cache.dtype)
    bt.q[..., 0] = bt.q[..., 0].abs() + 1
    check_tree(bt, *run_tree(bt))
    bt.q[..., 0] = -bt.q[..., 0]
    check_tree(bt, *run_tree(bt))


def test_appended_prompt_rows():
    """Hundreds of causal rows per sequence: several row tiles."""
    bt = Batch([500, 333], [300, 333], kvh=2, group=3, seed=5)
    check_tree(bt, *run_tree(bt))


def test_ragged_rows_and_empty_sequences():
    bt = Batch([40, 17, 300, 0, 9], [0, 17, 1, 0, 4], seed=2)
    check_tree(bt, *run_tree(bt))


def test_many_sequences():
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(1, 200, (333,), generator=g).tolist()
    bt = Batch(lens, [1] * 333, kvh=1, group=2, d=64, seed=8)
    check_tree(bt, *run_tree(bt))


def test_rows_that_see_nothing():
    """A mask without a bit and no context; more rows than positions; length 0."""
    bt = Batch([6, 20], [6, 4], seed=4)
    mask = tree_masks(bt.rows, 1, torch.Generator().manual_seed(0))
    mask[2] = 0   # sees no drafted token, and there is no context
    mask[8] = 0   # sees the context alone
    out, lse = run_tree(bt, mask)
    check_tree(bt, out, lse, mask)
    assert (out[2] == 0).all() and (lse[2] == -math.inf).all()
    bt.seq_lens[0] = 2   # rows 0..3 stand before the first position
    bt.seq_lens[1] = 0
    out, lse = run_tree(bt)
    assert (out[:4] == 0).all() and (lse[:4] == -math.inf).all()
    assert (out[6:] == 0).all() and (lse[6:] == -math.inf).all()
    assert torch.isfinite(lse[4:6]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("group", [2, 20])
def test_nonfinite_values_stay_where_they_are_seen(dtype, group):
    t = 6
    bt = Batch([50, 37], [t, t], group=group, dtype=dtype, seed=6)
    mask = tree_masks(bt.rows, 1, torch.Generator().manual_seed(9))
    # drafted token 3 of sequence 0 is poisoned; only row 3 of it sees it
    mask[:t] &= ~(1 << 3)
    mask[3] |= 1 << 3
    pos = 50 - t + 3
    blk = int(bt.table[0, pos // 16])
    bt.v[blk, pos % 16, 0, 5] = math.inf
    bt.v[blk, pos % 16, 1, 7] = math.nan
    bt.k[blk, pos % 16, 1, 0] = math.nan
    # behind the end of sequence 1, in its last block
    blk1 = int(bt.table[1, 2])
    bt.v[blk1, 5:] = math.nan
    bt.k[blk1, 5:] = math.inf
    out, lse = run_tree(bt, mask)
    check_tree(bt, out, lse, mask)
    others = [r for r in range(2 * t) if r != 3]
    assert torch.isfinite(out[others]).all()
    assert (out[3, :group, 5] == math.inf).all() and torch.isnan(out[3, group:]).all()


@pytest.mark.parametrize("kvh,group,t", [(1, 4, 1), (1, 4, 5), (2, 4, 16), (1, 8, 33), (1, 20, 6), (1, 20, 16), (1, 4, 200)])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("at", ["last", "tile"])
def test_nonfinite_values_of_the_context_reach_every_row(kvh, group, t, masked, at):
    """At the last position before the drafted tokens, and at the first one of
    the 128 keys that hold it, in every form."""
    bt = Batch([900, 300 + t], [t, t], kvh=kvh, group=group, seed=6)
    mask = tree_masks(bt.rows, -(-t // 64), torch.Generator().manual_seed(9)) if masked else None
    for b in range(2):
        ctx = bt.lens[b] - t
        pos = ctx - 1 if at == "last" else ctx // 128 * 128
        blk = int(bt.table[b, pos // 16])
        bt.v[blk, pos % 16, 0, 5] = math.inf
        bt.v[blk, pos % 16, kvh - 1, 70] = math.nan
    out, lse = run_tree(bt, mask)
    check_tree(bt, out, lse, mask)
    assert (out[:, :group, 5] == math.inf).all() and torch.isnan(out[:, -group:, 70]).all()


@pytest.mark.parametrize("kvh,group,t", [(1, 4, 1), (1, 4, 5), (2, 4, 16), (1, 8, 33), (1, 20, 16)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("logit", [12.0, 18.0, 20.0])
def test_many_small_weights_count_together(kvh, group, t, dtype, logit):
    """One key far above thousands of others: the output is what those sum to
    (weights of 2^-17, 2^-26 and 2^-29; fp16 itself ends at 2^-24)."""
    bt = Batch([5000], [t], kvh=kvh, group=group, dtype=dtype, seed=3)
    bt.q.zero_()
    bt.q[..., 0] = 1.0
    bt.k.zero_()
    bt.v.fill_(1.0)
    blk = int(bt.table[0, 0])
    bt.k[blk, 0, :, 0] = logit
    bt.v[blk, 0] = 0.0
    out, lse = run_tree(bt, scale=1.0)
    check_tree(bt, out, lse, scale=1.0)
    if t == 1:
        pages = torch.arange(bt.table.shape[1], dtype=torch.int32).expand(1, kvh, -1)
        out, lse = sparse_attention(bt.copier, "l", bt.q, pages.cuda(), bt.table.clamp(min=1), bt.seq_lens, scale=1.0)
        check_tree(bt, out, lse, scale=1.0)


def test_lowest_values_and_large_logits():
    bt = Batch([90, 200], [2, 2], seed=12, spread=30.0)
    bt.k[int(bt.table[0, 0]), 3] = torch.finfo(torch.bfloat16).min / 1e30
    check_tree(bt, *run_tree(bt, scale=0.7), scale=0.7)


def test_strided_queries_outputs_and_tables():
    bt = Batch([70, 150, 40], [3, 1, 2], kvh=2, group=4, seed=13)
    wide = torch.zeros((bt.n, 3, bt.kvh * bt.group, bt.d), dtype=bt.q.dtype, device="cuda")
    wide[:, 1] = bt.q
    table = torch.full((3, bt.table.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    table[:, :bt.table.shape[1]] = bt.table
    out = torch.full_like(wide, 9.0)
    lse = torch.full((bt.n, 40), 9.0, device="cuda")
    ref, ref_lse = run_tree(bt)
    got, got_lse = tree_attention(bt.copier, "l", wide[:, 1], table[:, :bt.table.shape[1]], bt.seq_lens, cu_q=bt.cu_q,
                                  out=out[:, 1], lse=lse[:, 8:16])
    assert torch.equal(got, ref) and torch.equal(got_lse, ref_lse)
    assert (out[:, 0] == 9).all() and (out[:, 2] == 9).all()
    assert (lse[:, :8] == 9).all() and (lse[:, 16:] == 9).all()


def test_rows_behind_the_last_sequence_are_left():
    bt = Batch([70, 33], [3, 2], seed=14)
    q = torch.cat([bt.q, torch.full((4, *bt.q.shape[1:]), math.nan, dtype=bt.q.dtype, device="cuda")])
    out, lse = torch.full_like(q, 5.0), torch.full(q.shape[:2], 5.0, device="cuda")
    tree_attention(bt.copier, "l", q, bt.table, bt.seq_lens, cu_q=bt.cu_q, out=out, lse=lse)
    assert (out[5:] == 5).all() and (lse[5:] == 5).all()
    check_tree(bt, out[:5], lse[:5])
    pages = torch.zeros((9, bt.kvh, 2), dtype=torch.int32, device="cuda")
    out.fill_(5.0), lse.fill_(5.0)
    sparse_attention(bt.copier, "l", q, pages, bt.table, bt.seq_lens, cu_q=bt.cu_q, out=out, lse=lse)
    assert (out[5:] == 5).all() and (lse[5:] == 5).all() and torch.isfinite(out[:5]).all()


def test_bad_blocks_lengths_and_offsets_set_error_bits():
    bt = Batch([70, 33], [1, 1], seed=15)
    ref, _ = run_tree(bt)
    table = bt.table.clone()
    table[0, 1] = bt.nb + 5
    table[1, 0] = -1
    out, _ = tree_attention(bt.copier, "l", bt.q, table, bt.seq_lens, cu_q=bt.cu_q)
    assert _lib.device_errors(0) == 1 and torch.isfinite(out).all()
    # sequence 0 without its second block equals attention over the other keys
    k, v = bt.kv64(0)
    ok = bt.sees(0).repeat(bt.group, 1)[None].clone()
    ok[..., 16:32] = False
    check_attend(bt, out, tree_attention(bt.copier, "l", bt.q, table, bt.seq_lens, cu_q=bt.cu_q)[1], 0,
                 *attend64(bt.q64(0), k, v, ok, 1 / math.sqrt(bt.d)))
    _lib.device_errors(0)
    lens = bt.seq_lens.clone()
    lens[0] = 10_000_000
    table = bt.table.clamp(min=1)
    tree_attention(bt.copier, "l", bt.q, table, lens, cu_q=bt.cu_q)
    assert _lib.device_errors(0) == 4
    cu = torch.tensor([0, 1, 99], dtype=torch.int32, device="cuda")
    out = torch.full_like(bt.q, 5.0)
    tree_attention(bt.copier, "l", bt.q, bt.table, bt.seq_lens, cu_q=cu, out=out)
    assert _lib.device_errors(0) == 4 and torch.equal(out[0], ref[0]) and (out[1] == 5).all()
    pages = torch.tensor([0, 999, -3], dtype=torch.int32, device="cuda").expand(2, bt.kvh, 3).contiguous()
    out, _ = sparse_attention(bt.copier, "l", bt.q, pages, bt.table, bt.seq_lens, cu_q=bt.cu_q)
    assert _lib.device_errors(0) == 4 and torch.isfinite(out).all()


def test_another_stream_and_a_graph():
    """The same call on a side stream, and captured twice with other data at replay."""
    bt = Batch([700, 1500], [1, 1], kvh=4, group=4, seed=16)
    ref, ref_lse = run_tree(bt)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out, lse = tree_attention(bt.copier, "l", bt.q, bt.table, bt.seq_lens, cu_q=bt.cu_q, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(out, ref) and torch.equal(lse, ref_lse)
    lens = bt.seq_lens.clone()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o, z = tree_attention(bt.copier, "l", bt.q, bt.table, lens, cu_q=bt.cu_q)
        graphs.append((g, o, z))
    lens -= 123
    expect, expect_lse = tree_attention(bt.copier, "l", bt.q, bt.table, lens, cu_q=bt.cu_q)
    for g, o, z in graphs:
        o.fill_(3.0)
        g.replay()
        assert torch.equal(o, expect) and torch.equal(z, expect_lse)
    lens += 123
    graphs[0][0].replay()
    assert torch.equal(graphs[0][1], ref) and torch.equal(graphs[1][1], expect)


def test_results_do_not_depend_on_timing():
    bt = Batch([5000, 777, 12000], [2, 2, 2], kvh=2, group=4, seed=17)
    first = run_tree(bt)
    for _ in range(5):
        again = run_tree(bt)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# ------------------------------------------------------------- sparse --
def random_pages(bt, k, gen, holes=True):
    """Ascending random pages per row and head among those the row sees, padded with -1."""
    pages = torch.full((bt.n, bt.kvh, k), -1, dtype=torch.int32)
    for b, t in enumerate(bt.rows):
        for j in range(t):
            have = (bt.lens[b] - t + j) // bt.bs + 1
            for h in range(bt.kvh):
                m = min(k, have) if not holes else int(torch.randint(0, min(k, have) + 1, (1,), generator=gen))
                pages[bt.cu[b] + j, h, :m] = torch.randperm(have, generator=gen)[:m].sort().values.int()
    return pages


def check_sparse(bt, pages, out, lse, scale=None):
    scale = 1 / math.sqrt(bt.d) if scale is None else scale
    for b in range(len(bt.lens)):
        t = bt.rows[b]
        if t == 0:
            continue
        k, v = bt.kv64(b)
        page_of = torch.arange(bt.lens[b]) // bt.bs
        ok = torch.zeros((bt.kvh, t, bt.lens[b]), dtype=torch.bool)
        for j in range(t):
            for h in range(bt.kvh):
                ok[h, j] = torch.isin(page_of, pages[bt.cu[b] + j, h])
        ok = (ok.cuda() & bt.sees(b)[None]).repeat(1, bt.group, 1)
        check_attend(bt, out, lse, b, *attend64(bt.q64(b), k, v, ok, scale))


@pytest.mark.parametrize("layout,dtype,d", [("5d", "bf16", 128), ("5dpf", "f16", 64), ("4d", "bf16", 256),
                                            ("4d", "f16", 128)])
@pytest.mark.parametrize("kvh,group", [(2, 4), (1, 7), (1, 20)])
def test_sparse_layouts(layout, dtype, d, kvh, group):
    bt = Batch([300, 5, 1000], [1, 2, 3], kvh=kvh, group=group, layout=layout, dtype=dtype, d=d, seed=21)
    pages = random_pages(bt, 9, torch.Generator().manual_seed(1))
    out, lse = sparse_attention(bt.copier, "l", bt.q, pages.cuda(), bt.table, bt.seq_lens, cu_q=bt.cu_q)
    assert _lib.device_errors(0) == 0
    check_sparse(bt, pages, out, lse)


@pytest.mark.parametrize("bs,k", [(1, 40), (8, 1), (16, 33), (64, 3), (5, 17)])
def test_sparse_block_sizes(bs, k):
    bt = Batch([200, 333], [2, 2], bs=bs, seed=bs + k)
    pages = random_pages(bt, k, torch.Generator().manual_seed(k), holes=k > 1)
    out, lse = sparse_attention(bt.copier, "l", bt.q, pages.cuda(), bt.table, bt.seq_lens, cu_q=bt.cu_q)
    check_sparse(bt, pages, out, lse)


def test_sparse_many_rows_and_sequences():
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(4, 90, (70,), generator=g).tolist()
    bt = Batch(lens, torch.randint(0, 4, (70,), generator=g).tolist(), kvh=1, group=2, d=64, seed=22)
    pages = random_pages(bt, 3, g)
    out, lse = sparse_attention(bt.copier, "l", bt.q, pages.cuda(), bt.table, bt.seq_lens, cu_q=bt.cu_q)
    check_sparse(bt, pages, out, lse)


@pytest.mark.parametrize("layout,dtype,d", [("5d", "bf16", 128), ("4d", "f16", 64), ("5dpf", "f16", 128)])
@pytest.mark.parametrize("kvh,group,t", [(2, 4, 70), (1, 7, 33), (1, 16, 20), (2, 5, 40), (2, 3, 40)])
def test_sparse_rows_of_one_sequence(layout, dtype, d, kvh, group, t):
    """Many rows per sequence, each with a list of its own (some empty), ragged."""
    bt = Batch([t, 700, 1500], [t, t - 7, t], kvh=kvh, group=group, layout=layout, dtype=dtype, d=d, seed=t)
    pages = random_pages(bt, 11, torch.Generator().manual_seed(t))
    out, lse = sparse_attention(bt.copier, "l", bt.q, pages.cuda(), bt.table, bt.seq_lens, cu_q=bt.cu_q)
    assert _lib.device_errors(0) == 0
    check_sparse(bt, pages, out, lse)


@pytest.mark.parametrize("bs,k", [(1, 40), (8, 5), (64, 3), (5, 17), (128, 2)])
def test_sparse_rows_of_one_sequence_block_sizes(bs, k):
    bt = Batch([200, 333, 7], [64, 50, 7], bs=bs, kvh=1, group=4, seed=bs + k)
    pages = random_pages(bt, k, torch.Generator().manual_seed(k))
    out, lse = sparse_attention(bt.copier, "l", bt.q, pages.cuda(), bt.table, bt.seq_lens, cu_q=bt.cu_q)
    check_sparse(bt, pages, out, lse)


def test_sparse_rows_padding_repeats_bad_pages_and_graph():
    t = 40
    bt = Batch([900, 300], [t, t], kvh=2, group=4, seed=61)
    pages = random_pages(bt, 6, torch.Generator().manual_seed(3), holes=False).cuda()
    ref, ref_lse = sparse_attention(bt.copier, "l", bt.q, pages, bt.table, bt.seq_lens, cu_q=bt.cu_q)
    q = torch.cat([bt.q, torch.full((9, *bt.q.shape[1:]), math.nan, dtype=bt.q.dtype, device="cuda")])
    more = torch.cat([pages, torch.zeros((9, *pages.shape[1:]), dtype=torch.int32, device="cuda")])
    out, lse = torch.full_like(q, 5.0), torch.full(q.shape[:2], 5.0, device="cuda")
    sparse_attention(bt.copier, "l", q, more, bt.table, bt.seq_lens, cu_q=bt.cu_q, out=out, lse=lse)
    assert torch.equal(out[:2 * t], ref) and (out[2 * t:] == 5).all() and (lse[2 * t:] == 5).all()
    twice = pages.repeat_interleave(2, dim=2)
    out, lse = sparse_attention(bt.copier, "l", bt.q, twice, bt.table, bt.seq_lens, cu_q=bt.cu_q)
    assert torch.equal(out, ref) and torch.equal(lse, ref_lse) and _lib.device_errors(0) == 0
    far = torch.cat([pages, torch.full_like(pages[:, :, :1], 12345)], 2)
    out, lse = sparse_attention(bt.copier, "l", bt.q, far, bt.table, bt.seq_lens, cu_q=bt.cu_q)
    assert torch.equal(out, ref) and _lib.device_errors(0) == 4
    lens = bt.seq_lens.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, z = sparse_attention(bt.copier, "l", bt.q, pages, bt.table, lens, cu_q=bt.cu_q)
    o.fill_(3.0)
    g.replay()
    assert torch.equal(o, ref) and torch.equal(z, ref_lse)
    lens -= 60
    expect = sparse_attention(bt.copier, "l", bt.q, pages, bt.table, lens, cu_q=bt.cu_q)
    g.replay()
    assert torch.equal(o, expect[0]) and torch.equal(z, expect[1])


def test_sparse_nonfinite_values_stay_where_they_are_listed():
    """Rows of one tile: a page with infinities and NaN that only some of them list."""
    t = 32
    bt = Batch([500], [t], kvh=1, group=4, seed=62)
    pages = random_pages(bt, 8, torch.Generator().manual_seed(5), holes=False)
    pages[:, :, 0] = 0
    bad = 7
    for r in range(t):
        keep = [x for x in pages[r, 0].tolist() if x != bad]
        if r % 5 == 0:
            keep = sorted(set(keep[:7] + [bad]))
        pages[r, 0] = torch.tensor((keep + [-1] * 8)[:8], dtype=torch.int32)
    blk = int(bt.table[0, bad])
    bt.v[blk, 3, 0, 5] = math.inf
    bt.v[blk, 9, 0, 70] = math.nan
    out, lse = sparse_attention(bt.copier, "l", bt.q, pages.cuda(), bt.table, bt.seq_lens, cu_q=bt.cu_q)
    check_sparse(bt, pages, out, lse)
    for r in range(t):
        assert torch.isfinite(out[r]).all() == (r % 5 != 0)
        if r % 5 == 0:
            assert (out[r, :, 5] == math.inf).all() and torch.isnan(out[r, :, 70]).all()


@pytest.mark.parametrize("every", [1, 40])
def test_sparse_nonfinite_values_in_many_pages(every):
    """Long lists with an infinity in every page, or in every 40th: put back for
    the rows that list it and for no other."""
    t, k = 128, 40
    bt = Batch([16 * 500], [t], kvh=2, group=4, seed=63)
    pages = random_pages(bt, k, torch.Generator().manual_seed(7), holes=False)
    call = lambda: sparse_attention(bt.copier, "l", bt.q, pages.cuda(), bt.table, bt.seq_lens)
    finite, lse = call()
    marked = torch.arange(0, 500, every)
    bt.v[bt.table[0, marked.cuda()].long(), 3, :, 5] = math.inf  # token 3: a row may stand before it in its own page
    own = (bt.lens[0] - t + torch.arange(t)) // 16
    tok = (bt.lens[0] - t + torch.arange(t)) % 16
    hit = torch.isin(pages, marked.int()) & ((pages != own[:, None, None]) | (tok >= 3)[:, None, None])
    hit = hit.any(-1).repeat_interleave(bt.group, 1).cuda()
    out, lse2 = call()
    assert _lib.device_errors(0) == 0 and torch.equal(lse, lse2)
    assert torch.equal(out[..., 5] == math.inf, hit)
    out[..., 5] = finite[..., 5]
    assert torch.equal(out, finite)


def test_sparse_of_every_page_is_full_attention():
    bt = Batch([257, 64], [1, 1], seed=23)
    full, full_lse = run_tree(bt)
    pages = torch.arange(17, dtype=torch.int32, device="cuda").expand(2, bt.kvh, 17)  # stride 0 rows and heads
    table = bt.table.clamp(min=1)
    out, lse = sparse_attention(bt.copier, "l", bt.q, pages, table, bt.seq_lens, cu_q=bt.cu_q)
    for b in range(2):
        k, v = bt.kv64(b)
        check_attend(bt, out, lse, b, *attend64(bt.q64(b), k, v, bt.sees(b).repeat(bt.group, 1)[None], 1 / math.sqrt(bt.d)))
    assert torch.allclose(lse, full_lse, atol=1e-4, rtol=0)


def test_sparse_repeated_page_and_nothing_listed():
    bt = Batch([100], [1], seed=24)
    pages = torch.tensor([2, 2], dtype=torch.int32, device="cuda").expand(1, bt.kvh, 2).contiguous()
    once = sparse_attention(bt.copier, "l", bt.q, pages[:, :, :1].contiguous(), bt.table, bt.seq_lens)
    twice = sparse_attention(bt.copier, "l", bt.q, pages, bt.table, bt.seq_lens)
    assert torch.equal(twice[0], once[0]) and torch.equal(twice[1], once[1])
    none = sparse_attention(bt.copier, "l", bt.q, torch.full_like(pages, -1), bt.table, bt.seq_lens)
    assert (none[0] == 0).all() and (none[1] == -math.inf).all()


# ----------------------------------------------------------- refusals --
def test_refusals():
    bt = Batch([70, 33], [1, 1], seed=30)
    call = lambda q=bt.q, table=bt.table, lens=bt.seq_lens, **kw: tree_attention(bt.copier, "l", q, table, lens, **kw)
    bad = [
        dict(q=bt.q.float()), dict(q=bt.q.cpu()), dict(q=bt.q[:, :3]), dict(q=bt.q[:, :, :64]),
        dict(q=bt.q.transpose(0, 2)), dict(table=bt.table.long()), dict(table=bt.table[0]),
        dict(table=bt.table.cpu()), dict(table=bt.table.t().contiguous().t()), dict(lens=bt.seq_lens.long()),
        dict(lens=bt.seq_lens[:1]), dict(cu_q=bt.cu_q[:2]), dict(cu_q=bt.cu_q.long()), dict(scale=0.0),
        dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(out=torch.empty_like(bt.q, dtype=torch.float32)),
        dict(out=bt.q[:1]), dict(lse=torch.empty(2, 3, device="cuda")), dict(tree_mask=torch.zeros(1, dtype=torch.int64, device="cuda")),
        dict(tree_mask=torch.zeros(2, dtype=torch.int32, device="cuda")), dict(tree_mask=torch.zeros((2, 0), dtype=torch.int64, device="cuda")),
    ]
    for kw in bad:
        with pytest.raises((RuntimeError, ValueError)):
            call(**kw)
    with pytest.raises(RuntimeError, match="layer not registered"):
        tree_attention(bt.copier, "nope", bt.q, bt.table, bt.seq_lens)
    with pytest.raises(RuntimeError, match="divide evenly"):
        call(q=bt.q[:1])
    shifted = torch.empty(bt.q.numel() + 1, dtype=bt.q.dtype, device="cuda")[1:].view(bt.q.shape)
    with pytest.raises(RuntimeError, match="aligned"):
        call(q=shifted)
    pages = torch.zeros((2, bt.kvh, 2), dtype=torch.int32, device="cuda")
    for p in (pages.long(), pages[:1], pages[:, :1], pages[:, :, :0], pages.cpu()):
        with pytest.raises(RuntimeError):
            sparse_attention(bt.copier, "l", bt.q, p, bt.table, bt.seq_lens)
    for d, dt in ((80, torch.bfloat16), (128, torch.float32)):
        kv = torch.zeros((2, 4, 16, 2, d), dtype=dt, device="cuda")
        bt.copier.register_layer("x", kv, False)
        with pytest.raises((RuntimeError, ValueError)):
            tree_attention(bt.copier, "x", torch.zeros((2, 4, d), dtype=dt, device="cuda"), bt.table, bt.seq_lens)
    empty = call(q=bt.q[:0], cu_q=torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert empty[0].shape[0] == 0
    assert _lib.device_errors(0) == 0
