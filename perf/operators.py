"""Cases of the paged-cache attention, block selection and eviction operators, with plain forms in elementary torch.

Shapes follow this repository's configurations: 8 KV heads of 128 with 4 query heads each (Llama-3-8B, Mistral-7B), 4 KV
heads with 7 (Qwen2.5-7B), one KV head with 8 (a Llama-3-70B rank of eight), blocks of 16 tokens, prompts of 512 to 32K
tokens; the generic ones add 64 and 256 wide heads, other block sizes and the other cache layouts.
"""
import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------ cases --
def listed():
    a = {"op": "tree", "layout": "5d", "dtype": "bf16", "bs": 16, "hd": 128}
    s = {"op": "scores", "layout": "5d", "dtype": "bf16", "bs": 16, "hd": 128}
    b = {"op": "select", "layout": "5d", "dtype": "bf16", "bs": 16, "hd": 128}
    p = {"op": "sparse", "layout": "5d", "dtype": "bf16", "bs": 16, "hd": 128}
    c = {"op": "compact", "layout": "5d", "dtype": "bf16", "bs": 16, "hd": 128}
    return [
        # one request decodes one token over one reused chunk: latency
        dict(a, name="tree_one_token", batch=1, lo=513, hi=513, t=1, kvh=8, group=4),
        # a decode batch of 64 requests of mixed length, odd group of query heads, fp16
        dict(a, name="tree_decode_ragged", batch=64, lo=131, hi=8192, t=1, kvh=4, group=7, dtype="f16"),
        # 16 requests verify trees of up to 16 drafted tokens after an 8K prompt
        dict(a, name="tree_draft_8k", batch=16, lo=6001, hi=8209, t=16, kvh=8, group=4),
        # one rank of eight of the 70B shape verifies 64 drafted tokens at 32K: the most arithmetic
        dict(a, name="tree_shard_32k", batch=8, lo=30001, hi=32768, t=64, kvh=1, group=8),
        # a window of the last 32 prompt tokens scores an 8K prompt (no lse in hand)
        dict(s, name="scores_window_8k", batch=1, lo=8192, hi=8192, t=32, kvh=8, group=4, lse=False, add=False),
        # each decode step adds its weights to the scores of 32 long requests (lse from the attention)
        dict(s, name="scores_decode_32k", batch=32, lo=4099, hi=32768, t=1, kvh=8, group=4, lse=True, add=True),
        # page bounds of a whole batch of prompts, then the first selection
        dict(b, name="select_after_prefill", batch=16, lo=2047, hi=8192, t=1, kvh=8, group=4, k=64, whole=True),
        # one decode step over long requests: refresh the last page, select of 8K pages
        dict(b, name="select_decode_128k", batch=8, lo=98765, hi=131072, t=1, kvh=8, group=4, k=128, whole=False),
        # the attention of that step over 128 selected pages, 64 requests
        dict(p, name="sparse_decode_32k", batch=64, lo=17001, hi=32768, t=1, kvh=8, group=4, k=128),
        # 512 prompt tokens of one request, each with its own 64 pages of an 8K context
        dict(p, name="sparse_chunk_8k", batch=1, lo=8191, hi=8191, t=512, kvh=8, group=4, k=64),
        # an 8K prompt of all 32 layers shrinks to 40%, keys re-rotated to their new places
        dict(c, name="compact_prompt_8k", batch=1, lo=8192, hi=8192, kvh=8, layers=32, keep=0.4, per_head=False, rotate=True),
        # one layer of 6 requests shrinks to 60% per KV head, keys as they are, head-major packed layout, fp16
        dict(c, name="compact_layer_ragged", batch=6, lo=257, hi=6001, kvh=4, layers=1, keep=0.6, per_head=True, rotate=False,
             layout="4d", dtype="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "scores", "select", "sparse", "compact"])
    case = {"op": op, "layout": rng.choice(["5d", "5dpf", "4d"]), "dtype": rng.choice(["bf16", "bf16", "f16"]),
            "bs": rng.choice([16, 16, 16, 8, 32, 64]), "hd": rng.choice([128, 128, 64, 256])}
    kvh, group = rng.choice([(8, 4), (8, 4), (4, 7), (1, 8), (2, 5), (8, 1), (1, 16)])
    case |= {"kvh": kvh, "group": group}
    row = 2 * kvh * case["hd"] * 2  # K and V bytes of a token
    most = 300_000_000 // row  # tokens of a batch
    case["batch"] = _log(rng, 1, 48)
    case["hi"] = _log(rng, 33, min(32768, max(256, most // case["batch"])))
    case["lo"] = rng.randint(max(1, case["hi"] // 4), case["hi"])
    if op in ("tree", "scores"):
        rows = max(1, min(64, 120_000_000 // (case["batch"] * case["hi"] * kvh * group)))
        case["t"] = _log(rng, 1, rows)
        case["lo"], case["hi"] = max(case["lo"], case["t"]), max(case["hi"], case["t"])
    if op == "scores":
        case |= {"lse": rng.random() < 0.5, "add": rng.random() < 0.5}
    if op == "select":
        case |= {"t": 1, "k": _log(rng, 4, 160), "whole": rng.random() < 0.5}
    if op == "sparse":
        case["t"] = _log(rng, 1, max(1, 256 // case["batch"]))
        case["k"] = _log(rng, 2, max(2, 2048 // case["bs"]))
        case["lo"], case["hi"] = max(case["lo"], case["t"]), max(case["hi"], case["t"])
    if op == "compact":
        case.pop("group")
        case |= {"layers": rng.choice([1, 1, 2, 4]), "keep": round(rng.uniform(0.05, 0.95), 3),
                 "per_head": rng.random() < 0.4, "rotate": rng.random() < 0.6}
    return case


def _lens(case):
    """Length and query rows of each request of the case, in a fixed order (a seed permutes the requests)."""
    n, lo, hi = case["batch"], case["lo"], case["hi"]
    lens = [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]
    t = case.get("t", 0)
    rows = [t if i == n - 1 or t < 2 or case["op"] != "tree" else max(1, t - (5 * i) % t) for i in range(n)]
    return lens, rows


def work(case):
    lens, rows = _lens(case)
    h, d, bs, es = case["kvh"], case["hd"], case["bs"], 4 if case["dtype"] == "f32" else 2
    tok, nrows = sum(lens), sum(rows)
    op = case["op"]
    if op == "compact":
        kept = sum(int(case["keep"] * n) for n in lens) * case["layers"]
        idx = 4 * kept * (h if case["per_head"] else 1)
        table = 2 * 4 * d * max(lens) if case["rotate"] else 0
        return {"bytes": 2 * 2 * kept * h * d * es + idx + table, "flops": 6 * kept * h * d if case["rotate"] else 0}
    hq = h * case["group"]
    pages = sum(-(-n // bs) for n in lens)
    qio = nrows * hq * d * es
    if op == "tree":
        dots = sum(t * n for t, n in zip(rows, lens)) * hq
        return {"bytes": 2 * tok * h * d * es + 2 * qio + 4 * nrows * hq + 4 * pages + 8 * nrows, "flops": 4 * dots * d}
    if op == "scores":
        dots = sum(t * n for t, n in zip(rows, lens)) * hq
        lse = 4 * nrows * hq if case["lse"] else 0
        return {"bytes": tok * h * d * es + qio + lse + 4 * pages + (8 if case["add"] else 4) * h * tok,
                "flops": 2 * dots * d * (1 if case["lse"] else 2)}
    if op == "select":
        new = tok if case["whole"] else sum((n - 1) % bs + 1 for n in lens)
        fresh = pages if case["whole"] else len(lens)
        bounds = 2 * h * d * es
        return {"bytes": new * h * d * es + fresh * bounds + (0 if case["whole"] else pages * bounds) + qio + 4 * pages
                + 4 * nrows * h * case["k"], "flops": 4 * pages * hq * d + 2 * new * h * d}
    seen, dots = 0, 0  # sparse: distinct pages are read once
    for n, t in zip(lens, rows):
        full = -(-n // bs)
        per = min(case["k"], full)
        seen += min(per * t, full)
        dots += per * t * bs
    return {"bytes": 2 * seen * bs * h * d * es + 2 * qio + 4 * nrows * hq + 4 * nrows * h * case["k"],
            "flops": 4 * dots * hq * d}


# ----------------------------------------------------------------- inputs --
def _planes(cache, layout, d):
    """K and V of a layer (or a stack of layers) as [..., block, token, head, dim] views."""
    if layout == "5d":
        return cache.select(-5, 0), cache.select(-5, 1)
    if layout == "5dpf":
        return cache.select(-4, 0), cache.select(-4, 1)
    return cache[..., :d].transpose(-3, -2), cache[..., d:].transpose(-3, -2)


def _shape(layout, nb, bs, h, d):
    return {"5d": (2, nb, bs, h, d), "5dpf": (nb, 2, bs, h, d), "4d": (nb, h, bs, 2 * d)}[layout]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, d, h, bs = _DT[case["dtype"]], case["hd"], case["kvh"], case["bs"]
    lens, rows = _lens(case)
    order = list(range(case["batch"]))
    random.Random(seed).shuffle(order)
    lens, rows = [lens[i] for i in order], [rows[i] for i in order]
    pages = [-(-n // bs) for n in lens]
    wide = max(pages)
    nb = sum(pages) + 1
    layers = case.get("layers", 1)
    cache = torch.empty((layers, *_shape(case["layout"], nb, bs, h, d)), dtype=dt, device="cuda")
    for l in range(layers):
        cache[l].normal_(generator=g)
        k = _planes(cache[l], case["layout"], d)[0]
        k[..., torch.randperm(d, generator=g, device="cuda")[:4]] *= 8.0  # outlier key channels
    ids = torch.randperm(nb - 1, generator=g, device="cuda").to(torch.int32) + 1
    at = torch.tensor([0] + pages, device="cuda").cumsum(0)
    col = torch.arange(wide, device="cuda")
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    inside = col[None] < torch.tensor(pages, device="cuda")[:, None]
    table = torch.where(inside, ids[(at[:-1, None] + col[None]).clamp(max=nb - 2)], 0).to(torch.int32)
    st = {"case": dict(case), "cache": cache, "table": table, "lens": lens_t}
    names = ["layers.%d" % l for l in range(layers)]
    if case["op"] == "compact":
        kept = [int(case["keep"] * n) for n in lens]
        lists = layers * (h if case["per_head"] else 1)
        idx = torch.empty((lists, max(1, sum(kept))), dtype=torch.int32, device="cuda")
        off = 0
        for n, m in zip(lens, kept):  # the kept positions, ascending, as a top-k selection gives them
            pick = torch.rand((lists, n), generator=g, device="cuda").topk(m, dim=1).indices if m else idx[:, :0].long()
            idx[:, off:off + m] = pick.sort(dim=1).values.to(torch.int32)
            off += m
        freq = 5e5 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
        angle = torch.arange(max(lens), dtype=torch.float64, device="cuda")[:, None] * freq[None]
        st |= {"idx": idx, "kept": kept, "rope": torch.cat([angle.cos(), angle.sin()], 1).float(), "names": names}
        st["flat_table"] = ids
        st["table_off"] = at[:-1].tolist()
    else:
        n, hq = sum(rows), h * case["group"]
        st["q"] = torch.randn((n, hq, d), generator=g, device="cuda", dtype=torch.float32).to(dt)
        st["rows"], st["widest"] = rows, max(rows)
        st["cu_q"] = torch.tensor([0] + rows, device="cuda").cumsum(0).to(torch.int32)
    if case["op"] == "tree":
        masks, r = [], random.Random(seed + 1)
        for t in rows:  # token j hangs from an earlier one, or starts a branch
            bits = []
            for j in range(t):
                up = r.randint(max(-1, j - 4), j - 1) if j else -1
                bits.append((bits[up] if up >= 0 else 0) | 1 << j)
            masks += [b - (1 << 64) if b >> 63 else b for b in bits]
        st["mask"] = torch.tensor(masks, dtype=torch.int64, device="cuda")
    if case["op"] == "scores":
        total = sum(lens)
        st["col_off"] = torch.tensor([0] + lens, device="cuda").cumsum(0)[:-1].contiguous()
        st["scores"] = torch.rand((h, total), generator=g, device="cuda") if case["add"] else \
            torch.zeros((h, total), device="cuda")
        # about the log-sum of normal logits of this spread, per row and head
        base = torch.log(lens_t.float()).repeat_interleave(st["cu_q"].diff().long()) + 1.5
        st["lse"] = base[:, None] + 0.3 * torch.rand((n, hq), generator=g, device="cuda") if case["lse"] else None
    if case["op"] == "select":
        st["start"] = torch.zeros_like(lens_t) if case["whole"] else lens_t - 1
        k = _planes(cache[0], case["layout"], d)[0]
        st["bounds"] = torch.stack([k.amin(1), k.amax(1)], 2).contiguous()  # as earlier steps left them
    if case["op"] == "sparse":
        last = (lens_t - torch.tensor(rows, device="cuda")).repeat_interleave(st["cu_q"].diff().long()) + \
            torch.cat([torch.arange(t, device="cuda") for t in rows])
        have = (last // bs + 1)[:, None, None]
        luck = torch.rand((n, h, wide), generator=g, device="cuda")
        luck = torch.where((col == 0) | (col == have - 1), 2.0, luck).where(col < have, -1.0)
        best = luck.topk(min(case["k"], wide), dim=2)
        pick = torch.where(best.values < 0, wide, best.indices).sort(dim=2).values
        pick = torch.where(pick == wide, -1, pick)
        fill = torch.full((n, h, case["k"] - pick.shape[2]), -1, device="cuda", dtype=pick.dtype)
        st["pages"] = torch.cat([pick, fill], 2).to(torch.int32).contiguous()
    if own:
        from daric_b200.cache_ops import CacheCopier
        from daric_b200.select import Selection
        st["copier"] = CacheCopier()
        for l in range(layers):
            st["copier"].register_layer("layers.%d" % l, cache[l], case["layout"] != "5d")
            if case["op"] == "compact" and case["rotate"]:
                st["copier"].register_rotary("layers.%d" % l, st["rope"], d, True)
        if case["op"] == "compact":
            import numpy as np
            lists = st["idx"].shape[0]
            count = torch.tensor([st["kept"]] * lists, dtype=torch.int32, device="cuda")
            off = np.concatenate([[0], np.cumsum(st["kept"])[:-1]]).astype(np.int64)
            st["keep"] = Selection(idx=st["idx"], slot=None, count=count, out_off=off)
    return st


# -------------------------------------------------------------- the calls --
def run(st):
    case = st["case"]
    return (_own if own else _plain)[case["op"]](st, case)


def _own_tree(st, case):
    from daric_b200.attend import tree_attention
    return tree_attention(st["copier"], "layers.0", st["q"], st["table"], st["lens"], cu_q=st["cu_q"], tree_mask=st["mask"])


def _own_scores(st, case):
    from daric_b200.evict import attention_scores
    return attention_scores(st["copier"], "layers.0", st["q"], st["table"], st["lens"], st["scores"], st["col_off"],
                            cu_q=st["cu_q"], lse=st["lse"], accumulate=case["add"])


def _own_select(st, case):
    from daric_b200.blocks import page_bounds, select_pages
    page_bounds(st["copier"], "layers.0", st["table"], st["lens"], st["bounds"], start=st["start"])
    pages = select_pages(st["q"], st["bounds"], st["table"], st["lens"], case["k"], case["bs"], cu_q=st["cu_q"])
    return st["bounds"], pages


def _own_sparse(st, case):
    from daric_b200.attend import sparse_attention
    return sparse_attention(st["copier"], "layers.0", st["q"], st["pages"], st["table"], st["lens"], cu_q=st["cu_q"])


def _own_compact(st, case):
    from daric_b200.evict import compact
    compact(st["copier"], st["names"], st["keep"], st["flat_table"], seg_blk_off=st["table_off"],
            per_head=case["per_head"], mode="flexible" if case["rotate"] else "none")
    return st["cache"]


# ---------------------------------------------------------- plain forms --
def _rows_of(st, lens):
    """Each query row's request, place in it and position in its request."""
    cu = st["cu_q"].long()
    req = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), cu.diff(), output_size=st["q"].shape[0])
    j = torch.arange(st["q"].shape[0], device="cuda") - cu[req]
    return req, j, lens.long()[req] - cu.diff()[req] + j


def _padded(st, x, fill=0.0):
    """Rows [N, ...] as [batch, widest, ...]; and where the rows stand in it."""
    req, j, _ = _rows_of(st, st["lens"])
    out = torch.full((st["lens"].shape[0], st["widest"], *x.shape[1:]), fill, dtype=x.dtype, device="cuda")
    out[req, j] = x
    return out, req, j


def _logits(st, case):
    """Scaled logits [batch, kv head, group * widest, position] and what each row sees."""
    h, d, group, w = case["kvh"], case["hd"], case["group"], st["widest"]
    k = _planes(st["cache"][0], case["layout"], d)[0][st["table"].long()].flatten(1, 2).float()
    q, req, j = _padded(st, st["q"].float())
    q = q.view(-1, w, h, group, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))
    pos = torch.arange(k.shape[1], device="cuda")
    ctx = st["lens"].long() - st["cu_q"].long().diff()
    draft = pos[None, None] - ctx[:, None, None]  # [batch, 1, position]
    rowno = torch.arange(w, device="cuda")[None, :, None]
    if "mask" in st:
        bits = _padded(st, st["mask"], 0)[0][:, :, None]
        sees = (draft < 0) | ((draft < 64) & ((bits >> draft.clamp(0, 63)) & 1).bool())
    else:
        sees = draft <= rowno
    sees = sees & (rowno < st["cu_q"].long().diff()[:, None, None]) & (pos < st["lens"][:, None, None])
    sees = sees[:, None, None].expand(-1, 1, group, -1, -1).flatten(2, 3)
    return x.masked_fill(~sees, -math.inf), req, j


def _softmax(x):
    """exp(x - max), its sum and the log-sum along the last axis; rows without a finite value have sum 0."""
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return p, total, (top + torch.log(total)).squeeze(-1)


def _unpad(x, case, w, req, j):
    """[batch, kv head, group * widest, ...] back to rows [N, query head, ...]."""
    x = x.unflatten(2, (case["group"], w)).flatten(1, 2)
    return x[req, :, j]


def _plain_tree(st, case):
    x, req, j = _logits(st, case)
    p, total, lse = _softmax(x)
    v = _planes(st["cache"][0], case["layout"], case["hd"])[1][st["table"].long()].flatten(1, 2).float()
    v = v.masked_fill((torch.arange(v.shape[1], device="cuda") >= st["lens"][:, None])[..., None, None], 0.0)
    out = torch.matmul(p, v.transpose(1, 2)) / torch.where(total == 0, 1.0, total)
    w = st["widest"]
    return _unpad(out, case, w, req, j).to(st["q"].dtype), _unpad(lse, case, w, req, j)


def _plain_scores(st, case):
    x, req, j = _logits(st, case)
    if case["lse"]:
        lse, _, _ = _padded(st, st["lse"], 0.0)
        lse = lse.view(len(lse), -1, case["kvh"], case["group"]).permute(0, 2, 3, 1).flatten(2, 3)
    else:
        lse = _softmax(x)[2]
        lse = torch.where(lse == -math.inf, 0.0, lse)
    weight = torch.exp(x - lse[..., None]).sum(2)  # [batch, kv head, position]
    inside = torch.arange(weight.shape[2], device="cuda") < st["lens"][:, None]
    found = weight.transpose(0, 1)[:, inside]
    return st["scores"].add_(found) if case["add"] else st["scores"].copy_(found)


def _plain_select(st, case):
    h, d, bs, k = case["kvh"], case["hd"], case["bs"], case["k"]
    table, lens = st["table"].long(), st["lens"].long()
    keys = _planes(st["cache"][0], case["layout"], d)[0]
    page = torch.arange(table.shape[1], device="cuda")
    fresh = (page >= st["start"].long()[:, None] // bs) & (page * bs < lens[:, None])
    seq = fresh.nonzero()[:, 0]
    ids = table[fresh]
    part = keys[ids]
    tok = (page.expand_as(table)[fresh] * bs)[:, None] + torch.arange(bs, device="cuda")
    gone = (tok >= lens[seq][:, None])[..., None, None]
    st["bounds"][ids] = torch.stack([part.masked_fill(gone, math.inf).amin(1), part.masked_fill(gone, -math.inf).amax(1)], 2)
    req, _, pos = _rows_of(st, st["lens"])
    q = st["q"].double().view(-1, h, case["group"], d)  # 64 bits: pages next to the border
    near = st["bounds"][table].double()  # [batch, page, head, 2, dim]
    lo = near[:, :, :, 0].permute(0, 2, 3, 1)[req]
    hi = near[:, :, :, 1].permute(0, 2, 3, 1)[req]
    u = (torch.matmul(q.clamp(min=0), hi) + torch.matmul(q.clamp(max=0), lo)).amax(2)  # [row, head, page]
    have = (pos // bs + 1)[:, None, None]
    u = torch.where((page < 1) | (page >= have - 1), math.inf, u).masked_fill(page >= have, -math.inf)
    best = u.sort(dim=2, descending=True, stable=True).indices[:, :, :k]
    best = torch.where(best < have, best, page.shape[0]).sort(dim=2).values
    out = torch.full((best.shape[0], h, k), -1, dtype=torch.int32, device="cuda")
    out[:, :, :best.shape[2]] = torch.where(best == page.shape[0], -1, best)
    return st["bounds"], out


def _plain_sparse(st, case):
    h, d, bs, group = case["kvh"], case["hd"], case["bs"], case["group"]
    req, _, pos = _rows_of(st, st["lens"])
    logical = st["pages"].long()
    ids = st["table"].long()[req[:, None, None], logical.clamp(min=0)]  # [row, head, k]
    head = torch.arange(h, device="cuda")[None, :, None]
    k, v = _planes(st["cache"][0], case["layout"], d)
    at = logical[..., None] * bs + torch.arange(bs, device="cuda")
    sees = ((logical >= 0)[..., None] & (at <= pos[:, None, None, None])).flatten(2, 3)
    keys = k[ids, :, head].flatten(2, 3).float()  # [row, head, k * bs, dim]
    x = torch.matmul(st["q"].float().view(-1, h, group, d), keys.transpose(2, 3)) * (1.0 / math.sqrt(d))
    p, total, lse = _softmax(x.masked_fill(~sees[:, :, None], -math.inf))
    del keys
    vals = v[ids, :, head].flatten(2, 3).float().masked_fill(~sees[..., None], 0.0)
    out = torch.matmul(p, vals) / torch.where(total == 0, 1.0, total)
    return out.flatten(1, 2).to(st["q"].dtype), lse.flatten(1, 2)


def _plain_compact(st, case):
    h, d, bs = case["kvh"], case["hd"], case["bs"]
    lists, n = st["idx"].shape[0], sum(st["kept"])
    layers = case["layers"]
    kept = torch.tensor(st["kept"], device="cuda")
    seg = torch.repeat_interleave(torch.arange(len(st["kept"]), device="cuda"), kept)
    new = torch.arange(n, device="cuda") - (kept.cumsum(0) - kept)[seg]
    first = torch.tensor(st["table_off"], device="cuda")[seg]
    ids = st["flat_table"].long()
    old = st["idx"][:, :n].long().view(layers, lists // layers, n).expand(layers, h, n)
    l = torch.arange(layers, device="cuda")[:, None, None]
    head = torch.arange(h, device="cuda")[None, :, None]
    src, dst = ids[first + old // bs], ids[first + new // bs].expand(layers, h, n)
    k, v = _planes(st["cache"], case["layout"], d)
    keys, vals = k[l, src, old % bs, head], v[l, src, old % bs, head]
    if case["rotate"]:
        oc, os = st["rope"][old].chunk(2, dim=-1)
        nc, ns = st["rope"][new].chunk(2, dim=-1)
        c, s = nc * oc + ns * os, ns * oc - nc * os
        a, b = keys.float().chunk(2, dim=-1)
        keys = torch.cat([a * c - b * s, b * c + a * s], -1).to(keys.dtype)
    k[l, dst, (new % bs).expand(layers, h, n), head] = keys
    v[l, dst, (new % bs).expand(layers, h, n), head] = vals
    return st["cache"]


_own = {"tree": _own_tree, "scores": _own_scores, "select": _own_select, "sparse": _own_sparse, "compact": _own_compact}
_plain = {"tree": _plain_tree, "scores": _plain_scores, "select": _plain_select, "sparse": _plain_sparse,
          "compact": _plain_compact}


# ---------------------------------------------------------------- exact --
def exact(case, seed):
    """The operators by their definitions in 64 bits, request by request."""
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return {"tree": _exact_attend, "scores": _exact_scores, "select": _exact_select, "sparse": _exact_attend,
            "compact": _exact_compact}[case["op"]](st, case)


def _exact_kv(st, case, b, positions):
    """K and V in 64 bits of request b at the positions, [head, position, dim]."""
    bs = case["bs"]
    k, v = _planes(st["cache"][0], case["layout"], case["hd"])
    ids = st["table"][b].long()[positions // bs]
    return k[ids, positions % bs].double().transpose(0, 1), v[ids, positions % bs].double().transpose(0, 1)


def _exact_attend(st, case):
    hq, d, h, bs = case["kvh"] * case["group"], case["hd"], case["kvh"], case["bs"]
    n = st["q"].shape[0]
    out = torch.zeros((n, hq, d), dtype=torch.float64, device="cuda")
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64, device="cuda")
    row = 0
    for b, t in enumerate(st["rows"]):
        s = int(st["lens"][b])
        q = st["q"][row:row + t].double().view(t, h, case["group"], d)
        every = torch.arange(s, device="cuda")
        step = max(1, min(t, 400_000_000 // (s * hq)))
        for r in range(0, t, step):
            m = min(step, t - r)
            k, v = _exact_kv(st, case, b, every)
            x = torch.einsum("thgd,hsd->thgs", q[r:r + m], k) / math.sqrt(d)
            if case["op"] == "tree":
                ok = torch.ones((m, s), dtype=torch.bool, device="cuda")
                bits = st["mask"][row + r:row + r + m]
                for i in range(t):
                    ok[:, s - t + i] = (bits >> i) & 1 == 1
                ok = ok[:, None, None]
            else:
                listed_ = torch.zeros((m, h, -(-s // bs) + 1), dtype=torch.bool, device="cuda")
                pg = st["pages"][row + r:row + r + m].long()
                listed_.scatter_(2, torch.where(pg < 0, listed_.shape[2] - 1, pg), True)
                ok = listed_[:, :, every // bs] & (every <= torch.arange(s - t + r, s - t + r + m, device="cuda")[:, None])[:, None]
                ok = ok[:, :, None]
            x = torch.where(ok, x, -math.inf)
            z = torch.logsumexp(x, -1)
            p = torch.where(ok, (x - z[..., None]).exp(), 0.0)
            out[row + r:row + r + m] = torch.einsum("thgs,hsd->thgd", p, v).flatten(1, 2)
            lse[row + r:row + r + m] = z.flatten(1, 2)
            del x, p, k, v
        row += t
    return out, lse


def _exact_scores(st, case):
    d, h = case["hd"], case["kvh"]
    total = st["scores"].double().clone()
    row = 0
    for b, t in enumerate(st["rows"]):
        s, c0 = int(st["lens"][b]), int(st["col_off"][b])
        every = torch.arange(s, device="cuda")
        k = _exact_kv(st, case, b, every)[0]
        q = st["q"][row:row + t].double().view(t, h, case["group"], d)
        x = torch.einsum("thgd,hsd->thgs", q, k) / math.sqrt(d)
        x = x.masked_fill((every > torch.arange(s - t, s, device="cuda")[:, None])[:, None, None], -math.inf)
        z = st["lse"][row:row + t].double().view(t, h, -1) if case["lse"] else torch.logsumexp(x, -1)
        total[:, c0:c0 + s] += (x - z[..., None]).exp().sum((0, 2))
        row += t
    return total


def _exact_select(st, case):
    bs, h, k = case["bs"], case["kvh"], case["k"]
    bounds = st["bounds"].double().clone()
    pages = torch.full((st["q"].shape[0], h, k), -1, dtype=torch.int32, device="cuda")
    row = 0
    for b, t in enumerate(st["rows"]):
        s = int(st["lens"][b])
        have = -(-s // bs)
        p0 = int(st["start"][b]) // bs
        keys = _exact_kv(st, case, b, torch.arange(p0 * bs, s, device="cuda"))[0]
        for i in ([have - 1] if not case["whole"] else [p0, have - 1]):  # the first and the (ragged) last by themselves
            part = keys[:, i * bs - p0 * bs:(i + 1) * bs - p0 * bs]
            bounds[st["table"][b, i].long()] = torch.stack([part.min(1).values, part.max(1).values], 1)
        if case["whole"] and have > 2:
            part = keys[:, :(have - 1) * bs].unflatten(1, (have - 1, bs)).transpose(0, 1)
            bounds[st["table"][b, :have - 1].long()] = torch.stack([part.min(2).values, part.max(2).values], 2)
        near = bounds[st["table"][b, :have].long()]  # [page, head, 2, dim]
        for r in range(t):
            q = st["q"][row + r].double().view(h, case["group"], 1, -1)
            u = torch.empty((h, have), dtype=torch.float64, device="cuda")
            for at in range(0, have, 512):
                part = near[at:at + 512].transpose(0, 1)[:, None]  # [head, 1, page, 2, dim]
                u[:, at:at + 512] = torch.maximum(q * part[:, :, :, 0], q * part[:, :, :, 1]).sum(-1).amax(1)
            seen = (s - t + r) // bs + 1
            u[:, 0] = math.inf
            u[:, seen - 1] = math.inf
            best = u[:, :seen].sort(dim=1, descending=True, stable=True).indices[:, :k].sort(dim=1).values
            pages[row + r, :, :best.shape[1]] = best.to(torch.int32)
        row += t
    return bounds, pages


def _exact_compact(st, case):
    h, d, bs = case["kvh"], case["hd"], case["bs"]
    if st["cache"].numel() > 1_200_000_000:
        return None
    out = st["cache"].double()
    k, v = _planes(out, case["layout"], d)
    k0, v0 = _planes(st["cache"], case["layout"], d)
    per = h if case["per_head"] else 1
    for l in range(case["layers"]):
        off = 0
        for b, m in enumerate(st["kept"]):
            ids = st["flat_table"][st["table_off"][b]:].long()
            new = torch.arange(m, device="cuda")
            for e in range(per):
                old = st["idx"][l * per + e, off:off + m].long()
                hs = slice(e, e + 1) if case["per_head"] else slice(0, h)
                a = k0[l, ids[old // bs], old % bs, hs].double()
                if case["rotate"]:
                    f = st["rope"].double()
                    o, w = torch.complex(f[old, :d // 2], f[old, d // 2:]), torch.complex(f[new, :d // 2], f[new, d // 2:])
                    z = torch.complex(a[..., :d // 2], a[..., d // 2:]) * (w * o.conj())[:, None]
                    a = torch.cat([z.real, z.imag], -1)
                k[l, ids[new // bs], new % bs, hs] = a
                v[l, ids[new // bs], new % bs, hs] = v0[l, ids[old // bs], old % bs, hs].double()
            off += m
    return out
