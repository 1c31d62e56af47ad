"""Batches and 64-bit references of the paged-cache attention operators."""
from __future__ import annotations

import math

import torch

from daric_b200.cache_ops import CacheCopier

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def planes(cache, layout, d):
    """K and V of a layer as [block, token, head, dim] views."""
    if layout == "5d":
        return cache[0], cache[1]
    if layout == "5dpf":
        return cache[:, 0], cache[:, 1]
    return cache[..., :d].transpose(1, 2), cache[..., d:].transpose(1, 2)


class Batch:
    """A registered layer with random contents, a block table of shuffled
    blocks per sequence and query rows."""

    def __init__(self, lens, rows, *, kvh=2, group=4, d=128, bs=16, dtype="bf16", layout="5d", seed=0, spread=1.0,
                 extra_cols=1, uniform_rows=False):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.rows, self.kvh, self.group, self.d, self.bs, self.layout = lens, rows, kvh, group, d, bs, layout
        dt = DT[dtype]
        pages = [-(-n // bs) for n in lens]
        self.nb = nb = sum(pages) + 3
        shape = {"5d": (2, nb, bs, kvh, d), "5dpf": (nb, 2, bs, kvh, d), "4d": (nb, kvh, bs, 2 * d)}[layout]
        self.cache = (torch.randn(shape, generator=g) * spread).to(dt).cuda()
        ids = torch.randperm(nb - 1, generator=g) + 1
        cols = max(pages) + extra_cols
        self.table = torch.zeros((len(lens), max(cols, 1)), dtype=torch.int32)
        at = 0
        for b, n in enumerate(pages):
            self.table[b, :n] = ids[at:at + n]
            at += n
        self.table = self.table.cuda()
        self.seq_lens = torch.tensor(lens, dtype=torch.int32).cuda()
        self.cu = [0]
        for r in rows:
            self.cu.append(self.cu[-1] + r)
        self.cu_q = None if uniform_rows else torch.tensor(self.cu, dtype=torch.int32).cuda()
        self.n = self.cu[-1]
        self.q = torch.randn((self.n, kvh * group, d), generator=g).to(dt).cuda()
        self.copier = CacheCopier()
        self.copier.register_layer("l", self.cache, layout != "5d")
        self.k, self.v = planes(self.cache, layout, d)

    def kv64(self, b):
        """K and V of sequence b in 64 bits: [head, position, dim]."""
        pos = torch.arange(self.lens[b], device="cuda")
        blk = self.table[b].long()[pos // self.bs]
        return (self.k[blk, pos % self.bs].double().transpose(0, 1).contiguous(),
                self.v[blk, pos % self.bs].double().transpose(0, 1).contiguous())

    def q64(self, b):
        """[head, group * rows, dim] with row j of group member e at e * rows + j."""
        t = self.rows[b]
        q = self.q[self.cu[b]:self.cu[b + 1]].double().view(t, self.kvh, self.group, self.d)
        return q.permute(1, 2, 0, 3).reshape(self.kvh, self.group * t, self.d)

    def sees(self, b, mask=None):
        """[rows, positions] truth table. mask: int64 [n, words] on the CPU or None."""
        t, s = self.rows[b], self.lens[b]
        i = torch.arange(s)[None] - (s - t)
        j = torch.arange(t)[:, None]
        if mask is None:
            return ((i < 0) | (i <= j)).cuda()
        m = mask[self.cu[b]:self.cu[b + 1]]
        word = (i.clamp(min=0) // 64).expand(t, s)
        bits = torch.gather(m, 1, word.clamp(max=m.shape[1] - 1)) >> (i.clamp(min=0) % 64)
        return ((i < 0) | ((bits & 1).bool() & (word < m.shape[1]))).cuda()


def attend64(q, k, v, ok, scale):
    """out, lse, sum of weight * |v| and the error bound of a logit, in 64 bits.
    q [h, r, d], k and v [h, s, d], ok broadcastable to [h, r, s]."""
    x = torch.matmul(q, k.transpose(1, 2)) * scale
    x = torch.where(ok, x, -math.inf)
    top = x.amax(-1, keepdim=True) if x.shape[-1] else torch.full((*x.shape[:2], 1), -math.inf, device=x.device, dtype=x.dtype)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    p = torch.where(ok, p, 0.0)
    total = p.sum(-1, keepdim=True)
    w = p / torch.where(total == 0, 1.0, total)
    any_v = ok.expand(x.shape)
    out = torch.where(any_v.any(-1, keepdim=True), torch.matmul(w, v), 0.0) if torch.isfinite(v).all() else \
        torch.where(any_v[..., None], w[..., None] * v[:, None], 0.0).sum(2)
    lse = (top + torch.log(total)).squeeze(-1)
    # |fp32 logit - exact|: d products, exact each, every addition off by at most 2^-23 of the
    # sum of magnitudes (two units in the last place: matrix instructions may cut off), then the
    # scale and the difference to the maximum
    mag = torch.matmul(q.abs(), torch.nan_to_num(k, 0.0, 0.0, 0.0).abs().transpose(1, 2))
    mag = torch.where(any_v, mag, 0.0).amax(-1) if mag.shape[-1] else torch.zeros(q.shape[:2], device=q.device, dtype=q.dtype)
    e = (q.shape[-1] + 8) * 2.0 ** -23 * mag * scale + 2.0 ** -22
    absv = torch.matmul(w, torch.nan_to_num(v, 0.0, 0.0, 0.0).abs())
    return out, lse, absv, e


def check_attend(bt, got_out, got_lse, b, out, lse, absv, e):
    """Compares rows of sequence b. Tolerance: the output's rounding (half), each
    weight's rounding before the second product (half of the same type) and
    twice the logit error on both numerator and denominator, of sum w |v|."""
    t = bt.rows[b]
    h = HALF[bt.cache.dtype]
    o = got_out[bt.cu[b]:bt.cu[b + 1]].double().view(t, bt.kvh, bt.group, bt.d).permute(1, 2, 0, 3).reshape(out.shape)
    z = got_lse[bt.cu[b]:bt.cu[b + 1]].double().view(t, bt.kvh, bt.group).permute(1, 2, 0).reshape(lse.shape)
    fine = torch.isfinite(out)
    assert torch.equal(torch.isnan(out), torch.isnan(o))
    assert torch.equal(out[~fine & ~torch.isnan(out)], o[~fine & ~torch.isnan(out)])
    # sums over up to n keys in fp32: n 2^-24 relative, far below the rest for n < 2^15
    tol = h * out.abs() * (1 + h) + (h + 4 * e[..., None] + 2.0 ** -9 * h) * absv + 2.0 ** -24
    bad = ((o - out).abs() > tol) & fine
    assert not bad.any(), (int(bad.sum()), float(((o - out).abs() / tol)[fine].max()))
    none = lse == -math.inf
    assert torch.equal(none, z == -math.inf)
    ztol = 2 * e + 2.0 ** -22 * (lse.abs() + 1) + bt.lens[b] * 2.0 ** -24
    bad = ((z - lse).abs() > ztol) & torch.isfinite(lse)
    assert not bad.any(), float(((z - lse).abs() / ztol)[torch.isfinite(lse)].max())


def tree_masks(rows, words, gen, shape="random"):
    """int64 [sum rows, words]: each drafted token sees itself and the line it hangs from."""
    out = []
    for t in rows:
        m = torch.zeros((t, t), dtype=torch.bool)
        for j in range(t):
            up = int(torch.randint(-1, j, (1,), generator=gen)) if j else -1
            if up >= 0:
                m[j] = m[up]
            m[j, j] = True
        bits = torch.zeros((t, words), dtype=torch.int64)
        for w in range(words):
            for i in range(64):
                if w * 64 + i < t:
                    v = m[:, w * 64 + i].long()
                    bits[:, w] |= torch.where(v.bool(), torch.tensor(-(1 << 63) if i == 63 else 1 << i), 0)
        out.append(bits)
    return torch.cat(out) if out else torch.zeros((0, words), dtype=torch.int64)
