"""Float64 restatements of the operators on paged latents, beams and cache moves (CPU), from their definitions, row by row."""

from __future__ import annotations

import random

import torch


def page_key(pages, table, slot, j):
    """The latent of key j, or None."""
    if not 0 <= slot < table.size(0) or j // pages.size(1) >= table.size(1):
        return None
    page = int(table[slot, j // pages.size(1)])
    return pages[page, j % pages.size(1)] if 0 <= page < pages.size(0) else None


def attn(qa, pages, table, cu, kv_len, slots, scale, max_new):
    """(out, mass, size, written): out float64 [rows, heads, rank]; mass the sum of p |c|; size the greatest sum of |q c| scale of a
    (row, head); written: the rows that the operator writes."""
    rows, heads, rank = qa.shape
    out = torch.zeros(rows, heads, rank, dtype=torch.float64)
    mass, size, written = torch.zeros_like(out), torch.zeros(rows, heads, dtype=torch.float64), torch.zeros(rows, dtype=torch.bool)
    for s in range(len(kv_len)):
        first, n = int(cu[s]), int(cu[s + 1]) - int(cu[s])
        slot = s if slots is None else int(slots[s])
        total = int(kv_len[s])
        found = [(j, page_key(pages, table, slot, j)) for j in range(max(0, min(total, table.size(1) * pages.size(1))))]
        at = torch.tensor([j for j, c in found if c is not None], dtype=torch.long)
        keys = torch.stack([c for _, c in found if c is not None]).double() if len(at) else torch.zeros(0, rank, dtype=torch.float64)
        for i in range(min(n, max_new)):
            r, seen = first + i, keys[at <= total - n + i]
            written[r] = True
            if not len(seen):
                continue
            q = qa[r].double()
            p = torch.softmax(q @ seen.T * scale, -1)
            out[r], mass[r] = p @ seen, p @ seen.abs()
            size[r] = (q.abs() @ seen.abs().T * scale).max(-1).values
    return out, mass, size, written


class Paged:
    """Sequences in pages: a pool whose unused places hold NaN, a table in no order.  ``news[s]`` new tokens of ``lens[s]`` in all."""

    def __init__(self, news, lens, *, page=16, heads=16, rank=128, dtype=torch.bfloat16, seed=0, behind=0, q_std=1.5, spare=1):
        rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
        self.news, self.lens, self.page = list(news), list(lens), page
        self.cu = torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], dtype=torch.int32)
        self.kv_len = torch.tensor(lens, dtype=torch.int64)
        self.rows = sum(news) + behind
        width = max([-(-max(n, 0) // page) for n in lens] + [1]) + spare
        slots = list(range(len(news) + 2))
        rng.shuffle(slots)
        self.slots = torch.tensor(slots[:len(news)], dtype=torch.int32)
        ids = list(range(sum(-(-max(n, 0) // page) for n in lens) + 3))
        rng.shuffle(ids)
        self.table = torch.full((len(slots), width), -1, dtype=torch.int32)
        self.pages = torch.full((len(ids), page, rank), float("nan"), dtype=dtype)
        for s, n in enumerate(lens):
            for j in range(-(-max(n, 0) // page)):
                p = ids.pop()
                self.table[slots[s], j] = p
                k = min(page, n - j * page)
                self.pages[p, :k] = torch.randn(k, rank, generator=gen).to(dtype)
        self.qa = (torch.randn(self.rows, heads, rank, generator=gen) * q_std).to(dtype)
        self.gen = gen

    def place(self, s, j):
        return int(self.table[int(self.slots[s]), j // self.page]), j % self.page


def norms(q, kv, q_w, q_eps, kv_w, kv_eps):
    """Both normalised rows in float64; the weights rounded to the rows' type."""
    out = []
    for x, w, eps in ((q, q_w, q_eps), (kv, kv_w, kv_eps)):
        y = x.double()
        out.append(y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.to(x.dtype).double())
    return out


def beam(logits, scores, beams, keep, ended=None, pad=0):
    """(score float64, parent, token) [groups, keep] by sorting all candidates."""
    groups = logits.size(0) // beams
    score = torch.full((groups, keep), float("-inf"), dtype=torch.float64)
    parent, token = torch.full((groups, keep), -1), torch.full((groups, keep), -1)
    inf = float("inf")
    for g in range(groups):
        found = []
        for b in range(beams):
            r = g * beams + b
            s = float(scores[r])
            if not abs(s) < inf:
                continue
            if ended is not None and bool(ended[r]):
                found.append((-s, b, pad))
                continue
            x = logits[r].double()
            x = torch.where(torch.isnan(x), -inf, x)
            if float(x.max()) in (inf, -inf):
                continue
            v = s + (x - torch.logsumexp(x, -1))
            order = torch.sort(v, descending=True, stable=True).indices[:keep]
            found += [(-float(v[t]), b, int(t)) for t in order if float(v[t]) > -inf]
        for i, (v, b, t) in enumerate(sorted(found)[:keep]):
            score[g, i], parent[g, i], token[g, i] = -v, b, t
    return score, parent, token


def moves(src, dst, limit):
    """The moves that count: (index, src, dst)."""
    last = {}
    for i, (s, d) in enumerate(zip(src, dst)):
        if 0 <= s < limit and 0 <= d < limit:
            last[d] = (i, s)
    return [(i, s, d) for d, (i, s) in last.items() if s != d]


def moved(t, src, dst):
    new = t.clone()
    for _, s, d in moves(src, dst, t.size(0)):
        new[d] = t[s]
    return new


def fork_latents(t, src, dst, cached):
    new = t.clone()
    for i, s, d in moves(src, dst, t.size(0)):
        n = max(0, min(int(cached[i]), t.size(1)))
        new[d, :n] = t[s, :n]
    return new


def fork_pages(table, pools, src, dst, cached, n_slots):
    page = pools[0].size(1)
    new_table, new = table.clone(), [p.clone() for p in pools]
    for i, s, d in moves(src, dst, n_slots):
        full, rest = max(0, int(cached[i])) // page, max(0, int(cached[i])) % page
        new_table[d, :full] = table[s, :full]
        if rest and full < table.size(1):
            a, b = int(table[s, full]), int(table[d, full])
            if 0 <= a < pools[0].size(0) and 0 <= b < pools[0].size(0):
                for p, q in zip(new, pools):
                    p[b, :rest] = q[a, :rest]
    return new_table, new
