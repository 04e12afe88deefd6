"""Trees of drafted tokens and float64 restatements of the operators over them, node by node, for the tests."""

from __future__ import annotations

import random

import torch


def parents_of(n: int, kind: str, rng: random.Random) -> list[int]:
    """Parents of one tree: a chain, a wide tree, random ones, long branches, several roots, or entries that the operators read as
    roots (not an earlier node)."""
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "wide":
        return [(i - 1) // 4 if i else -1 for i in range(n)]
    if kind == "forest":
        return [rng.randint(-1, i - 1) if rng.random() < 0.7 else -1 for i in range(n)]
    if kind == "branches":     # one after the other, each from the root down
        return [-1 if i == 0 else 0 if i % 21 == 0 else i - 1 for i in range(n)]
    if kind == "odd":
        return [rng.choice([i, i + 1, 70, -5, 2 ** 31 - 1, -2 ** 31, rng.randint(-1, i - 1)]) for i in range(n)]
    return [rng.randint(max(0, i - 5), i - 1) if i else -1 for i in range(n)]


def paths_of(parents: list[int]) -> list[list[int]]:
    """Of each node: the nodes from its root down to it."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if 0 <= p < i else []) + [i])
    return out


class Trees:
    """Packed trees of ``lens`` nodes with ``behind`` rows of no tree after them."""

    def __init__(self, lens, kind: str, seed: int, behind: int = 0) -> None:
        rng = random.Random(seed)
        self.lens = list(lens)
        self.parents = [parents_of(n, kind, rng) for n in self.lens]
        self.paths = [paths_of(p) for p in self.parents]
        self.offsets = [sum(self.lens[:i]) for i in range(len(self.lens) + 1)]
        self.total = self.offsets[-1]
        self.rows = self.total + behind
        self.max_nodes = max(1, max(self.lens, default=1))
        flat = [p for t in self.parents for p in t] + [-1] * behind
        self.cu = torch.tensor(self.offsets, dtype=torch.int32)
        self.par = torch.tensor(flat, dtype=torch.int32)

    def slots(self, n_slots: int, seed: int) -> torch.Tensor:
        order = list(range(n_slots))
        random.Random(seed).shuffle(order)
        return torch.tensor(order[:len(self.lens)], dtype=torch.int32)

    def nodes(self):
        """(tree, row, nodes of the path as rows, node) of every node."""
        for s, paths in enumerate(self.paths):
            for i, path in enumerate(paths):
                yield s, self.offsets[s] + i, [self.offsets[s] + j for j in path], i


def attention(tr: Trees, qa, latent, cache, slots, cached, scale):
    """(out [rows, H, r], sum of p |key| of the same shape, largest sum of |q key| scale per row and head)."""
    out = torch.zeros(tr.total, *qa.shape[1:], dtype=torch.float64)
    mass, size = torch.zeros_like(out), torch.zeros(tr.total, qa.size(1), dtype=torch.float64)
    for s, row, path, _ in tr.nodes():
        slot, n = int(slots[s]), min(max(int(cached[s]), 0), cache.size(1))
        if not 0 <= slot < cache.size(0):
            continue
        keys = torch.cat([cache[slot, :n].double(), latent[path].double()])
        q = qa[row].double()
        p = torch.softmax(q @ keys.T * scale, -1)
        out[row], mass[row] = p @ keys, p @ keys.abs()
        size[row] = (q.abs() @ keys.abs().T * abs(scale)).amax(-1)
    return out, mass, size


def kda_step(tr: Trees, x, conv_w, conv_state, g, beta, state, slots, *, A_log=None, dt_bias=None, scale=None, lower=-5.0,
             l2norm=True, gate=True, beta_sigmoid=True):
    """(o [rows, H, 128], tape [rows, H, 3, 128], the states after every node {row: [H, 128, 128]})."""
    H, D, taps = g.size(1), g.size(2), conv_w.size(1)
    scale = D ** -0.5 if scale is None else scale
    o, tape, states = torch.zeros(tr.total, H, D, dtype=torch.float64), torch.zeros(tr.total, H, 3, D, dtype=torch.float64), {}
    w = conv_w.double()
    for s, row, path, i in tr.nodes():
        slot = int(slots[s])
        if not 0 <= slot < state.size(0):
            continue
        hist = torch.zeros(0, 3 * H * D, dtype=torch.float64) if taps == 1 else conv_state[slot].double().T
        z = (torch.cat([hist, x[path].double()])[-taps:] * w.T).sum(0)
        q, k, v = (z * torch.sigmoid(z)).view(3, H, D)
        if l2norm:
            q = q / q.norm(dim=-1, keepdim=True).clamp(min=1e-12)
            k = k / k.norm(dim=-1, keepdim=True).clamp(min=1e-12)
        q = q * scale
        a = g[row].double()
        if gate:
            a = lower * torch.sigmoid(torch.exp(A_log.double())[:, None] * (a + dt_bias.double().view(H, D)))
        b = beta[row].double()
        if beta_sigmoid:
            b = torch.sigmoid(b)
        S0 = states[path[-2]] if len(path) > 1 else state[slot].double()
        S = S0 * torch.exp(a)[..., None]
        u = b[:, None] * (v - (S * k[..., None]).sum(1))
        S = S + k[..., None] * u[:, None]
        states[row] = S
        o[row] = (S * q[..., None]).sum(1)
        tape[row, :, 0], tape[row, :, 1] = u, k
        tape[row, :, 2] = a + (tape[path[-2], :, 2] if len(path) > 1 else 0.0)
    return o, tape, states


def accept(tr: Trees, logits, tokens, max_nodes: int):
    """(path, n_path, next_token, chosen) as lists."""
    clean = torch.where(torch.isnan(logits.double()), float("-inf"), logits.double())
    chosen = [int((r == r.max()).nonzero()[0, 0]) if float(r.max()) > float("-inf") else 0 for r in clean]
    paths, counts, following = [], [], []
    for s, parents in enumerate(tr.parents):
        base, path = tr.offsets[s], [0] if parents else []
        while path:
            nxt = [i for i, p in enumerate(parents)
                   if 0 <= p < i and p == path[-1] and int(tokens[base + i]) == chosen[base + path[-1]]]
            if not nxt:
                break
            path.append(nxt[0])
        paths.append(path + [-1] * (max_nodes - len(path)))
        counts.append(len(path))
        following.append(chosen[base + path[-1]] if path else -1)
    return paths, counts, following, chosen


def adjust(rows, logits, *, vocab, history=None, history_len=None, prompt_len=None, repetition=None, presence=None,
           frequency=None, bias_ids=None, bias=None, allowed=None, allowed_rows=None, tokens=None):
    """(adjusted logits, sum of the magnitudes that entered each) in float64; ``rows``: (sequence, path rows) of each row."""
    out, size = [], []
    for r, (s, path) in enumerate(rows):
        x = logits[r].double()
        seen, count = torch.zeros(vocab, dtype=torch.bool), torch.zeros(vocab, dtype=torch.float64)
        if history is not None:
            for at, tok in enumerate(history[s, :max(0, int(history_len[s]))].tolist()):
                if 0 <= tok < vocab:
                    seen[tok] = True
                    count[tok] += at >= (0 if prompt_len is None else int(prompt_len[s]))
        if tokens is not None:
            for tok in tokens[path].tolist():
                if 0 <= tok < vocab:
                    seen[tok] = True
                    count[tok] += 1
        rep, pres, freq = ((d if t is None else float(t[s])) for t, d in ((repetition, 1.0), (presence, 0.0), (frequency, 0.0)))
        y = torch.where(seen, torch.where(x > 0, x / rep, x * rep) - freq * count - pres * (count > 0), x)
        m = torch.where(seen, torch.where(x > 0, x / rep, x * rep).abs() + abs(freq) * count + abs(pres), x.abs())
        if bias_ids is not None:
            for tok, b in zip(bias_ids[s].tolist(), bias[s].tolist()):
                if 0 <= tok < vocab:
                    y[tok] += b
                    m[tok] += abs(b)
        if allowed is not None:
            at = r if allowed_rows is None else int(allowed_rows[r])
            if 0 <= at < allowed.size(0):
                bits = ((allowed[at][:, None] >> torch.arange(32)) & 1).reshape(-1)[:vocab]
                y[bits == 0] = float("-inf")
        out.append(y)
        size.append(m)
    return torch.stack(out), torch.stack(size)
