"""How far the KDA tree step and its commit may be off a float64 form, value by value: the roundings of what enters each
value, first order (and 5 % for the rest).

E is the largest relative error of one rounding to fp32, 2^-24.  A hardware e^x, 2^x or 1/x is off by one unit in the last
place, 2 E; the argument of e^x is multiplied by a rounded log2(e) first, so e^x is off by (1.3 |x| + 2) E.  A sum of n terms is
off by n E of the sum of their magnitudes, in any order.
"""

from __future__ import annotations

import torch

E = 2.0 ** -24
FACTORED = 60.0   # |G| up to which pairs are weighted by e^G e^-G; beyond, by e^(G - R) e^(R - G) with |R - G| <= FAR
FAR = 80.0


def _exp(x):
    return (1.3 * x.abs() + 2) * E


def _sigmoid(x, dx):
    """The error of 1 / (1 + e^-x)."""
    s = torch.sigmoid(x)
    return s * (1 - s) * (dx + _exp(x)) + 3 * E * s


def _silu(y, dy):
    z = y * torch.sigmoid(y)
    return z, 1.1 * dy + y.abs() * _sigmoid(y, 0.0) + E * z.abs()


def step(tr, x, conv_w, conv_state, g, beta, state, slots, *, A_log=None, dt_bias=None, scale=None, lower=-5.0, l2norm=True,
         gate=True, beta_sigmoid=True):
    """Float64 values and bounds of the step's outputs, and parts of them: a dict of o, tape, tol_o (before o is rounded to its
    type), tol_tape, ``from_state`` and ``from_nodes`` (o's two terms), and per tree ``commit(s, nodes)``, the state after a path
    and its bound.  Trees whose slot is out of range: zeros."""
    H, D, taps = g.size(1), g.size(2), conv_w.size(1)
    scale = D ** -0.5 if scale is None else scale
    shape = (tr.total, H, D)
    res = {n: torch.zeros(shape, dtype=torch.float64) for n in ("o", "tol_o", "from_state", "from_nodes")}
    res["tape"], res["tol_tape"] = (torch.zeros(tr.total, H, 3, D, dtype=torch.float64) for _ in range(2))
    kept = {}
    w = conv_w.double()
    for s, n in enumerate(tr.lens):
        slot, base = int(slots[s]), tr.offsets[s]
        if n == 0 or not 0 <= slot < state.size(0):
            continue
        rows = slice(base, base + n)
        S = state[slot].double()
        hist = torch.zeros(0, 3 * H * D, dtype=torch.float64) if taps == 1 else conv_state[slot].double().T
        xs = x[rows].double()
        samples = torch.stack([torch.cat([hist, xs[p]])[-taps:] for p in tr.paths[s]])                 # [n, taps, C]
        y, dy = (samples * w.T).sum(1), 4 * E * (samples * w.T).abs().sum(1)
        z, dz = (t.view(n, 3, H, D).permute(1, 2, 0, 3) for t in _silu(y, dy))                          # [3, H, n, D]
        v, dv = z[2], dz[2]

        def normed(z, dz, scale):
            if not l2norm:
                return z * scale, (dz + E * z.abs()) * scale
            size = z.norm(dim=-1, keepdim=True)
            return z / size * scale, (dz + z.abs() * (dz.norm(dim=-1, keepdim=True) / size + 12 * E)) / size * scale
        (q, dq), (k, dk) = normed(z[0], dz[0], scale), normed(z[1], dz[1], 1.0)
        a, da = g[rows].double().transpose(0, 1), torch.zeros(H, n, D, dtype=torch.float64)
        if gate:
            A = A_log.double()[:, None, None]
            at = torch.exp(A) * (a + dt_bias.double().view(H, 1, D))
            a, da = lower * torch.sigmoid(at), abs(lower) * (_sigmoid(at, at.abs() * (_exp(A) + 2 * E)) + E * torch.sigmoid(at))
        b, db = beta[rows].double().T, torch.zeros(H, n, dtype=torch.float64)
        if beta_sigmoid:
            b, db = torch.sigmoid(b), _sigmoid(b, 0.0)
        anc = torch.zeros(n, n, dtype=torch.float64)
        for i, p in enumerate(tr.paths[s]):
            anc[i, p] = 1.0
        G = torch.einsum("ij,hjd->hid", anc, a)
        dG = torch.einsum("ij,hjd->hid", anc, da + 6 * E * a.abs())
        A, B, dA, dB = (torch.zeros(H, n, n, dtype=torch.float64) for _ in range(4))
        for h in range(H):
            Gh = G[h]
            far = float(Gh.abs().max()) > FACTORED * (1 - 1e-5)
            diff = Gh[:, None] - Gh[None]
            pair = torch.exp(diff.masked_fill(anc[:, :, None] == 0, float("-inf")))
            off = (Gh.abs()[:, None] + Gh.abs()[None]) * (6 * E) + torch.einsum("ij,jd->id", anc, da[h])[:, None].expand_as(diff)
            off = off + (2.3 * (diff.abs() + 2 * FAR) * E if far else 1.3 * (Gh.abs()[:, None] + Gh.abs()[None]) * E) + 4 * E
            for left, dleft, out, dout in ((k[h], dk[h], A, dA), (q[h], dq[h], B, dB)):
                out[h] = (left[:, None] * k[h][None] * pair).sum(-1)
                dout[h] = ((dleft[:, None] * k[h].abs()[None] + left.abs()[:, None] * dk[h][None]
                            + (left[:, None] * k[h][None]).abs() * (off + 136 * E)) * pair).sum(-1)
        eye = torch.eye(n, dtype=torch.float64)
        A, dA = A * (1 - eye), dA * (1 - eye)
        eG, rel = torch.exp(G), dG + _exp(G) + E

        def through(left, dleft):
            """(left e^G) S and its error."""
            mass = (left.abs() * eG) @ S.abs()
            return (left * eG) @ S, ((dleft + left.abs() * rel) * eG) @ S.abs() + 132 * E * mass
        (P, dP), (Q, dQ) = through(k, dk), through(q, dq)
        M = eye + b[:, :, None] * A
        X = torch.linalg.inv(M)
        u = X @ (b[:, :, None] * (v - P))
        inner = v - P - A @ u
        r = b[:, :, None] * (v.abs() + P.abs()) + (M - eye).abs() @ u.abs()
        delta = db[:, :, None] * inner.abs() + b[:, :, None] * (dv + dP + dA @ u.abs()) + 3 * E * r + 80 * E * (M - eye).abs() @ u.abs()
        # (the diagonal blocks' inverses, of 16 rows, are formed: 16 E |X| |M| |X| off, and applied)
        du = X.abs() @ (delta + 40 * E * M.abs() @ (X.abs() @ r))
        near = B @ u
        do = dQ + dB @ u.abs() + B.abs() @ du + 66 * E * B.abs() @ u.abs() + 2 * E * (Q + near).abs()
        put = lambda name, t: res[name].__setitem__(rows, t.transpose(0, 1))  # noqa: E731
        put("o", Q + near), put("tol_o", 1.05 * do + 1e-30), put("from_state", Q), put("from_nodes", near)
        res["tape"][rows] = torch.stack([u, k, G], 2).transpose(0, 1)
        res["tol_tape"][rows] = 1.05 * torch.stack([du, dk, dG], 2).transpose(0, 1) + 1e-30
        kept[s] = (S, u, du, k, dk, G, dG, a, da, eG, rel)

    def commit(s, nodes):
        S, u, du, k, dk, G, dG, a, da, eG, rel = kept[s]
        i, m = nodes[-1], list(nodes)
        between = torch.flip(torch.cumsum(torch.flip(da[:, m], [1]), 1), [1])
        diff = G[:, [i]] - G[:, m]
        weight = torch.exp(diff)
        off = between + 7 * E * (G[:, [i]].abs() + G[:, m].abs()) + _exp(diff) + 2 * E
        out = eG[:, i, :, None] * S + (k[:, m] * weight).transpose(1, 2) @ u[:, m]
        mass = (eG[:, i, :, None] * S).abs() + (k[:, m].abs() * weight).transpose(1, 2) @ u[:, m].abs()
        tol = (rel[:, i, :, None] * (eG[:, i, :, None] * S).abs() + ((dk[:, m] + k[:, m].abs() * off) * weight).transpose(1, 2) @ u[:, m].abs()
               + (k[:, m].abs() * weight).transpose(1, 2) @ du[:, m] + (len(m) + 3) * E * mass)
        return out, 1.05 * tol + 1e-30
    res["commit"] = commit
    return res


def step_f32(tr, x, conv_w, conv_state, g, beta, state, slots, *, A_log=None, dt_bias=None, gate=True, lower=-5.0,
             operands=torch.float32, nodes=True):
    """The step's output in fp32 on the CPU, in the kernel's chunk form; ``operands``: the type that what enters the products with
    the state is rounded to; without ``nodes``, the drafted term left out."""
    H, D, taps = g.size(1), g.size(2), conv_w.size(1)
    o = torch.zeros(tr.total, H, D)
    to = lambda t: t.to(operands).float()  # noqa: E731
    for s, n in enumerate(tr.lens):
        slot, rows = int(slots[s]), slice(tr.offsets[s], tr.offsets[s] + n)
        if n == 0 or not 0 <= slot < state.size(0):
            continue
        hist = torch.zeros(0, 3 * H * D) if taps == 1 else conv_state[slot].float().T
        y = (torch.stack([torch.cat([hist, x[rows].float()[p]])[-taps:] for p in tr.paths[s]]) * conv_w.T).sum(1)
        q, k, v = (y * torch.sigmoid(y)).view(n, 3, H, D).permute(1, 2, 0, 3)
        q, k = q / q.norm(dim=-1, keepdim=True) * D ** -0.5, k / k.norm(dim=-1, keepdim=True)
        a = g[rows].float().transpose(0, 1)
        if gate:
            a = lower * torch.sigmoid(torch.exp(A_log)[:, None, None] * (a + dt_bias.view(H, 1, D)))
        b = torch.sigmoid(beta[rows].float()).T
        anc = torch.zeros(n, n)
        for i, p in enumerate(tr.paths[s]):
            anc[i, p] = 1.0
        G = torch.stack([sum(a[:, j] for j in p) for p in tr.paths[s]], 1)
        w = torch.exp((G[:, :, None] - G[:, None]).masked_fill(anc[None, :, :, None] == 0, float("-inf")))
        A, B = ((t[:, :, None] * k[:, None] * w).sum(-1) for t in (k, q))
        S = to(state[slot])
        rhs, u = b[..., None] * (v - to(k * torch.exp(G)) @ S), torch.zeros_like(v)
        for i in range(n):
            u[:, i] = rhs[:, i] - b[:, i, None] * (A[:, i:i + 1, :i] @ u[:, :i])[:, 0]
        out = to(q * torch.exp(G)) @ S + (B @ u if nodes else 0.0)
        o[rows] = out.transpose(0, 1)
    return o
