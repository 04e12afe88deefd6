"""The drafted-token operators against float64 restatements (tests/tree_ref.py).

Tolerances count roundings.  One rounding of a value to bf16 is off by at most 2^-8 of it, to fp32 by 2^-24; a sum of n
products in fp32 by n 2^-24 of the sum of their magnitudes.
"""

from __future__ import annotations

import pytest
import torch

import tree_ref as ref

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
E32 = 2.0 ** -24


def _dev(*ts):
    return [None if t is None else t.cuda() for t in ts]


def _within(got, want, tol):
    assert got.shape == want.shape
    err = (got.double().cpu() - want).abs()
    assert torch.isfinite(got.float()).all()
    bad = err > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, worst {float((err / tol).max()):.2f} x the tolerance"


# ------------------------------------------------------------------ attention
def _attn_case(lens, cached, *, kind="mixed", dtype=BF, heads=16, rank=128, max_seq=600, seed=0, behind=0, q_std=1.5):
    tr = ref.Trees(lens, kind, seed, behind)
    gen = torch.Generator().manual_seed(seed)
    n_slots = len(lens) + 2
    cache = torch.randn(n_slots, max_seq, rank, generator=gen).to(dtype).float()
    latent = torch.randn(tr.rows, rank, generator=gen).to(dtype)
    qa = (torch.randn(tr.rows, heads, rank, generator=gen) * q_std).to(dtype)
    slots = tr.slots(n_slots, seed)
    cached = torch.tensor(cached, dtype=torch.int64)
    for s, slot in enumerate(slots.tolist()):   # what lies behind the cached keys is never read
        cache[slot, min(max(int(cached[s]), 0), max_seq):] = float("nan")
    return tr, qa, latent, cache, slots, cached


def _attn_tol(tr, want, mass, size, dtype, rank):
    # scores: `rank` products (and the scale) in fp32, two of them in each probability (with the maximum); exponentials
    # to 2^-22; the sums over keys in fp32
    p = (2 * (rank + 4) * E32 * size + 2.0 ** -21)[..., None] * 2 * mass + 700 * E32 * mass
    if dtype == F32:
        return p + E32 * want.abs() + 1e-30
    return p + 2.0 ** -8 * mass + 2.0 ** -8 * want.abs() + 1e-30   # probabilities and the result to bf16


ATTN = [
    dict(lens=[1], cached=[0]),
    dict(lens=[1], cached=[1]),
    dict(lens=[2, 7], cached=[63, 64]),
    dict(lens=[64, 64], cached=[65, 0], kind="chain"),
    dict(lens=[9, 0, 16, 17], cached=[128, 50, 599, 600], kind="forest"),
    dict(lens=[33, 5, 64], cached=[-3, 10 ** 12, 200], kind="odd"),
    dict(lens=[8, 24, 63], cached=[300, 1, 577], kind="wide", heads=3, behind=5),
    dict(lens=[5, 31], cached=[90, 191], rank=32),
    dict(lens=[5, 31], cached=[90, 191], rank=64, heads=1),
    dict(lens=[5, 31], cached=[90, 191], rank=256, heads=16),
]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("splits", [None, 1, 3, 40])
@pytest.mark.parametrize("case", range(len(ATTN)))
def test_tree_attention_matches_reference(case, splits, dtype):
    from sophia_amd import ops
    tr, qa, latent, cache, slots, cached = _attn_case(**ATTN[case], dtype=dtype, seed=case)
    rank, scale = qa.size(2), 128 ** -0.5
    out = torch.full((tr.rows, qa.size(1), rank), 7.0, dtype=dtype, device="cuda")
    got = ops.mla_tree_attn(*_dev(qa, latent, cache, tr.cu, tr.par, slots, cached), scale, max_nodes=tr.max_nodes,
                            max_len=None if case % 2 else 600, splits=splits, out=out)
    assert got is out
    want, mass, size = ref.attention(tr, qa, latent, cache, slots, cached, scale)
    _within(got[:tr.total], want, _attn_tol(tr, want, mass, size, dtype, rank))
    assert (got[tr.total:] == 7.0).all()   # rows of no tree


def test_tree_attention_of_single_nodes_is_decode_attention():
    from sophia_amd import ops
    tr, qa, latent, cache, slots, cached = _attn_case([1] * 9, [0, 1, 15, 16, 63, 64, 100, 500, 599])
    got = ops.mla_tree_attn(*_dev(qa, latent, cache, tr.cu, tr.par, slots, cached), 0.09, max_nodes=1)
    for s, slot in enumerate(slots.tolist()):
        cache[slot, int(cached[s])] = latent[s].float()
    old = ops.mla_decode_attn(*_dev(qa, cache, slots, cached), 0.09)
    # both round the probabilities to bf16 and then the result
    want, mass, _ = ref.attention(tr, qa, latent, cache, slots, cached, 0.09)
    _within(got, old.double().cpu(), 2 * (2.0 ** -8 * mass + 2.0 ** -8 * want.abs()) + 1e-3 * mass)


def test_tree_attention_strides_slots_and_outliers():
    """Strided rows, an out-of-range slot, scores far apart and large, a key that takes everything."""
    from sophia_amd import ops
    tr, qa, latent, cache, slots, cached = _attn_case([12, 3, 20], [77, 40, 130], q_std=30.0, seed=4)
    slots[1] = 99
    wide_q = torch.zeros(tr.rows, 16 * 128 + 64, dtype=BF)
    wide_q[:, :2048] = qa.reshape(tr.rows, 2048)
    wide_l = torch.zeros(tr.rows, 136, dtype=BF)
    wide_l[:, :128] = latent
    roomy = torch.full((cache.size(0), cache.size(1) + 16, 128), float("nan"))
    roomy[:, :600] = cache
    dq, dl, dc = _dev(wide_q, wide_l, roomy)
    out = torch.zeros(tr.rows, 2056, dtype=BF, device="cuda")
    ops.mla_tree_attn(dq[:, :2048].unflatten(1, (16, 128)), dl[:, :128], dc[:, :600],
                      *_dev(tr.cu, tr.par, slots, cached), 128 ** -0.5, max_nodes=32,
                      out=out[:, :2048].unflatten(1, (16, 128)))
    want, mass, size = ref.attention(tr, qa, latent, cache, slots, cached, 128 ** -0.5)
    _within(out[:, :2048].reshape(tr.rows, 16, 128), want, _attn_tol(tr, want, mass, size, BF, 128))
    assert (out[12:15] == 0).all() and (out[:, 2048:] == 0).all()


def test_tree_attention_nan_stays_on_its_paths():
    """A drafted latent that is not finite reaches its own node and the nodes below it, no others."""
    from sophia_amd import ops
    tr, qa, latent, cache, slots, cached = _attn_case([40, 11], [100, 0], kind="wide", seed=7)
    clean = latent.clone()
    latent[3, 5], latent[9, 100], latent[44, 0] = float("nan"), float("inf"), float("-inf")
    for dtype in (BF, F32):
        got = ops.mla_tree_attn(*_dev(qa.to(dtype), latent.to(dtype), cache, tr.cu, tr.par, slots, cached), 0.08, max_nodes=40)
        want, mass, size = ref.attention(tr, qa, clean, cache, slots, cached, 0.08)
        tol = _attn_tol(tr, want, mass, size, dtype, 128)
        for _, row, path, _ in tr.nodes():
            if {3, 9, 44} & set(path):
                assert torch.isnan(got[row]).any(-1).all(), row
            else:
                _within(got[row], want[row], tol[row])


# ------------------------------------------------------------------ KDA step
def _step_case(lens, *, kind="mixed", dtype=BF, heads=2, taps=4, gate=True, seed=0, behind=0, g_dtype=None, strong=False):
    tr = ref.Trees(lens, kind, seed, behind)
    gen = torch.Generator().manual_seed(seed + 100)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    inner, n_slots = heads * 128, len(lens) + 2
    c = dict(x=rn(tr.rows, 3 * inner).to(dtype), conv_w=(rn(3 * inner, taps) * 0.5).to(dtype).float(),
             conv_state=rn(n_slots, 3 * inner, taps - 1).to(dtype).float() if taps > 1 else None,
             g=rn(tr.rows, heads, 128), beta=rn(tr.rows, heads).to(dtype), state=rn(n_slots, heads, 128, 128) * 0.2,
             slots=tr.slots(n_slots, seed), A_log=rn(heads) * 0.3, dt_bias=rn(inner) - (0.0 if strong else 2.0))
    if strong:
        c["g"] = c["g"] * 2 + 3     # decays near the lower bound: e^-5 a step
    c["g"] = c["g"].to(g_dtype or dtype)
    if not gate:
        c["g"] = -torch.nn.functional.softplus(c["g"].float() - 1.0)
    return tr, c


def _run_step(tr, c, *, gate=True, out=None, max_nodes=None, **kw):
    from sophia_amd import ops
    d = {k: (None if v is None else v.cuda()) for k, v in c.items()}
    return ops.kda_tree_step(d["x"], d["conv_w"], d["conv_state"], d["g"], d["beta"], d["state"], *_dev(tr.cu, tr.par),
                             max_nodes=max_nodes or tr.max_nodes, A_log=d["A_log"], dt_bias=d["dt_bias"], use_gate=gate,
                             state_slots=d["slots"], out=out, **kw)


def _step_tol(tr, o, tape, dtype):
    """u and o: sums over 128 channels and the path's nodes in fp32, each node's u entering those below it: a path of n
    nodes is off by (128 + n) n 2^-24 of the largest magnitude at most, with the exponentials (an argument |G| is off by
    |G| 2^-23) on top; G is a sum of n log-decays, each off by 2^-22 of its bound 5."""
    n = torch.zeros(tr.total, 1, 1, dtype=torch.float64)
    for _, row, path, _ in tr.nodes():
        n[row] = len(path)
    gmax = tape[:, :, 2].abs().amax(-1, keepdim=True) if tr.total else torch.zeros(0)
    rel = ((128 + n) * n + 2 * gmax + 16) * E32
    big_u = tape[:, :, 0].abs().amax().clamp(min=1.0) if tr.total else 1.0
    tol_u = rel * 4 * big_u
    tol_o = rel * 4 * torch.maximum(o.abs().amax(), big_u) + (2.0 ** -8 * o.abs() if dtype == BF else 0.0)
    tol = torch.stack([tol_u.expand_as(o), torch.full_like(o, 140 * E32), (n * 5 * 2.0 ** -22).expand_as(o)], 2)
    return tol_o, tol


STEP = [
    dict(lens=[1]),
    dict(lens=[2, 0, 16, 7], kind="forest"),
    dict(lens=[17, 32, 1], kind="wide"),
    dict(lens=[33, 64], kind="chain"),
    dict(lens=[64, 3, 50], kind="odd", behind=4),
    dict(lens=[16, 9], taps=1, heads=1),
    dict(lens=[20, 5], taps=2, heads=3),
    dict(lens=[48], taps=3, gate=False),
    dict(lens=[15, 8], kind="chain", gate=False, g_dtype=F32),
    dict(lens=[64, 30, 16], kind="chain", strong=True),
    dict(lens=[64, 41, 26], kind="branches", strong=True),
    dict(lens=[64, 20, 15], strong=True, g_dtype=F32),
    dict(lens=[64, 50], kind="branches", gate=False, g_dtype=F32),
    dict(lens=[31, 64], kind="odd", strong=True, taps=1),
    dict(lens=[13], g_dtype=F32, heads=16),
]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(STEP)))
def test_tree_step_matches_reference(case, dtype):
    kw = dict(STEP[case])
    tr, c = _step_case(**kw, dtype=dtype, seed=case)
    gate = kw.get("gate", True)
    out = torch.full((tr.rows, c["g"].size(1), 128), 3.0, dtype=dtype, device="cuda")
    tape = torch.full((tr.rows, c["g"].size(1), 3, 128), 5.0, device="cuda")
    got, tape2 = _run_step(tr, c, gate=gate, out=out, tape=tape)
    assert got is out and tape2 is tape
    o, want, _ = ref.kda_step(tr, **{k: v for k, v in c.items()}, gate=gate)
    tol_o, tol = _step_tol(tr, o, want, dtype)
    _within(tape[:tr.total], want, tol)
    _within(got[:tr.total], o, tol_o)
    assert (out[tr.total:] == 3.0).all() and (tape[tr.total:] == 5.0).all()


@pytest.mark.parametrize("flags", [dict(use_qk_l2norm=False, use_beta_sigmoid=False, scale=0.5), dict(lower_bound=-1.0)])
def test_tree_step_switches(flags):
    tr, c = _step_case([24, 6], dtype=F32, seed=20)
    if "scale" in flags:
        c["x"], c["beta"] = c["x"] * 0.3, torch.sigmoid(c["beta"])   # without the norm k is small enough to contract
        c["conv_w"] = c["conv_w"] * 0.3
    got, tape = _run_step(tr, c, **flags)
    o, want, _ = ref.kda_step(tr, **c, l2norm=flags.get("use_qk_l2norm", True), lower=flags.get("lower_bound", -5.0),
                              beta_sigmoid=flags.get("use_beta_sigmoid", True), scale=flags.get("scale"))
    tol_o, tol = _step_tol(tr, o, want, F32)
    _within(tape, want, tol)
    _within(got, o, tol_o)


def test_tree_step_larger_bound_strides_and_bad_slots():
    """A bound above the trees' sizes (another variant) agrees to the roundings; strided rows; a slot out of range."""
    tr, c = _step_case([10, 4, 12], seed=31, heads=2)
    c["slots"][1] = -1
    rows = torch.zeros(tr.rows, 1024, dtype=BF)
    rows[:, :768] = c["x"]
    x = rows.cuda()[:, :768]
    o, want, _ = ref.kda_step(tr, **c)
    tol_o, tol = _step_tol(tr, o, want, BF)
    for bound in (12, 32, 64):
        got, tape = _run_step(tr, dict(c, x=x), max_nodes=bound)
        _within(tape, want, tol)
        _within(got, o, tol_o)
        assert (got[10:14] == 0).all() and (tape[10:14] == 0).all()


def test_tree_step_of_a_chain_is_the_decode_steps():
    """A chain through the tree step and the same tokens through the decode step, whose conv outputs are rounded to the
    activation type: fp32 here, so that nothing is."""
    from sophia_amd import ops
    tr, c = _step_case([20], kind="chain", dtype=F32, seed=8, heads=4)
    got, tape = _run_step(tr, c)
    slot = c["slots"].cuda()
    state, hist = c["state"].cuda(), c["conv_state"].cuda()
    x, g, beta, w = _dev(c["x"], c["g"], c["beta"], c["conv_w"])
    outs = [ops.kda_decode_conv_step(x[i:i + 1], w, hist, g[i:i + 1], beta[i:i + 1], state, A_log=c["A_log"].cuda(),
                                     dt_bias=c["dt_bias"].cuda(), state_slots=slot) for i in range(20)]
    o, want, _ = ref.kda_step(tr, **c)
    tol_o, _ = _step_tol(tr, o, want, F32)
    _within(got, torch.cat(outs).double().cpu(), 2 * tol_o)
    # and its commit is the state and history that they leave
    state2, hist2 = c["state"].cuda(), c["conv_state"].cuda()
    path = torch.arange(20, dtype=torch.int32, device="cuda")[None]
    ops.tree_commit(path, torch.tensor([20], dtype=torch.int32, device="cuda"), tr.cu.cuda(), slot,
                    kda=[(tape, x, hist2, state2)])
    assert torch.equal(hist, hist2)
    _within(state2, state.double().cpu(), torch.full_like(state2, 2 * float(tol_o.max())).double().cpu())


@pytest.mark.parametrize("low", [float("-inf"), torch.finfo(torch.float32).min, -1e5])
def test_tree_step_log_decays_that_forget_the_state(low):
    """Log-decays whose exponential is 0 in fp32 count as -104, the last whole number of that kind (e^-104 = 7e-46): what
    follows a forgotten state keeps its own decays, and so does a commit."""
    from sophia_amd import ops
    tr, c = _step_case([18, 40, 5], kind="wide", dtype=F32, gate=False, seed=17)
    gen = torch.Generator().manual_seed(3)
    hit = torch.rand(c["g"].shape, generator=gen) < 0.1
    hit[tr.offsets[1] + 1] = True      # a whole row, near the root
    o, want, states = ref.kda_step(tr, **{**c, "g": torch.where(hit, -104.0, c["g"])}, gate=False)
    c["g"] = torch.where(hit, low, c["g"])
    got, tape = _run_step(tr, c, gate=False)
    tol_o, tol = _step_tol(tr, o, want, F32)
    n = torch.zeros(tr.total, 1, 1, dtype=torch.float64)
    for _, row, path, _ in tr.nodes():
        n[row] = len(path)
    tol[:, :, 2] = n * want[:, :, 2].abs() * E32     # (sums beyond the bound of 5 that _step_tol counts)
    _within(tape, want, tol)
    _within(got, o, tol_o)
    last = [tr.paths[s][-1] for s in range(3)]
    path = torch.full((3, max(map(len, last))), -1, dtype=torch.int32)
    for s, nodes in enumerate(last):
        path[s, :len(nodes)] = torch.tensor(nodes, dtype=torch.int32)
    state = c["state"].cuda()
    ops.tree_commit(path.cuda(), torch.tensor([len(p) for p in last], dtype=torch.int32, device="cuda"), tr.cu.cuda(),
                    c["slots"].cuda(), kda=[(tape, c["x"].cuda(), c["conv_state"].cuda(), state)])
    for s in range(3):
        row = tr.offsets[s] + last[s][-1]
        full = torch.full_like(states[row], float(tol[row, :, 0].max()) * 4)
        _within(state[int(c["slots"][s])], states[row], full)


def test_tree_step_nan_stays_on_its_paths():
    tr, c = _step_case([40, 12], kind="wide", dtype=F32, seed=9)
    o, want, _ = ref.kda_step(tr, **c)
    tol_o, tol = _step_tol(tr, o, want, F32)
    inner = c["g"].size(1) * 128
    c["x"][3, 7] = float("nan")              # q of head 0 (and, by the conv, of the nodes below)
    c["x"][6, inner + 200] = float("inf")    # k of head 1
    c["x"][45, 2 * inner + 5] = float("nan")   # v of head 0
    c["beta"][42, 1] = float("nan")
    got, tape = _run_step(tr, c)
    for _, row, path, _ in tr.nodes():
        if not {3, 6, 45, 42} & set(path):
            _within(got[row], o[row], tol_o[row])
            _within(tape[row], want[row], tol[row])
    for _, row, path, _ in tr.nodes():
        if 45 in path:     # the node's value is in the state of those below it
            assert not torch.isfinite(tape[row, 0, 0]).all()
        if 42 in path:
            assert not torch.isfinite(got[row, 1]).all()


# ------------------------------------------------------------------ commit
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("taps,heads,layers", [(4, 2, 1), (1, 1, 2), (2, 3, 1), (3, 1, 50)])
def test_commit_writes_the_paths(taps, heads, layers, dtype):
    from sophia_amd import ops
    cases = [_step_case([12, 5, 64, 1, 20, 3], kind="mixed", dtype=dtype, taps=taps, heads=heads, seed=3) for _ in range(layers)]
    tr, c0 = cases[0]
    slots, n_slots = c0["slots"].clone(), c0["state"].size(0)
    slots[4] = n_slots          # out of range: left out
    paths = [tr.paths[0][11], tr.paths[1][0], tr.paths[2][63], [], tr.paths[4][5], tr.paths[5][2][:1] + [9, 1]]
    count = [len(p) for p in paths]
    paths[1], count[1] = paths[1] + [2, 3], 1       # entries past the count
    width = max(len(p) for p in paths) + 1
    path = torch.tensor([p + [-1] * (width - len(p)) for p in paths], dtype=torch.int32)
    taken = [paths[0], paths[1][:1], paths[2], [], [], paths[5][:1]]   # the last ends at the index 9 of 3 nodes
    gen = torch.Generator().manual_seed(1)
    kda, states = [], None
    for _, c in cases:
        tape = torch.empty(tr.rows, heads, 3, 128)
        tape[:, :, 0] = torch.randn(tr.rows, heads, 128, generator=gen)
        tape[:, :, 1] = torch.nn.functional.normalize(torch.randn(tr.rows, heads, 128, generator=gen), dim=-1)
        tape[:, :, 2] = -torch.rand(tr.rows, heads, 128, generator=gen)
        for s, p in enumerate(tr.paths):
            for i, q in enumerate(p):
                if len(q) > 1:
                    tape[tr.offsets[s] + i, :, 2] += tape[tr.offsets[s] + q[-2], :, 2]
        kda.append(_dev(tape, c["x"], c["conv_state"], c["state"]))
    caches = [(torch.randn(tr.rows, 32, generator=gen).to(dtype), torch.randn(n_slots, 40, 32, generator=gen)) for _ in range(2)]
    mla = [tuple(_dev(*m)) for m in caches]
    cached = torch.tensor([39, 0, 5, 7, 8, -1], dtype=torch.int64)
    ops.tree_commit(*_dev(path, torch.tensor(count, dtype=torch.int32), tr.cu, slots), kda=kda, mla=mla, cached=cached.cuda())
    for (_, c), (tape, x, hist, state) in zip(cases, kda):
        want, want_hist, tol = c["state"].double(), None if taps == 1 else c["conv_state"].clone(), torch.zeros_like(c["state"].double())
        for s, p in enumerate(taken):
            if not p:
                continue
            rows = [tr.offsets[s] + i for i in p]
            t, slot = tape.cpu().double()[rows], int(slots[s])
            end = t[-1, :, 2]
            w = t[:, :, 1] * torch.exp(end - t[:, :, 2])
            keep = torch.exp(end)[..., None] * want[slot]
            mass = keep.abs() + torch.einsum("nhk,nhv->hkv", w.abs(), t[:, :, 0].abs())
            # exponentials off by their argument's rounding and 2^-22, one product and sum per node
            tol[slot] = (len(p) + 8 + 2 * float(t[:, :, 2].abs().max())) * 2.0 ** -23 * mass + 1e-30
            want[slot] = keep + torch.einsum("nhk,nhv->hkv", w, t[:, :, 0])
            if want_hist is not None:
                want_hist[slot] = torch.cat([want_hist[slot], c["x"][rows].float().T], 1)[:, len(p):]
        _within(state, want, tol)
        if want_hist is not None:
            assert torch.equal(hist.cpu(), want_hist)
    for (latent, cache), (_, got) in zip(caches, mla):
        want = cache.clone()
        for s, p in enumerate(taken):
            for t, i in enumerate(p):
                if 0 <= int(cached[s]) + t < 40:
                    want[int(slots[s]), int(cached[s]) + t] = latent[tr.offsets[s] + i].float()
        assert torch.equal(got.cpu(), want)


# ------------------------------------------------------------------ logits
def _adjust_case(rows_of, vocab, *, dtype, n, rows, seed, history=60, n_bias=7, masks=3, tokens=None):
    gen = torch.Generator().manual_seed(seed)
    ri = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=gen)  # noqa: E731
    x = (torch.randn(rows, vocab, generator=gen) * 3).to(dtype)
    args = dict(history=ri(-2, min(vocab, 90) + 2, n, history), history_len=ri(-1, history + 3, n).int(),
                prompt_len=ri(0, history, n).int(), repetition=torch.rand(n, generator=gen) + 0.6,
                presence=torch.rand(n, generator=gen) - 0.3, frequency=torch.rand(n, generator=gen) * 0.5,
                bias_ids=ri(-1, min(vocab, 40) + 1, n, n_bias), bias=torch.randn(n, n_bias, generator=gen),
                allowed=ri(-2 ** 31, 2 ** 31, masks, -(-vocab // 32)).int(), allowed_rows=ri(-1, masks + 1, rows).int())
    args["allowed"][0] = 0     # nothing allowed
    return x, args


def _check_adjust(got, x, rows_of, vocab, args, tokens=None):
    a = dict(args)
    if a.get("history_len") is not None:
        a["history_len"] = a["history_len"].clamp(0, a["history"].size(1))
    want, size = ref.adjust(rows_of, x, vocab=vocab, tokens=tokens, **a)
    got = got.double().cpu()
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    fin = torch.isfinite(want)
    # a reciprocal and a product, two subtractions, the biases' sum
    tol = 16 * E32 * size + 1e-30 + (2.0 ** -8 * want.abs() if x.dtype == BF else 0.0)
    err = (got - want)[fin].abs()
    assert (err <= tol[fin]).all(), float((err / tol[fin]).max())


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 31), (5, 2048), (2, 2049), (4, 5000), (7, 4104), (1, 65536)])
def test_adjust_rows_matches_reference(rows, vocab, dtype):
    from sophia_amd import ops
    x, args = _adjust_case(None, vocab, dtype=dtype, n=rows, rows=rows, seed=vocab + rows)
    rows_of = [(r, None) for r in range(rows)]
    dev = {k: v.cuda() for k, v in args.items()}
    got = ops.adjust_logits(x.cuda(), **dev)
    _check_adjust(got, x, rows_of, vocab, args)
    inplace = x.cuda()
    assert ops.adjust_logits(inplace, **dev, out=inplace) is inplace and torch.equal(inplace, got)
    wide = torch.zeros(rows, vocab + 3, dtype=dtype, device="cuda")   # rows off every boundary
    wide[:, 1:vocab + 1] = x.cuda()
    y = ops.adjust_logits(wide[:, 1:vocab + 1], **dev, out=wide[:, 1:vocab + 1])
    assert torch.equal(y, got) and (wide[:, 0] == 0).all() and (wide[:, vocab + 1:] == 0).all()


@pytest.mark.parametrize("drop", ["history", "prompt_len", "repetition", "presence", "frequency", "bias", "allowed",
                                  "allowed_rows", "everything"])
def test_adjust_parts_are_optional(drop):
    from sophia_amd import ops
    x, args = _adjust_case(None, 700, dtype=F32, n=3, rows=3, seed=2)
    gone = {"history": ("history", "history_len", "prompt_len"), "bias": ("bias", "bias_ids"),
            "allowed": ("allowed", "allowed_rows"), "everything": tuple(args)}.get(drop, (drop,))
    args = {k: v for k, v in args.items() if k not in gone}
    got = ops.adjust_logits(x.cuda(), **{k: v.cuda() for k, v in args.items()})
    if drop == "everything":
        assert torch.equal(got.cpu(), x)
    _check_adjust(got, x, [(r, None) for r in range(3)], 700, args)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("lens,kind,vocab", [([1], "mixed", 300), ([16, 0, 5], "wide", 2500), ([64, 33], "chain", 777),
                                             ([9, 64, 2], "odd", 6000)])
def test_adjust_trees_matches_reference(lens, kind, vocab, dtype):
    from sophia_amd import ops
    tr = ref.Trees(lens, kind, 5, behind=2)
    x, args = _adjust_case(None, vocab, dtype=dtype, n=len(lens), rows=tr.rows, seed=vocab)
    tokens = torch.randint(-1, min(vocab, 30), (tr.rows,), generator=torch.Generator().manual_seed(6))
    out = torch.full((tr.rows, vocab), 9.0, dtype=dtype, device="cuda")
    got = ops.adjust_logits(x.cuda(), **{k: v.cuda() for k, v in args.items()}, tokens=tokens.cuda(), cu_nodes=tr.cu.cuda(),
                            parents=tr.par.cuda(), max_nodes=tr.max_nodes, out=out)
    rows_of = [(s, path) for s, _, path, _ in tr.nodes()]
    _check_adjust(got[:tr.total], x[:tr.total], rows_of, vocab, dict(args, allowed_rows=args["allowed_rows"][:tr.total]), tokens)
    assert (got[tr.total:] == 9.0).all()


def test_adjust_infinities_and_nan():
    from sophia_amd import ops
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[inf, -inf, nan, 1.0, -1.0, 0.0, nan, -inf]])
    hist = torch.tensor([[0, 1, 2, 3, 4, 5]])
    got = ops.adjust_logits(x.cuda(), history=hist.cuda(), history_len=torch.tensor([6], dtype=torch.int32, device="cuda"),
                            repetition=torch.tensor([2.0], device="cuda"), frequency=torch.tensor([0.25], device="cuda"),
                            allowed=torch.tensor([[0b10111111]], dtype=torch.int32, device="cuda"))[0].tolist()
    assert got[0] == inf and got[1] == -inf and got[2] != got[2] and got[3] == 0.25 and got[4] == -2.25
    assert got[5] == -0.25 and got[6] == -inf and got[7] == -inf


# ------------------------------------------------------------------ accept
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("lens,kind,vocab", [([1], "mixed", 1), ([7, 0, 64, 16], "mixed", 5), ([33, 12], "chain", 2),
                                             ([64, 1, 9], "odd", 4099), ([20, 30], "wide", 8192), ([5], "forest", 65536)])
def test_accept_matches_reference(lens, kind, vocab, dtype):
    from sophia_amd import ops
    tr = ref.Trees(lens, kind, 3, behind=1)
    gen = torch.Generator().manual_seed(vocab)
    x = torch.randn(tr.rows, vocab, generator=gen).to(dtype)
    x[0] = x[0, 0]                       # all alike: the lowest index
    if vocab > 3 and tr.rows > 3:
        x[1], x[2, :2] = float("-inf"), float("nan")
        x[3, vocab // 2:] = float("inf")
    tokens = torch.randint(0, min(vocab, 3), (tr.rows,), generator=gen)
    _, _, _, chosen = ref.accept(tr, x, tokens, 64)
    for _, row, path, _ in tr.nodes():   # most nodes are what follows their parent
        if len(path) > 1 and torch.rand((), generator=gen) < 0.8:
            tokens[row] = chosen[path[-2]]
    bound = min(64, tr.max_nodes + 3)
    want = ref.accept(tr, x, tokens, bound)
    wide = torch.zeros(tr.rows, vocab + 1, dtype=dtype, device="cuda")
    wide[:, :vocab] = x.cuda()
    for logits in (x.cuda(), wide[:, :vocab]):
        path, n_path, following, said = ops.tree_accept(logits, tokens.cuda(), tr.cu.cuda(), tr.par.cuda(), max_nodes=bound)
        assert (path.tolist(), n_path.tolist(), following.tolist(), said.tolist()) == want
        assert path.dtype == n_path.dtype == torch.int32 and following.dtype == said.dtype == torch.int64


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [4, 13, 2051, 9003])
def test_accept_of_padded_rows_without_a_choice(vocab, dtype):
    """Rows of -inf and NaN alone choose 0, whatever the alignment of the row's last logits; values behind a row are not
    its own."""
    from sophia_amd import ops
    tr = ref.Trees([6], "wide", 0)
    wide = torch.full((6, -(-vocab // 8) * 8), 9.0, dtype=dtype)
    x = wide[:, :vocab]
    x[:] = float("-inf")
    x[1] = float("nan")
    x[2, -1] = float("nan")
    x[3, -1] = -3.0
    x[4, -2:] = 1.0
    x[5, 0] = torch.finfo(dtype).min
    tokens = torch.zeros(6, dtype=torch.int64)
    want = ref.accept(tr, x, tokens, 6)
    assert want[3] == [0, 0, 0, vocab - 1, vocab - 2, 0]
    got = ops.tree_accept(wide.cuda()[:, :vocab], tokens.cuda(), tr.cu.cuda(), tr.par.cuda(), max_nodes=6)
    assert tuple(t.tolist() for t in got) == want


def test_accept_chooses_for_rows_of_no_tree_too():
    from sophia_amd import ops
    x = torch.randn(70, 33, generator=torch.Generator().manual_seed(1)).cuda()
    tokens, par = torch.zeros(70, dtype=torch.int64, device="cuda"), torch.full((70,), -1, dtype=torch.int32, device="cuda")
    for cu in ([0], [0, 3], [5, 5, 5]):
        path, n_path, following, said = ops.tree_accept(x, tokens, torch.tensor(cu, dtype=torch.int32, device="cuda"), par,
                                                        max_nodes=3)
        assert torch.equal(said, x.argmax(-1)) and path.shape == (len(cu) - 1, 3)


def test_no_trees_and_no_rows():
    from sophia_amd import ops
    cu, par = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    none64, none32 = torch.zeros(0, dtype=torch.int64, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    cache = torch.zeros(2, 8, 128, device="cuda")
    assert ops.mla_tree_attn(torch.zeros(0, 4, 128, device="cuda"), torch.zeros(0, 128, device="cuda"), cache, cu, par, none32,
                             none64, 1.0, max_nodes=4).shape == (0, 4, 128)
    path, n_path, nxt, said = ops.tree_accept(torch.zeros(0, 5, device="cuda"), none64, cu, par, max_nodes=4)
    assert path.shape == (0, 4) and n_path.numel() == nxt.numel() == said.numel() == 0
    assert ops.adjust_logits(torch.zeros(0, 5, device="cuda")).shape == (0, 5)
    empty = torch.zeros(3, dtype=torch.int32, device="cuda")     # two trees without nodes
    path, n_path, nxt, _ = ops.tree_accept(torch.zeros(0, 5, device="cuda"), none64, empty, par, max_nodes=2)
    assert path.tolist() == [[-1, -1], [-1, -1]] and n_path.tolist() == [0, 0] and nxt.tolist() == [-1, -1]
    ops.tree_commit(path, n_path, empty, None, mla=[(torch.zeros(0, 128, device="cuda"), cache)],
                    cached=torch.zeros(2, dtype=torch.int64, device="cuda"))


# ------------------------------------------------------------------ refusals
def _refusal_args():
    tr, qa, latent, cache, slots, cached = _attn_case([3, 4], [5, 6])
    attn = dict(qa=qa, latent=latent, latent_cache=cache, cu_nodes=tr.cu, parents=tr.par, slots=slots, cached=cached)
    attn = {k: v.cuda() for k, v in attn.items()} | dict(scale=0.1, max_nodes=4)
    tr, c = _step_case([3, 4])
    step = dict(x_qkv=c["x"], conv_weight=c["conv_w"], conv_state=c["conv_state"], g=c["g"], beta=c["beta"], state=c["state"],
                cu_nodes=tr.cu, parents=tr.par, A_log=c["A_log"], dt_bias=c["dt_bias"], state_slots=c["slots"])
    step = {k: v.cuda() for k, v in step.items()} | dict(max_nodes=4)
    return attn, step


def test_operators_refuse_wrong_shapes_types_and_layouts():
    from sophia_amd import ops
    attn, step = _refusal_args()

    def refused(fn, args, **change):
        with pytest.raises(RuntimeError):
            fn(**{**args, **change})
    a = attn
    refused(ops.mla_tree_attn, a, max_nodes=65)
    refused(ops.mla_tree_attn, a, max_nodes=0)
    refused(ops.mla_tree_attn, a, scale=-1.0)
    refused(ops.mla_tree_attn, a, latent=a["latent"].float())
    refused(ops.mla_tree_attn, a, latent=a["latent"][:-1])
    refused(ops.mla_tree_attn, a, parents=a["parents"][:-1])
    refused(ops.mla_tree_attn, a, parents=a["parents"].long())
    refused(ops.mla_tree_attn, a, cu_nodes=a["cu_nodes"].long())
    refused(ops.mla_tree_attn, a, slots=a["slots"][:-1])
    refused(ops.mla_tree_attn, a, cached=a["cached"].int())
    refused(ops.mla_tree_attn, a, cached=a["cached"].cpu())
    refused(ops.mla_tree_attn, a, qa=a["qa"].half(), latent=a["latent"].half())
    refused(ops.mla_tree_attn, a, qa=a["qa"].transpose(0, 1).contiguous().transpose(0, 1))
    refused(ops.mla_tree_attn, a, latent_cache=a["latent_cache"].bfloat16())
    refused(ops.mla_tree_attn, a, latent_cache=a["latent_cache"][:, :, :64])
    refused(ops.mla_tree_attn, a, slots=None, latent_cache=a["latent_cache"][:1])
    refused(ops.mla_tree_attn, a, out=torch.zeros_like(a["qa"]).float())
    refused(ops.mla_tree_attn, a, out=torch.zeros_like(a["qa"])[:-1])
    refused(ops.mla_tree_attn, a, qa=torch.zeros(7, 17, 128, dtype=BF, device="cuda"))
    refused(ops.mla_tree_attn, a, qa=torch.zeros(7 * 2048 + 4, dtype=BF, device="cuda")[4:].view(7, 16, 128))   # off 16 bytes
    s = step
    refused(ops.kda_tree_step, s, max_nodes=70)
    refused(ops.kda_tree_step, s, x_qkv=s["x_qkv"][:, :-128])
    refused(ops.kda_tree_step, s, x_qkv=torch.zeros(7, 772, dtype=BF, device="cuda")[:, :768])   # row stride no multiple of 8
    refused(ops.kda_tree_step, s, conv_state=None)
    refused(ops.kda_tree_step, s, conv_state=s["conv_state"][:-1])
    refused(ops.kda_tree_step, s, conv_weight=s["conv_weight"].bfloat16())
    refused(ops.kda_tree_step, s, conv_weight=s["conv_weight"][:, :3])
    refused(ops.kda_tree_step, s, state=s["state"].bfloat16())
    refused(ops.kda_tree_step, s, state=s["state"][:1], conv_state=s["conv_state"][:1], state_slots=None)
    refused(ops.kda_tree_step, s, beta=s["beta"][:3])
    refused(ops.kda_tree_step, s, A_log=None)
    refused(ops.kda_tree_step, s, tape=torch.zeros(7, 2, 3, 128, dtype=BF, device="cuda"))
    refused(ops.kda_tree_step, s, out=torch.zeros(7, 2, 128, device="cuda"))
    _, tape = ops.kda_tree_step(**s)
    p = dict(path=torch.zeros(2, 4, dtype=torch.int32, device="cuda"), n_path=torch.zeros(2, dtype=torch.int32, device="cuda"),
             cu_nodes=s["cu_nodes"], slots=s["state_slots"], kda=[(tape, s["x_qkv"], s["conv_state"], s["state"])],
             mla=[(a["latent"], a["latent_cache"])], cached=a["cached"])
    before = s["state"].clone()
    ops.tree_commit(**p)
    assert torch.equal(before, s["state"])   # empty paths
    refused(ops.tree_commit, p, path=p["path"].long())
    refused(ops.tree_commit, p, path=torch.zeros(2, 65, dtype=torch.int32, device="cuda"))
    refused(ops.tree_commit, p, n_path=p["n_path"][:1])
    refused(ops.tree_commit, p, cached=None)
    refused(ops.tree_commit, p, kda=[(tape[:-1], s["x_qkv"], s["conv_state"], s["state"])])
    refused(ops.tree_commit, p, kda=[(tape, s["x_qkv"], s["conv_state"][:-1], s["state"])])
    refused(ops.tree_commit, p, kda=p["kda"] + [(tape, s["x_qkv"].float(), s["conv_state"], s["state"])])
    refused(ops.tree_commit, p, mla=[(a["latent"], a["latent_cache"][:1])])
    refused(ops.tree_commit, p, mla=p["mla"] + [(a["latent"].float(), a["latent_cache"])])
    x = torch.zeros(7, 100, device="cuda")
    i64 = torch.zeros(7, 9, dtype=torch.int64, device="cuda")
    n7 = torch.zeros(7, dtype=torch.int32, device="cuda")
    j = dict(logits=x)
    refused(ops.adjust_logits, j, history=i64)
    refused(ops.adjust_logits, j, history_len=n7)
    refused(ops.adjust_logits, j, history=i64.int(), history_len=n7)
    refused(ops.adjust_logits, j, history=i64[:3], history_len=n7)
    refused(ops.adjust_logits, j, repetition=torch.ones(6, device="cuda"))
    refused(ops.adjust_logits, j, presence=torch.ones(7, device="cuda").double())
    refused(ops.adjust_logits, j, bias_ids=i64)
    refused(ops.adjust_logits, j, bias_ids=i64, bias=torch.zeros(7, 8, device="cuda"))
    refused(ops.adjust_logits, j, allowed=torch.zeros(7, 3, dtype=torch.int32, device="cuda"))
    refused(ops.adjust_logits, j, allowed=torch.zeros(2, 4, dtype=torch.int32, device="cuda"))
    refused(ops.adjust_logits, j, allowed_rows=n7)
    refused(ops.adjust_logits, j, cu_nodes=s["cu_nodes"])
    refused(ops.adjust_logits, j, tokens=i64[:, 0])
    refused(ops.adjust_logits, j, out=x.bfloat16())
    room = torch.zeros(8, 100, device="cuda")
    refused(ops.adjust_logits, dict(logits=room[:7]), out=room[1:])      # overlaps, and is not logits itself
    refused(ops.adjust_logits, dict(logits=x.T))
    k = dict(logits=x, tokens=i64[:, 0].contiguous(), cu_nodes=s["cu_nodes"], parents=s["parents"], max_nodes=4)
    refused(ops.tree_accept, k, tokens=n7)
    refused(ops.tree_accept, k, max_nodes=0)
    refused(ops.tree_accept, k, parents=s["parents"][:2])
    refused(ops.tree_accept, k, logits=x[:, :0])
    refused(ops.tree_accept, k, logits=x.half())


def test_tree_attention_of_many_trees():
    """More trees than a wavefront has lanes, of all sizes, some without nodes, some without slots."""
    from sophia_amd import ops
    lens = [(7 * i) % 19 for i in range(150)]
    tr, qa, latent, cache, slots, cached = _attn_case(lens, [(37 * i) % 200 for i in range(150)], max_seq=200, heads=2, rank=32)
    slots[70], slots[149] = -1, 500
    for dtype in (BF, F32):
        for splits in (1, 4, None):
            got = ops.mla_tree_attn(*_dev(qa.to(dtype), latent.to(dtype), cache, tr.cu, tr.par, slots, cached), 0.1,
                                    max_nodes=18, splits=splits)
            want, mass, size = ref.attention(tr, qa, latent, cache, slots, cached, 0.1)
            _within(got, want, _attn_tol(tr, want, mass, size, dtype, 32))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rank,heads,trees", [(32, 2, 90), (128, 3, 30), (256, 1, 66)])
def test_tree_attention_of_more_work_than_fits_at_once(rank, heads, trees, dtype):
    """Ranges as long as the kernel makes them, long contexts beside short ones, partials of some trees alone."""
    from sophia_amd import ops
    lens, seq = [1 + (11 * i) % 40 for i in range(trees)], 2500
    cached = [(997 * i) % seq if i % 3 else i for i in range(trees)]
    tr, qa, latent, cache, slots, cached = _attn_case(lens, cached, max_seq=seq, heads=heads, rank=rank, dtype=dtype, q_std=0.5)
    slots[7] = -1
    want, mass, size = ref.attention(tr, qa, latent, cache, slots, cached, 0.1)
    tol = _attn_tol(tr, want, mass, size, dtype, rank) + 1800 * E32 * mass     # (sums of up to 2,500 keys)
    dev = _dev(qa, latent, cache, tr.cu, tr.par, slots, cached)
    for kw in (dict(), dict(max_len=64), dict(splits=7)):
        _within(ops.mla_tree_attn(*dev, 0.1, max_nodes=64, **kw), want, tol)
