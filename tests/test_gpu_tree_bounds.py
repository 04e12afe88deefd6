"""The drafted-token operators against float64 restatements at bounds that hold for each value by itself: the roundings of
what enters it (tests/tree_bounds.py), and the rounding of the result."""

from __future__ import annotations

import pytest
import torch

import tree_bounds
import tree_ref as ref
from test_gpu_tree_ops import _attn_case, _attn_tol, _dev, _run_step, _step_case, _within

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
E32 = 2.0 ** -24


@pytest.mark.parametrize("splits", [None, 1])
@pytest.mark.parametrize("rank,heads", [(32, 2), (64, 3), (128, 16), (256, 4)])
def test_tree_attention_loses_nothing_of_its_probabilities(rank, heads, splits):
    """bf16 inputs, small scores: many keys of opposite signs share the weight, so a result is far smaller than the sum of
    what enters it.  Probabilities enter the value product as two bf16 numbers (2^-8 of 2^-8 is lost)."""
    from sophia_amd import ops
    tr, qa, latent, cache, slots, cached = _attn_case([9, 30, 1], [600, 250, 599], heads=heads, rank=rank, seed=rank, q_std=0.3)
    got = ops.mla_tree_attn(*_dev(qa, latent, cache, tr.cu, tr.par, slots, cached), 128 ** -0.5, max_nodes=30, splits=splits)
    want, mass, size = ref.attention(tr, qa, latent, cache, slots, cached, 128 ** -0.5)
    _within(got, want, _attn_tol(tr, want, mass, size, F32, rank) + 2.0 ** -16 * mass + 2.0 ** -8 * want.abs())


# ------------------------------------------------------------------ KDA step
STEP = [
    dict(lens=[1]),
    dict(lens=[33, 64], kind="chain"),
    dict(lens=[2, 0, 16, 7], kind="forest"),
    dict(lens=[64, 3, 50], kind="odd", behind=4),
    dict(lens=[16, 9], taps=1, heads=1),
    dict(lens=[20, 5], taps=2, heads=3),
    dict(lens=[48], taps=3, gate=False),
    dict(lens=[64, 30, 16], kind="chain", strong=True),
    dict(lens=[64, 41, 26], kind="branches", strong=True),
    dict(lens=[64, 50], kind="branches", gate=False, g_dtype=F32),
    dict(lens=[31, 64], kind="odd", strong=True, taps=1),
    dict(lens=[13], g_dtype=F32, heads=16),
]


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", range(len(STEP)))
def test_tree_step_and_commit_at_the_roundings_of_each_value(case, dtype):
    """o, u, k and G of every node, and the state that a commit of each tree's last node leaves."""
    from sophia_amd import ops
    kw = dict(STEP[case])
    tr, c = _step_case(**kw, dtype=dtype, seed=case + 40)
    gate = kw.get("gate", True)
    want = tree_bounds.step(tr, **c, gate=gate)
    got, tape = _run_step(tr, c, gate=gate)
    _within(tape[:tr.total], want["tape"], want["tol_tape"])
    _within(got[:tr.total], want["o"], want["tol_o"] + (2.0 ** -8 * want["o"].abs() if dtype == BF else 0.0))
    trees = [s for s, n in enumerate(tr.lens) if n]
    nodes = {s: tr.paths[s][-1] for s in trees}
    path = torch.full((len(tr.lens), max(map(len, nodes.values()))), -1, dtype=torch.int32)
    for s in trees:
        path[s, :len(nodes[s])] = torch.tensor(nodes[s], dtype=torch.int32)
    hist, state = _dev(c["conv_state"], c["state"])
    ops.tree_commit(path.cuda(), torch.tensor([len(nodes.get(s, [])) for s in range(len(tr.lens))], dtype=torch.int32).cuda(),
                    tr.cu.cuda(), c["slots"].cuda(), kda=[(tape, c["x"].cuda(), hist, state)])
    for s in trees:
        _within(state[int(c["slots"][s])], *want["commit"](s, nodes[s]))


@pytest.mark.parametrize("drop", [55.0, 75.0, 100.0])
def test_tree_step_after_one_strong_decay(drop):
    """Channels that lose nearly everything at one node and little at those below it: weights near 1 behind large |G|, formed from
    e^G e^-G (to 60) or with a reference per tile; in one tree all channels, in the other every second one."""
    tr, c = _step_case([40, 64], kind="branches", dtype=F32, gate=False, seed=70)
    c["g"] = c["g"] * 0.01
    c["g"][2], c["g"][40 + 5, :, ::2] = -drop, -drop
    want = tree_bounds.step(tr, **c, gate=False)
    got, tape = _run_step(tr, c, gate=False)
    _within(tape, want["tape"], want["tol_tape"])
    _within(got, want["o"], want["tol_o"])


@pytest.mark.parametrize("taps", [1, 4])
def test_a_q_that_is_not_finite_is_its_own_nodes_output_alone(taps):
    """As in the decode step: q enters no state, so the tape and the other nodes' outputs are as without it (but for those whose
    conv reads the sample)."""
    tr, c = _step_case([40, 12], kind="mixed", dtype=F32, seed=11, taps=taps)
    want = tree_bounds.step(tr, **c)
    hit = {3: (0, float("nan")), 17: (1, float("inf")), 41: (0, float("-inf"))}     # row: head, value (of q)
    for row, (head, value) in hit.items():
        c["x"][row, head * 128 + 9] = value
    got, tape = _run_step(tr, c)
    _within(tape, want["tape"], want["tol_tape"])
    for _, row, path, _ in tr.nodes():
        for head in range(2):
            read = [r for r in path[-taps:] if r in hit and hit[r][0] == head]
            if read:
                assert torch.isnan(got[row, head]).all()
            else:
                _within(got[row, head], want["o"][row, head], want["tol_o"][row, head])
