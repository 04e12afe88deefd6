"""The bounds of tests/tree_bounds.py (CPU): an fp32 form lies within them; operands in bf16, a state in bf16 and an output
without the drafted nodes' term do not."""

from __future__ import annotations

import pytest
import torch

import tree_bounds
import tree_ref as ref

F32, BF = torch.float32, torch.bfloat16


def _case(lens, kind, seed, *, taps=4, gate=True, strong=False, heads=2):
    tr = ref.Trees(lens, kind, seed)
    gen = torch.Generator().manual_seed(seed + 100)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    inner, n_slots = heads * 128, len(lens) + 2
    c = dict(x=rn(tr.rows, 3 * inner), conv_w=rn(3 * inner, taps) * 0.5,
             conv_state=rn(n_slots, 3 * inner, taps - 1) if taps > 1 else None, g=rn(tr.rows, heads, 128) * (2 if strong else 1),
             beta=rn(tr.rows, heads), state=rn(n_slots, heads, 128, 128) * 0.2, slots=tr.slots(n_slots, seed),
             A_log=rn(heads) * 0.3, dt_bias=rn(inner) + (3.0 if strong else -2.0), gate=gate)
    if not gate:
        c["g"] = -torch.nn.functional.softplus(c["g"] - 1.0)
    return tr, c


CASES = [dict(lens=[1, 33, 64], kind="chain", seed=3), dict(lens=[17, 32, 1], kind="wide", seed=2),
         dict(lens=[20, 5], kind="mixed", seed=5, taps=2), dict(lens=[48], kind="mixed", seed=7, taps=3, gate=False),
         dict(lens=[64, 30], kind="chain", seed=9, strong=True), dict(lens=[64], kind="branches", seed=10, strong=True, taps=1)]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_bounds_hold_for_fp32_and_reject_less(case):
    tr, c = _case(**CASES[case])
    want = tree_bounds.step(tr, **c)
    o, tape, _ = ref.kda_step(tr, **c)
    # two float64 forms: the recurrence node by node, and the chunk form
    assert torch.allclose(want["o"], o, rtol=1e-9, atol=1e-12) and torch.allclose(want["tape"], tape, rtol=1e-9, atol=1e-12)

    def off(got):
        return (got.double() - want["o"]).abs() > want["tol_o"]
    assert not off(tree_bounds.step_f32(tr, **c)).any()
    depth = torch.zeros(tr.total, dtype=torch.long)
    for _, row, path, _ in tr.nodes():
        depth[row] = len(path)
    first = depth <= 2      # (strong decays leave little of the state below them)
    assert off(tree_bounds.step_f32(tr, **dict(c, state=c["state"].to(BF).float())))[first].double().mean() > 0.6
    assert off(tree_bounds.step_f32(tr, **c, operands=BF))[first].double().mean() > 0.6
    assert off(tree_bounds.step_f32(tr, **c, nodes=False)).double().mean() > 0.95   # (a node's own term is one of them)
    # an output of zeros is none either
    assert off(torch.zeros_like(o)).double().mean() > 0.95
    for s, n in enumerate(tr.lens):
        nodes = tr.paths[s][n - 1]
        state, tol = want["commit"](s, nodes)
        S = ref.kda_step(tr, **c)[2][tr.offsets[s] + n - 1]
        assert torch.allclose(state, S, rtol=1e-9, atol=1e-12)
        rounded = state.to(BF).double()
        assert ((rounded - state).abs() > tol)[state != 0].double().mean() > 0.6
