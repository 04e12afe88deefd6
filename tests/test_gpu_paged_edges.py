"""The operators on paged latents and beams at the ends of what their documentation allows: bounds below a sequence's rows in either
form of the attention, and logits of any size."""

from __future__ import annotations

import pytest
import torch

import paged_ref as ref
from test_gpu_paged_ops import BF, F32, _attn

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ max_new below a sequence's rows
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("splits", [0, 1, 3])
@pytest.mark.parametrize("heads,max_new", [(16, 1), (5, 3), (4, 4), (1, 7), (16, 2), (12, 1)])
def test_the_first_max_new_rows_are_computed_whatever_a_sequence_has(heads, max_new, splits, dtype):
    """16 columns or fewer are the narrow form's, more the wide one's; sequences of more and of fewer rows, one range of keys or several."""
    _attn(ref.Paged([9, 1, 4, 0, 7], [40, 2000, 700, 5, 1100], heads=heads, dtype=dtype, behind=2), max_new=max_new, splits=splits)


# ------------------------------------------------------------------ beams whose logits are large
def _beams(logits, scores, beams, keep):
    """(score, parent, token) in float64, the greatest logit subtracted before anything is rounded.  A beam's candidates are in the
    order of its logits, as score + x - lse is without roundings: in 64 bits sums of different logits may come out equal."""
    x, token = torch.sort(torch.where(torch.isnan(logits), -torch.inf, logits).double(), dim=-1, descending=True, stable=True)
    top, V = x[:, :1], x.size(1)
    value = (x - top) - torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    value, at = torch.sort((scores.double()[:, None] + value).view(-1, beams * V), dim=-1, descending=True, stable=True)
    token = torch.gather(token.view(-1, beams * V), 1, at)
    return value[:, :keep], at[:, :keep] // V, token[:, :keep]


def _check(logits, scores, beams, keep):
    from sophia_amd import ops
    got = [t.cpu() for t in ops.beam_select(logits.cuda(), scores.cuda(), beams, keep=keep)]
    want = _beams(logits, scores, beams, keep)
    assert torch.equal(got[1].long(), want[1]) and torch.equal(got[2], want[2])
    # An exponential of d = x - top: d to 2^-24 of it, its product with log2 e to another, the exponential to 2^-22; of the sum
    # the terms e^d |d| are at most (their entropy) ln 2^17 < 12 parts: 12 2^-23.  Sums in fp32 of 32 values in four chains, and of
    # 64 lanes in six steps: 16 2^-24.  Together below 2^-18, whatever the logits' size; then the result's rounding.
    tol = 2.0 ** -18 + 2.0 ** -24 * want[0].abs()
    err = (got[0].double() - want[0]).abs()
    assert bool((err <= tol).all()), f"off by {float(err.max()):.3g}"
    return got


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("offset", [0.0, 100.0, -1000.0, 1013.0, 10014.0, -10014.0, 1.0e6])
def test_beams_are_as_exact_far_from_zero(offset, dtype):
    gen = torch.Generator().manual_seed(int(abs(offset)))
    logits = (torch.randn(6, 65536, generator=gen) * 3 + offset).to(dtype)
    _check(logits, -torch.rand(6, generator=gen), 3, 8)


def _row(name, dtype, lowest):
    row = (torch.randn(1, 30000, generator=torch.Generator().manual_seed(len(name))) * 2).to(dtype)
    at, value = ROWS[name]
    for i, v in zip(at, value):
        row[0, i] = lowest if v is None else v
    return row


# Places of a row and what is there (None: the type's lowest value); 8,192 logits are a part of it, for one work-group.
ROWS = {
    "a part": ([slice(8192, 16384)], [None]),
    "all parts but the last": ([slice(0, 24576)], [None]),
    "all but a hundred": ([slice(100, None)], [None]),
    "all but one": ([slice(None), 12345], [None, 1.5]),
    "every other": ([slice(None, None, 2)], [None]),
    "a part, and one of -inf": ([slice(8192, 16384), slice(0, 8192)], [None, -torch.inf]),
    "parts above the lowest": ([slice(8192, None)], [-2.5e38]),
    "the last ones, above the lowest": ([slice(20000, None)], [-2.4e38]),
    "every one": ([slice(None)], [None]),
    "every one great": ([slice(None)], [2.5e38]),
    "all but one, which is low too": ([slice(None), 5], [-2.5e38, -2.4e38]),
    "one great": ([77], [3.0e38]),
    "one great behind the first part": ([9000], [2.5e38]),
    "tiny ones": ([slice(None), slice(0, None, 3), slice(1, None, 300), slice(2, None, 1000)], [0.0, -0.0, 1.0e-30, 2.0e-30]),
}


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("name", ROWS)
def test_tokens_masked_with_the_types_lowest_value(name, dtype):
    """Finite, so candidates: but behind all others, and without a share of the sums."""
    _check(_row(name, dtype, torch.finfo(dtype).min), torch.tensor([-0.5]), 1, 8)


def test_beams_that_differ_by_a_constant_are_ordered_by_their_scores():
    """The same logits, to which a row adds what leaves them exact: equal continuations, so the beams' own scores decide, and where
    these are equal the order of the beams."""
    gen = torch.Generator().manual_seed(3)
    row = torch.round(torch.randn(1, 40000, generator=gen) * 3 * 256) / 256          # (multiples of 2^-8 below 16)
    logits = row + torch.tensor([0.0, 8192.0, -1024.0, 100.0])[:, None]
    got = _check(logits, torch.tensor([-5.0, -5.0, -5.0, -5.0]), 4, 8)
    assert got[1].tolist() == [[0, 1, 2, 3, 0, 1, 2, 3]]
    got = _check(logits, torch.tensor([-5.00001, -5.0, -5.000005, -5.00002]), 4, 8)
    assert got[1].tolist()[0][:4] == [1, 2, 0, 3]
    for r in range(4):
        alone = _check(logits[r:r + 1].contiguous(), torch.tensor([-5.0]), 1, 16)
        assert torch.equal(alone[0], _check(row, torch.tensor([-5.0]), 1, 16)[0])


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("beams,keep", [(1, 8), (4, 12), (20, 64)])
def test_groups_of_rows_of_every_kind(beams, keep, dtype):
    """Sums that are equal in 64 bits though their logits are not, in several beams and in more of them than a set holds."""
    lowest, gen = torch.finfo(dtype).min, torch.Generator().manual_seed(8)
    logits = torch.cat([_row(name, dtype, lowest) for name in ROWS] * beams)[:4 * beams]
    _check(logits, -torch.rand(logits.size(0), generator=gen), beams, keep)
    _check(logits, torch.full((logits.size(0),), -1.0), beams, keep)
