"""The drafted-token operators against float64 restatements at bounds that hold for each value by itself: the roundings of
what enters it (tests/tree_bounds.py), and the rounding of the result."""

from __future__ import annotations

import pytest
import torch

import tree_ref as ref
from test_gpu_tree_ops import _attn_case, _attn_tol, _dev, _within

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
