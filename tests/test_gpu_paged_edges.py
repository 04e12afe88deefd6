"""The operators on paged latents and beams at the ends of what their documentation allows: bounds below a sequence's rows in either
form of the attention."""

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
