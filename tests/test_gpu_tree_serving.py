"""Calls that a server makes of the drafted-token step beside the ordinary ones."""

from __future__ import annotations

import pytest
import torch

import tree_ref as ref
from test_gpu_tree_decode import _caches, _decode, _load, _model, _prefill

pytestmark = pytest.mark.gpu


def _strict(tr, logits, tokens, bound):
    """tree_ref.accept with -1 for rows without a choice, at which walks end."""
    chosen = ref.accept(tr, logits, tokens, bound)[3]
    clean = torch.where(torch.isnan(logits.double()), float("-inf"), logits.double())
    chosen = [c if float(r.max()) > float("-inf") else -1 for c, r in zip(chosen, clean)]
    paths, counts, following = [], [], []
    for s, parents in enumerate(tr.parents):
        base, path = tr.offsets[s], [0] if parents else []
        while path and chosen[base + path[-1]] >= 0:
            nxt = [i for i, p in enumerate(parents) if 0 <= p < i and p == path[-1] and int(tokens[base + i]) == chosen[base + p]]
            if not nxt:
                break
            path.append(nxt[0])
        paths.append(path + [-1] * (bound - len(path)))
        counts.append(len(path))
        following.append(chosen[base + path[-1]] if path else -1)
    return paths, counts, following, chosen


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [1, 3, 2048, 4099])
def test_strict_walks_end_at_rows_without_a_choice(vocab, dtype):
    """Rows of -inf, of NaN and of both say -1 (also where a token is -1); the others, and walks that meet none, are as ever."""
    from sophia_amd import ops
    tr = ref.Trees([20, 0, 64, 7, 1], "wide", 2, behind=2)
    gen = torch.Generator().manual_seed(vocab)
    x = torch.randn(tr.rows, vocab, generator=gen).to(dtype)
    none = torch.rand(tr.rows, generator=gen) < 0.3
    none[20], none[0] = False, False
    x[none] = float("-inf")
    x[none.nonzero()[::2, 0], 0] = float("nan")
    tokens = torch.randint(-1, 1, (tr.rows,), generator=gen)
    chosen = ref.accept(tr, x, tokens, 64)[3]
    for _, row, path, _ in tr.nodes():
        if len(path) > 1 and torch.rand((), generator=gen) < 0.8:
            tokens[row] = chosen[path[-2]]      # (0 after a row without a choice)
    want = _strict(tr, x, tokens, 64)
    assert -1 in want[3] and max(want[1]) > 1 and want != ref.accept(tr, x, tokens, 64)
    got = ops.tree_accept(x.cuda(), tokens.cuda(), tr.cu.cuda(), tr.par.cuda(), max_nodes=64, strict=True)
    assert tuple(t.tolist() for t in got) == want


def test_a_mask_that_allows_nothing_ends_the_sequence():
    """A drafted child of token 0 below a node whose mask allows nothing is not kept, and no token follows; a sequence beside it
    goes on."""
    from sophia_amd.runtime import pack_trees, verify_trees
    model = _model(seed=9)
    slots, lens = [2, 0], [30, 11]
    _prefill(model, slots, lens)
    start = _caches(model)
    trees = pack_trees(model, [([5, 0, 0], [-1, 0, 1]), ([7, 0], [-1, 0])], slots, lens)
    one = torch.zeros(1, 16, dtype=torch.int32, device="cuda")      # nothing; the other rows have no mask
    rows = torch.tensor([0, -1, -1, -1, -1], dtype=torch.int32, device="cuda")
    only0 = torch.zeros(1, 16, dtype=torch.int32, device="cuda")
    only0[0, 0] = 1
    out = verify_trees(model, trees, allowed=torch.cat([one, only0]), allowed_rows=rows)
    assert out.n_path[0] == 1 and out.next_token[0] == -1 and out.path[0].tolist() == [0, -1, -1] and out.cached[0] == 31
    assert out.next_token[1] >= 0
    got = _caches(model)
    _load(model, start)
    model.commit_tree(model.forward_tree(trees), out.path, torch.minimum(out.n_path, out.n_path.new_tensor([1, 2])))
    for a, b in zip(got, _caches(model)):
        assert torch.equal(a, b)
    # where the mask allows token 0 alone, the child of token 0 is kept
    _load(model, start)
    out = verify_trees(model, trees, allowed=torch.cat([one, only0]), allowed_rows=rows + (rows == 0).int())
    assert out.n_path[0] >= 2 and out.path[0, :2].tolist() == [0, 1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_adjusted_nodes_are_the_single_rows_of_the_texts_that_they_end(dtype):
    """With the cached tokens as history, each node's logits are what a row of decoding gets whose history is the cached tokens
    and its path, node 0 counted once."""
    from sophia_amd import ops
    tr, vocab, width = ref.Trees([9, 1, 30], "mixed", 4), 777, 50
    gen = torch.Generator().manual_seed(1)
    ri = lambda *s: torch.randint(0, 40, s, generator=gen)  # noqa: E731
    x = (torch.randn(tr.rows, vocab, generator=gen) * 3).to(dtype)
    cached, prompt, text, tokens = [50, 7, 0], [20, 7, 0], ri(3, width), ri(tr.rows)
    pens = dict(repetition=torch.tensor([1.3, 1.1, 0.8]), presence=torch.tensor([0.4, 0.0, 0.2]),
                frequency=torch.tensor([0.1, 0.3, 0.25]))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    got = ops.adjust_logits(x.cuda(), history=text.cuda(), history_len=i32(cached), prompt_len=i32(prompt), tokens=tokens.cuda(),
                            cu_nodes=tr.cu.cuda(), parents=tr.par.cuda(), max_nodes=30, **{k: v.cuda() for k, v in pens.items()})
    of = [(s, path) for s, _, path, _ in tr.nodes()]
    full = [text[s, :cached[s]].tolist() + tokens[path].tolist() for s, path in of]
    hist = torch.tensor([t + [0] * (width + 30 - len(t)) for t in full])
    rows = ops.adjust_logits(x.cuda(), history=hist.cuda(), history_len=i32([len(t) for t in full]),
                             prompt_len=i32([prompt[s] for s, _ in of]),
                             **{k: v[[s for s, _ in of]].cuda() for k, v in pens.items()})
    assert torch.equal(got, rows)


def test_a_path_past_the_steps_bound_ends_there():
    """A tree with more nodes than the step's max_nodes: its tape holds nothing of the others (NaN here), and a commit along them
    takes the part before them."""
    from sophia_amd import ops
    from test_gpu_tree_ops import _run_step, _step_case
    tr, c = _step_case([20, 6], kind="chain", dtype=torch.float32, seed=2)
    tape = torch.full((tr.rows, 2, 3, 128), float("nan"), device="cuda")
    _run_step(tr, c, max_nodes=12, tape=tape)
    path = torch.arange(20, dtype=torch.int32, device="cuda").repeat(2, 1)
    latent, cached = torch.randn(tr.rows, 32, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    slots, x = c["slots"].cuda(), c["x"].cuda()
    left = []
    for count, bound in ((20, 12), (12, 64)):     # the whole path within the bound, and the part before it
        hist, state, cache = c["conv_state"].cuda(), c["state"].cuda(), torch.zeros(c["state"].size(0), 40, 32, device="cuda")
        ops.tree_commit(path, torch.tensor([count, 6], dtype=torch.int32, device="cuda"), tr.cu.cuda(), slots,
                        kda=[(tape, x, hist, state)], mla=[(latent, cache)], cached=cached, max_nodes=bound)
        left.append((hist, state, cache))
    for a, b in zip(*left):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    for bound in (0, 65):
        with pytest.raises(RuntimeError, match="max_nodes"):
            ops.tree_commit(path, torch.tensor([1, 1], dtype=torch.int32, device="cuda"), tr.cu.cuda(), slots,
                            kda=[(tape, x, *left[0][:2])], max_nodes=bound)


def test_commit_tree_keeps_to_the_steps_bound():
    from dataclasses import replace
    from sophia_amd.runtime import pack_trees
    model = _model(seed=12)
    _prefill(model, [1], [25])
    start = _caches(model)
    trees = replace(pack_trees(model, [([3, 4, 5, 6, 7], [-1, 0, 1, 2, 3])], [1], [25]), max_nodes=3)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    left = []
    for count in (5, 3):
        _load(model, start)
        model.commit_tree(model.forward_tree(trees), i32([[0, 1, 2, 3, 4]]), i32([count]))
        left.append(_caches(model))
    for a, b in zip(*left):
        assert torch.isfinite(a).all() and torch.equal(a, b)


def test_padded_prompts_are_refused_until_their_mask_is_cleared():
    """The step has no mask over cached keys: a left-padded prompt's pads would be attended to."""
    from sophia_amd.kda import set_pad_mask
    from sophia_amd.runtime import pack_trees, verify_trees
    model = _model(seed=13)
    ids = torch.randint(0, 512, (2, 20), generator=torch.Generator().manual_seed(1)).cuda()
    mask = torch.ones(2, 20, dtype=torch.bool, device="cuda")
    mask[0, :7] = False
    set_pad_mask(model, mask)
    with torch.no_grad():
        model(ids)
    before = _caches(model)
    trees = pack_trees(model, [([1, 2], [-1, 0]), ([3], [-1])], [0, 1], [20, 20])
    with pytest.raises(RuntimeError, match="set_pad_mask"):
        verify_trees(model, trees)
    for a, b in zip(before, _caches(model)):
        assert torch.equal(a, b)
    set_pad_mask(model, None)
    with torch.no_grad():
        model(ids)
    assert verify_trees(model, trees).n_path.min() >= 1


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-2), (torch.bfloat16, 6e-2)], ids=["f32", "bf16"])
def test_drafted_decoding_chooses_greatest_logits_of_decode_steps(dtype, tol):
    """Every token that decoding with drafted trees keeps or says has, in decode steps over the same text, a logit as great as
    any but for the roundings that the steps do not share (the tolerances of the decoder's own tests, relative to the greatest
    magnitude, on either logit)."""
    from sophia_amd.runtime import pack_trees, verify_trees
    model = _model(seed=14, dtype=dtype)
    _, first = _prefill(model, [3], [37])
    start = _caches(model)
    text, cached, known = [], 37, first[0]
    while len(text) < 24:      # drafts from the model itself: what it says after its last choice, and a wrong token beside
        probe = _caches(model)
        guess = [known]
        for _ in range(3):
            out = verify_trees(model, pack_trees(model, [([guess[-1]], [-1])], [3], [cached + len(guess) - 1]))
            guess.append(int(out.next_token[0]))
        _load(model, probe)
        tree = (guess[:1] + [(guess[1] + 1) % 512] + guess[1:], [-1, 0, 0, 2, 3])
        out = verify_trees(model, pack_trees(model, [tree], [3], [cached]))
        text += [tree[0][i] for i in out.path[0, :int(out.n_path[0])].tolist()]
        cached, known = int(out.cached[0]), int(out.next_token[0])
        assert cached == 37 + len(text)
    _load(model, start)
    rows = _decode(model, text, 3, 37)
    for said, row in zip(text[1:] + [known], rows):
        row = row.double()
        assert float(row.max() - row[said]) <= 2 * tol * float(row.abs().max())


def test_an_ended_sequences_token_may_come_back():
    """next_token -1 as node 0 of the next tree (a step whose tokens stay on the device): run as a token of the vocabulary, and
    the trees beside it are as they are without it."""
    from dataclasses import replace
    from sophia_amd.runtime import pack_trees, verify_trees
    model = _model(seed=15)
    _prefill(model, [0, 4], [12, 50])
    start = _caches(model)
    trees = pack_trees(model, [([0, 3], [-1, 0]), ([7, 1, 511], [-1, 0, 0])], [0, 4], [12, 50])
    want, kept = verify_trees(model, trees), _caches(model)
    _load(model, start)
    out = verify_trees(model, replace(trees, token_ids=torch.tensor([-1, 3, 7, 1, 600], device="cuda")))
    assert torch.equal(out.logits, want.logits) and torch.equal(out.n_path, want.n_path)
    for a, b in zip(_caches(model), kept):
        assert torch.equal(a, b)
