"""The drafted-token step of the whole decoder on the GPU: forward_tree, commit_tree, pack_trees and verify_trees, run
together as a server runs them, eager and captured."""

from __future__ import annotations

import random

import pytest
import torch

pytestmark = pytest.mark.gpu

SMALL = dict(vocab_size=512, n_layers=8, ffn_hidden=320, mla_q_rank=64, mla_kv_rank=32, dim=256, num_heads=2, max_seq_len=400,
             max_batch_size=6)


def _model(seed=0, dtype=torch.float32, **over):
    from sophia_amd.config import ModelArgs
    from sophia_amd.decoder import Transformer
    torch.manual_seed(seed)
    model = Transformer(ModelArgs(**{**SMALL, **over}))
    with torch.no_grad():
        for m in model.modules():
            if m.__class__.__name__ == "AttentionResidualMixer":
                m.query.weight.normal_(0.0, 0.05)
    return model.to("cuda").eval().cast_weights_(dtype)


def _prefill(model, slots, lens, seed=1):
    gen = torch.Generator().manual_seed(seed)
    prompts = [torch.randint(0, model.args.vocab_size, (n,), generator=gen) for n in lens]
    with torch.no_grad():
        logits = model.forward_step(prefill_ids=torch.cat(prompts).cuda(), prefill_lens=lens,
                                    prefill_slots=torch.tensor(slots, dtype=torch.int32, device="cuda"))
    return prompts, logits.float().argmax(-1).tolist()


def _caches(model):
    out = []
    for layer in model.layers:
        a = layer.attn
        out += [a.latent_cache.clone()] if layer.layer_type == "mla" else [a.recurrent_state.clone(), a.conv_state.clone()]
    return out


def _load(model, caches):
    it = iter(caches)
    for layer in model.layers:
        a = layer.attn
        for t in ([a.latent_cache] if layer.layer_type == "mla" else [a.recurrent_state, a.conv_state]):
            t.copy_(next(it))


def _rel(a, b):
    return float((a.double() - b.double()).abs().max() / b.double().abs().max().clamp(min=1e-30))


TREES = [([0, 9, 8, 7, 6, 5, 4], [-1, 0, 0, 1, 1, 2, 3]), ([3], [-1]), ([1, 2, 3, 4, 5], [-1, 0, 1, 2, 3])]


def _decode(model, tokens, slot, pos):
    """Logits after each of ``tokens``, one decode step each."""
    dev = dict(device="cuda")
    out = []
    with torch.no_grad():
        for i, t in enumerate(tokens):
            out.append(model.forward_step(decode_ids=torch.tensor([t], **dev), decode_slots=torch.tensor([slot], dtype=torch.int32, **dev),
                                          decode_pos=torch.tensor([pos + i], **dev), max_decode_len=pos + i + 1)[0])
    return out


# The decode step rounds what the tree step does not: conv outputs in a bf16 model, and the latent attention's operands to
# bf16 in an fp32 one too; logits are compared at the tolerances of the decoder's own tests.
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-2), (torch.bfloat16, 6e-2)], ids=["f32", "bf16"])
def test_every_node_is_the_decode_of_its_path_and_commit_its_caches(dtype, tol):
    from sophia_amd.runtime import pack_trees
    model = _model(dtype=dtype)
    slots, lens = [4, 0, 2], [70, 3, 131]
    _prefill(model, slots, lens)
    before = _caches(model)
    trees = pack_trees(model, TREES, slots, lens)
    draft = model.forward_tree(trees)
    for a, b in zip(before, _caches(model)):
        assert torch.equal(a, b)    # only read
    path = torch.tensor([[0, 1, 3, 6], [0, -1, -1, -1], [0, 1, 2, -1]], dtype=torch.int32, device="cuda")
    n_path = torch.tensor([4, 1, 3], dtype=torch.int32, device="cuda")
    model.commit_tree(draft, path, n_path)
    with pytest.raises(RuntimeError, match="committed"):
        model.commit_tree(draft, path, n_path)
    after = _caches(model)
    row = 0
    for (toks, pars), slot, pos in zip(TREES, slots, lens):
        for i in range(len(toks)):
            walk, j = [], i
            while j >= 0:
                walk.insert(0, toks[j])
                j = pars[j]
            _load(model, before)
            assert _rel(draft.logits[row + i], _decode(model, walk, slot, pos)[-1]) <= tol
        row += len(toks)
    _load(model, before)
    for s, (slot, pos) in enumerate(zip(slots, lens)):
        nodes = path[s, :int(n_path[s])].tolist()
        _decode(model, [TREES[s][0][i] for i in nodes], slot, pos)
    for got, want, old in zip(after, _caches(model), before):
        for slot in range(6):
            if slot not in slots:
                assert torch.equal(got[slot], old[slot])     # other sequences
            else:
                assert _rel(got[slot], want[slot]) <= tol


def _draft(rng, root, after, vocab):
    """A tree whose nodes are sometimes the true continuation ``after`` and sometimes not."""
    toks, pars, true_at = [root], [-1], 0
    for depth, t in enumerate(after[:rng.randint(0, 6)]):
        for _ in range(rng.randint(0, 2)):
            toks.append(rng.randrange(vocab))
            pars.append(rng.randrange(len(toks) - 1))
        toks.append(t if rng.random() < 0.8 else (t + 1) % vocab)
        pars.append(true_at)
        true_at = len(toks) - 1
    return toks, pars


def test_drafted_decoding_says_what_undrafted_decoding_says():
    """Greedy decoding with drafted trees, right and wrong, gives the tokens of decoding without drafts (trees of one node);
    an fp32 model, whose logits are then alike to about 1e-6 whatever rows a step has."""
    from sophia_amd.runtime import pack_trees, verify_trees
    model = _model(seed=3)
    slots, lens = [1, 5], [40, 9]
    prompts, first = _prefill(model, slots, lens)
    start = _caches(model)

    def controls(texts):
        width = max(len(t) for t in texts)
        hist = torch.tensor([t + [0] * (width - len(t)) for t in texts], device="cuda")
        n = torch.tensor([len(t) for t in texts], dtype=torch.int32, device="cuda")
        return dict(history=hist, history_len=n, repetition=torch.tensor([1.3, 1.1], device="cuda"),
                    frequency=torch.tensor([0.0, 0.01], device="cuda"))

    def run(drafter, steps):
        _load(model, start)
        texts, cached, known = [p.tolist() for p in prompts], list(lens), list(first)
        taken = 0
        while min(len(t) - n for t, n in zip(texts, lens)) < steps:
            batch = [drafter(s, known[s], len(texts[s])) for s in range(2)]
            out = verify_trees(model, pack_trees(model, batch, slots, cached), **controls(texts))
            cached = out.cached.tolist()
            for s in range(2):
                nodes = out.path[s, :int(out.n_path[s])].tolist()
                texts[s] += [batch[s][0][i] for i in nodes]
                taken = max(taken, len(nodes))
                assert cached[s] == len(texts[s])
            known = out.next_token.tolist()
        return [t + [k] for t, k in zip(texts, known)], taken

    plain, _ = run(lambda s, root, at: ([root], [-1]), 30)
    rng = random.Random(5)
    drafted, taken = run(lambda s, root, at: _draft(rng, root, plain[s][at + 1:], 512), 20)
    assert taken >= 4      # drafts were kept
    for s in range(2):
        n = lens[s] + 20
        assert drafted[s][:n] == plain[s][:n]


def test_verify_step_captured_replays_as_it_runs_eager():
    from sophia_amd.runtime import pack_trees, verify_trees
    model = _model(seed=2, dtype=torch.bfloat16, mla_kv_rank=128)
    slots, lens = [3, 0, 5], [100, 20, 64]
    _prefill(model, slots, lens)
    start = _caches(model)
    rng = random.Random(1)
    batches = []
    for _ in range(4):      # the same sizes, other trees
        trees = []
        for n in (9, 16, 1):
            trees.append(([rng.randrange(512) for _ in range(n)], [-1] + [rng.randrange(i) for i in range(1, n)]))
        batches.append(pack_trees(model, trees, slots, lens))
    static = pack_trees(model, [([0] * n, [-1] + [0] * (n - 1)) for n in (9, 16, 1)], slots, lens)
    bias_ids = torch.randint(0, 512, (3, 5), device="cuda")
    controls = dict(bias_ids=bias_ids, bias=torch.randn(3, 5, device="cuda"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        verify_trees(model, static, **controls)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = verify_trees(model, static, **controls)
    for batch in batches:
        _load(model, start)
        want = verify_trees(model, batch, **controls)
        eager = _caches(model)
        torch.cuda.synchronize()
        _load(model, start)
        for name in ("token_ids", "parents", "cached"):
            getattr(static, name).copy_(getattr(batch, name))
        graph.replay()
        torch.cuda.synchronize()
        for name in ("path", "n_path", "next_token", "cached", "logits"):
            assert torch.equal(getattr(out, name), getattr(want, name)), name
        for a, b in zip(_caches(model), eager):
            assert torch.equal(a, b)


def _pad(trees, n, rows):
    """``trees`` with trees without nodes up to ``n`` (their slots are taken by nobody), and rows of no tree up to ``rows``."""
    from dataclasses import replace
    grow = lambda t, size, v: torch.cat([t, t.new_full((size - t.numel(),), v)])  # noqa: E731
    return replace(trees, token_ids=grow(trees.token_ids, rows, 0), parents=grow(trees.parents, rows, -1),
                   cu_nodes=grow(trees.cu_nodes, n + 1, int(trees.cu_nodes[-1])), slots=grow(trees.slots, n, -1),
                   cached=grow(trees.cached, n, 0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_captured_step_takes_padded_batches_of_any_trees(dtype):
    """One captured step of 40 rows and 4 trees, with trees of other sizes, sequences and contexts at every replay, is what
    the step of those trees alone gives, and leaves all other slots as they were."""
    from dataclasses import replace
    from sophia_amd.runtime import pack_trees, verify_trees
    model = _model(seed=6, dtype=dtype, mla_kv_rank=64)
    lens = [90, 1, 300, 64, 7, 129]
    _prefill(model, list(range(6)), lens)
    start = _caches(model)
    rng = random.Random(4)

    def batch(sizes):
        trees = [([rng.randrange(512) for _ in range(n)], [-1] + [rng.randrange(i) for i in range(1, n)]) for n in sizes]
        slots = rng.sample(range(6), len(sizes))
        return pack_trees(model, trees, slots, [lens[s] for s in slots])
    static = replace(_pad(batch([3]), 4, 40), max_nodes=24, max_len=320)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        verify_trees(model, static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = verify_trees(model, static)
    for sizes in ([24, 1, 9, 6], [5], [13, 17], []):
        if sizes:
            trees = batch(sizes)
            padded = _pad(trees, 4, 40)
        else:
            padded = _pad(replace(trees, cu_nodes=trees.cu_nodes[:1], slots=trees.slots[:0], cached=trees.cached[:0]), 4, 40)
        for name in ("token_ids", "parents", "cu_nodes", "slots", "cached"):
            getattr(static, name).copy_(getattr(padded, name))
        _load(model, start)
        want = verify_trees(model, replace(padded, max_nodes=24, max_len=320))
        eager = _caches(model)
        _load(model, start)
        graph.replay()
        torch.cuda.synchronize()
        n, rows = len(sizes), sum(sizes)
        for name in ("path", "n_path", "next_token", "cached"):
            assert torch.equal(getattr(out, name), getattr(want, name)), name
        assert torch.equal(out.logits[:rows], want.logits[:rows])
        for a, b in zip(_caches(model), eager):
            assert torch.equal(a, b)
        assert out.n_path[n:].tolist() == [0] * (4 - n) and out.next_token[n:].tolist() == [-1] * (4 - n)
        used = trees.slots.tolist() if sizes else []
        for a, b in zip(eager, start):
            for slot in set(range(6)) - set(used):
                assert torch.equal(a[slot], b[slot])
        if sizes:     # the trees alone: other bounds, so other divisions of the work
            _load(model, start)
            alone = verify_trees(model, trees)
            assert _rel(out.logits[:rows].float(), alone.logits.float()) <= (1e-4 if dtype == torch.float32 else 6e-2)
            if dtype == torch.float32:
                assert alone.n_path.tolist() == out.n_path[:n].tolist() and alone.next_token.tolist() == out.next_token[:n].tolist()


def test_caches_may_grow_between_a_drafted_step_and_its_commit():
    from sophia_amd.runtime import pack_trees
    model, other = _model(seed=4), _model(seed=4)
    paths = torch.tensor([[0, 1], [0, -1]], dtype=torch.int32, device="cuda"), torch.tensor([2, 1], dtype=torch.int32, device="cuda")
    for m in (model, other):
        _prefill(m, [5, 1], [33, 60])
        draft = m.forward_tree(pack_trees(m, TREES[:2], [5, 1], [33, 60]))
        if m is other:
            m.ensure_batch_capacity(9)
        m.commit_tree(draft, *paths)
    for a, b in zip(_caches(model), _caches(other)):
        assert b.size(0) == 9 and torch.equal(a, b[:6]) and not b[6:].any()


def test_two_drafted_steps_of_different_sequences_on_two_streams():
    """Two steps under way at once, each on its stream, of different slots: as one after the other."""
    from sophia_amd.runtime import pack_trees, verify_trees
    model = _model(seed=5, dtype=torch.bfloat16, mla_kv_rank=128)
    slots, lens = [0, 3, 4], [200, 17, 80]
    _prefill(model, slots, lens)
    start = _caches(model)
    batches = [pack_trees(model, TREES[:2], slots[:2], lens[:2]), pack_trees(model, TREES[2:], slots[2:], lens[2:])]
    want = [verify_trees(model, b) for b in batches]
    after = _caches(model)
    _load(model, start)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    got = []
    for b, s in zip(batches, streams):
        with torch.cuda.stream(s):
            got.append(verify_trees(model, b))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for name in ("path", "n_path", "next_token", "cached", "logits"):
            assert torch.equal(getattr(g, name), getattr(w, name)), name
    for a, b in zip(_caches(model), after):
        assert torch.equal(a, b)


def test_trees_reach_the_end_of_the_context():
    """A short tree at the cache's last positions beside a long one elsewhere."""
    from sophia_amd.runtime import pack_trees, verify_trees
    model = _model()
    _prefill(model, [0, 1], [398, 5])
    trees = pack_trees(model, [([1, 2, 3], [-1, 0, 0]), ([4] * 64, [-1] + [0] * 63)], [0, 1], [398, 5])
    out = verify_trees(model, trees)
    assert out.cached.tolist()[0] in (399, 400)
    mla = next(layer.attn for layer in model.layers if layer.layer_type == "mla")
    assert mla.latent_cache[0, :int(out.cached[0])].abs().sum(-1).gt(0).all()
    with pytest.raises(ValueError, match="max_seq_len"):
        pack_trees(model, [([1, 2, 3], [-1, 0, 1])], [0], [398])


def test_tree_step_refusals():
    from sophia_amd.runtime import pack_trees
    model = _model()
    ok = ([1, 2], [-1, 0])
    for trees, slots, cached in (([ok], [0, 1], [3]), ([ok, ok], [1, 1], [3, 3]), ([ok], [6], [3]), ([ok], [-1], [3]), ([ok], [0], [-1]),
                                 ([([1], [-1, 0])], [0], [3]), ([([], [])], [0], [3]), ([([1] * 65, [-1] + [0] * 64)], [0], [3]),
                                 ([([1, 2], [-1, 1])], [0], [3]), ([([1, 2], [0, 0])], [0], [3]), ([([1, 512], [-1, 0])], [0], [3])):
        with pytest.raises(ValueError):
            pack_trees(model, trees, slots, cached)
    with pytest.raises(ValueError, match="max_seq_len"):
        model.forward_tree(pack_trees(model, [ok], [0], [399]))
    with pytest.raises(ValueError, match="empty"):
        model.forward_tree(pack_trees(model, [], [], []))
    with pytest.raises(RuntimeError, match="GPU"):
        trees = pack_trees(model, [ok], [0], [3])
        trees.token_ids = trees.token_ids.cpu()
        model.forward_tree(trees)
