"""Latents in pages and beams through the decoder: steps over pages equal the oracle and the slots' own caches, sequences share
pages, beams carry their caches with them, a captured step of beam search replays.

Logits are held to those of test_gpu_runtime.py: max|y - y_ref| / max|y_ref| <= 2e-2 of the float64 oracle (fp32 model), bf16
against the same step over the slots' own caches at 2e-2 (its prefill expands keys and values, rounded to bf16, and its decode
attends over the same latents).
"""

from __future__ import annotations

import pytest
import torch

from test_gpu_runtime import REL_TOL, _dev, _i32, _i64, _model, _np, _oracle_last, _rel

pytestmark = pytest.mark.gpu


def _setup(seed, *, dtype=None, page=16, n_pages=200, **over):
    from sophia_amd.runtime import PagedLatents, SlotAllocator
    dev = _dev()
    model, params = _model(dev, seed=seed, **over)
    if dtype is not None:
        model.cast_weights_(dtype)
    return model, params, SlotAllocator(model), PagedLatents(model, n_pages, page_size=page, max_len=2600), dev


def test_a_prompt_in_pieces_ragged_prompts_and_decodes_match_the_oracle():
    model, params, slots, pages, dev = _setup(1)
    gen = torch.Generator().manual_seed(2)
    seqs = [torch.randint(0, 512, (n,), generator=gen) for n in (150, 37, 5, 64)]
    with torch.no_grad():
        s = slots.allocate(4)
        for slot, q in zip(s.tolist(), seqs):
            pages.reserve(slot, len(q) + 3)
        # the first prompt in pieces of 70, 1 and 79, the others whole or beside them, then decode steps
        model.forward_step(prefill_ids=torch.cat([seqs[0][:70], seqs[1]]).to(dev), prefill_lens=[70, 37], prefill_slots=s[:2],
                           pages=pages)
        model.forward_step(prefill_ids=torch.cat([seqs[0][70:71], seqs[2]]).to(dev), prefill_lens=[1, 5], prefill_pos=[70, 0],
                           prefill_slots=s[[0, 2]].contiguous(), pages=pages)
        last = model.forward_step(prefill_ids=torch.cat([seqs[0][71:], seqs[3]]).to(dev), prefill_lens=[79, 64], prefill_pos=[71, 0],
                                  prefill_slots=s[[0, 3]].contiguous(), pages=pages, all_logits=True)
        assert _rel(_np(last[78]), _oracle_last(params, seqs[0].numpy())) < REL_TOL
        assert _rel(_np(last[100]), _oracle_last(params, seqs[3][:22].numpy())) < REL_TOL
        for t in range(3):
            nxt = torch.randint(0, 512, (4,), generator=gen)
            pos = [len(q) for q in seqs]
            out = model.forward_step(decode_ids=nxt.to(dev), decode_slots=s, decode_pos=_i64(pos, dev), max_decode_len=max(pos) + 1,
                                     pages=pages)
            seqs = [torch.cat([q, nxt[i:i + 1]]) for i, q in enumerate(seqs)]
            for i, q in enumerate(seqs):
                assert _rel(_np(out[i]), _oracle_last(params, q.numpy())) < REL_TOL
    # none of it went into the slots' own caches
    assert all(float(m.latent_cache.abs().max()) == 0.0 for m in pages.pools)


def test_a_bf16_step_over_pages_equals_one_over_the_slots_caches():
    model, _, slots, pages, dev = _setup(3, dtype=torch.bfloat16, num_heads=16, mla_kv_rank=128, page=64)
    gen = torch.Generator().manual_seed(4)
    lens = [300, 33, 90]
    ids = torch.randint(0, 512, (sum(lens),), generator=gen).to(dev)
    with torch.no_grad():
        outs = []
        for where in (None, pages):
            s = slots.allocate(3)
            if where is not None:
                for slot, n in zip(s.tolist(), lens):
                    pages.reserve(slot, n + 4)
            got = [model.forward_step(prefill_ids=ids, prefill_lens=lens, prefill_slots=s, pages=where, all_logits=True)]
            for t in range(3):
                got.append(model.forward_step(decode_ids=ids[t::90][:3], decode_slots=s, decode_pos=_i64([n + t for n in lens], dev),
                                              max_decode_len=304, pages=where))
            outs.append(got)
        for a, b in zip(*outs):
            assert _rel(_np(a), _np(b)) < 2e-2


def test_shared_prefix_moved_pages_and_freed_ones():
    """A second sequence goes on from the first 53 tokens of another one, pages are moved together in between, and all come back."""
    model, params, slots, pages, dev = _setup(5, n_pages=40)
    gen = torch.Generator().manual_seed(6)
    a, b = (torch.randint(0, 512, (n,), generator=gen) for n in (53, 9))
    nxt = torch.randint(0, 512, (2,), generator=gen)
    with torch.no_grad():
        s = slots.allocate(3)
        one, two, three = s.tolist()
        pages.reserve(three, 200)
        pages.reserve(one, 53)
        model.forward_step(prefill_ids=a.to(dev), prefill_lens=[53], prefill_slots=s[:1], pages=pages)
        pages.share(one, two, 53)
        assert pages.held(two)[:3] == pages.held(one)[:3] and pages.held(two)[3] != pages.held(one)[3]
        model.fork_slots(s[:1], s[1:2], _i64([0], dev))                    # the KDA states; no latent of the slots' own caches
        pages.release([three])
        assert pages.compact() == 5 and pages.pages_free == 35 and max(pages.held(one) + pages.held(two)) == 4
        pages.reserve(two, 53 + 9 + 1)
        pages.reserve(one, 54)
        out = model.forward_step(prefill_ids=b.to(dev), prefill_lens=[9], prefill_pos=[53], prefill_slots=s[1:2], decode_ids=nxt[:1].to(dev),
                                 decode_slots=s[:1], decode_pos=_i64([53], dev), max_decode_len=54, pages=pages)
        assert _rel(_np(out[0]), _oracle_last(params, torch.cat([a, b]).numpy())) < REL_TOL
        assert _rel(_np(out[1]), _oracle_last(params, torch.cat([a, nxt[:1]]).numpy())) < REL_TOL
        pages.release([one])
        out = model.forward_step(decode_ids=nxt[1:].to(dev), decode_slots=s[1:2], decode_pos=_i64([62], dev), max_decode_len=63, pages=pages)
        assert _rel(_np(out[0]), _oracle_last(params, torch.cat([a, b, nxt[1:]]).numpy())) < REL_TOL
        pages.release([two])
        assert pages.pages_free == 40 and int(pages.table.max()) == -1


def test_fork_slots_without_pages_takes_the_latents_along():
    model, params, slots, _, dev = _setup(7)
    gen = torch.Generator().manual_seed(8)
    a = torch.randint(0, 512, (40,), generator=gen)
    nxt = torch.randint(0, 512, (3,), generator=gen)
    with torch.no_grad():
        s = slots.allocate(3)
        model.forward_step(prefill_ids=a.to(dev), prefill_lens=[40], prefill_slots=s[:1])
        model.fork_slots(s[:1].expand(2).contiguous(), s[1:].contiguous(), _i64([40, 40], dev))
        out = model.forward_step(decode_ids=nxt.to(dev), decode_slots=s, decode_pos=_i64([40] * 3, dev), max_decode_len=41)
        for i in range(3):
            assert _rel(_np(out[i]), _oracle_last(params, torch.cat([a, nxt[i:i + 1]]).numpy())) < REL_TOL


def _rescored(model, slots, pages, prompts, tokens, dev):
    """Log probabilities of each of ``tokens`` [N, B, T] after its prompt: every beam decoded by itself, in a slot of its own."""
    N, B, T = tokens.shape
    s = slots.allocate(N * B)
    lens = [len(prompts[i // B]) for i in range(N * B)]
    for slot, n in zip(s.tolist(), lens):
        pages.reserve(slot, n + T)
    ids = torch.cat([torch.tensor(prompts[i // B]) for i in range(N * B)]).to(dev)
    logits = model.forward_step(prefill_ids=ids, prefill_lens=lens, prefill_pos=[0] * (N * B), prefill_slots=s, pages=pages)
    flat, out = tokens.reshape(N * B, T), torch.zeros(N * B, T, dtype=torch.float64)
    for t in range(T):
        out[:, t] = torch.log_softmax(logits.double(), -1).gather(1, flat[:, t:t + 1].clamp(min=0))[:, 0].cpu()
        if t + 1 < T:
            logits = model.forward_step(decode_ids=flat[:, t].clamp(min=0), decode_slots=s, decode_pos=_i64([n + t for n in lens], dev),
                                        max_decode_len=max(lens) + T, pages=pages)
    pages.release(s)
    slots.release(s)
    return out.view(N, B, T)


@pytest.mark.parametrize("dtype,page", [(None, 16), (torch.bfloat16, 4)], ids=["f32", "bf16"])
def test_beams_have_the_probabilities_of_their_own_tokens(dtype, page):
    """Whatever slots, pages and states a beam has gone through, its score is that of its tokens decoded alone; it is no worse than
    greedy decoding, the beams differ, and they are sorted."""
    from sophia_amd.runtime import beam_search
    model, _, slots, pages, dev = _setup(9, dtype=dtype, page=page, n_pages=600)
    with torch.no_grad():
        model.tok_embeddings.weight.mul_(12.0)          # (logits that differ: the output is the embedding)
    gen = torch.Generator().manual_seed(10)
    prompts = [torch.randint(0, 512, (n,), generator=gen).tolist() for n in (33, 16, 7)]
    free = pages.pages_free
    got = beam_search(model, slots, pages, prompts, beams=4, max_new=9)
    assert pages.pages_free == free and slots.in_use == 0 and not bool(got.ended.any())
    assert bool((got.scores[:, :-1] >= got.scores[:, 1:]).all())
    with torch.no_grad():
        each = _rescored(model, slots, pages, prompts, got.tokens, dev)
    # one row's logits depend on the rows beside it by roundings: 2^-8 of logits up to 40 a step in bf16, where sums are rounded
    tol = 9 * (0.02 if dtype is None else 0.3)
    assert float((each.sum(-1) - got.scores.double().cpu()).abs().max()) < tol
    for beam in got.tokens.tolist():
        assert len({tuple(t) for t in beam}) == 4
    greedy = beam_search(model, slots, pages, prompts, beams=1, max_new=9)
    assert bool((got.scores[:, 0] >= greedy.scores[:, 0] - tol).all())


def test_beams_end_and_few_tokens_leave_places_empty():
    from sophia_amd.runtime import beam_search
    model, _, slots, pages, dev = _setup(11)
    prompts = [[1, 2, 3], [7, 7]]
    end = 5

    def only(logits, tokens):
        """Tokens 4 and 5, the latter (the end) after the first one only."""
        out = torch.full_like(logits, float("-inf"))
        out[:, 4] = 0.0
        if tokens.size(1) >= 1:
            out[:, 5] = 0.0
        return out
    got = beam_search(model, slots, pages, prompts, beams=3, max_new=4, end_token=end, pad_token=9, adjust=only)
    log2 = float(torch.log(torch.tensor(2.0)))
    # 4 5, 4 4 5 and one of 4 4 4 4 / 4 4 4 5: after 0, 1 and 2 choices of two
    want = [[4, 5, 9, 9], [4, 4, 5, 9], [4, 4, 4, 4]]
    for b in range(2):
        assert got.tokens[b].tolist() == want
        assert torch.allclose(got.scores[b].cpu(), torch.tensor([-log2, -2 * log2, -3 * log2]), atol=1e-5)
        assert got.ended[b].tolist() == [True, True, False]
    one = beam_search(model, slots, pages, prompts, beams=3, max_new=1, adjust=lambda l, t: only(l, t))
    assert one.tokens[:, 0, 0].tolist() == [4, 4] and (one.tokens[:, 1:] == -1).all() and bool(torch.isinf(one.scores[:, 1:]).all())


def test_beam_search_refuses():
    from sophia_amd.runtime import PagedLatents, beam_search
    model, _, slots, pages, dev = _setup(12, n_pages=4)
    free = pages.pages_free
    for bad, word in ((dict(prompts=[[]]), "token"), (dict(prompts=[]), "token"), (dict(beams=0), "beams"), (dict(beams=65), "beams"),
                      (dict(max_new=0), "max_new"), (dict(max_new=2700), "max_seq_len")):
        with pytest.raises(ValueError, match=word):
            beam_search(model, slots, pages, **{**dict(prompts=[[1, 2]], beams=2, max_new=3), **bad})
    with pytest.raises(RuntimeError, match="pages needed"):
        beam_search(model, slots, pages, [[1] * 40], beams=4, max_new=30)
    assert slots.in_use == 0 and pages.pages_free == free
    with pytest.raises(ValueError, match="exceeds"):
        small = PagedLatents(model, 4, page_size=16, max_len=32)
        model.forward_step(prefill_ids=torch.zeros(40, dtype=torch.long, device=dev), prefill_lens=[40], prefill_slots=slots.allocate(1),
                           pages=small)


def test_a_captured_step_of_beam_search_replays():
    """One captured step, the choice, the fork and the next token's logits, against the same step run eagerly: every replay, with
    eager work and synchronisation between them, on beams whose parents change."""
    from sophia_amd import ops
    model, _, slots, pages, dev = _setup(13, dtype=torch.bfloat16, page=4)
    with torch.no_grad():
        model.tok_embeddings.weight.mul_(12.0)
    B, T = 3, 7
    prompt = torch.randint(0, 512, (21,), generator=torch.Generator().manual_seed(14)).to(dev)

    def fresh():
        s = slots.allocate(B)
        for i, slot in enumerate(s.tolist()):
            pages.reserve(slot, 21 + T + 1, first=21 if i else 0)
        logits = model.forward_step(prefill_ids=prompt, prefill_lens=[21], prefill_slots=s[:1].contiguous(), pages=pages)
        scores, parent, token = ops.beam_select(logits, torch.zeros(1, device=dev), 1, keep=B)
        model.fork_slots(s[:1].expand(B).contiguous(), s, _i64([21] * B, dev), pages=pages)
        return dict(s=s, scores=scores.reshape(-1).clone(), token=token.reshape(-1).clone(), at=_i64([21] * B, dev))

    def step(v):
        logits = model.forward_step(decode_ids=v["token"], decode_slots=v["s"], decode_pos=v["at"], max_decode_len=21 + T, pages=pages)
        scores, parent, token = ops.beam_select(logits, v["scores"], B)
        v["at"].add_(1)
        model.fork_slots(v["s"][parent.reshape(-1).long()].contiguous(), v["s"], v["at"], pages=pages)
        v["scores"].copy_(scores.reshape(-1))
        v["token"].copy_(token.reshape(-1))
        return parent

    with torch.no_grad():
        v = fresh()
        want = []
        for _ in range(T):
            parent = step(v)
            want.append((parent.clone(), v["token"].clone(), v["scores"].clone()))
        assert any(p.reshape(-1).tolist() != [0, 1, 2] for p, _, _ in want), "no beam changed its place"
        pages.release(v["s"])
        slots.release(v["s"])
        v = fresh()
        keep = {k: t.clone() for k, t in v.items()}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(v)                                   # warm-up, which moves the caches on: they are made anew
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            parent = step(v)
        pages.release(v["s"])
        slots.release(v["s"])
        again = fresh()
        assert torch.equal(again["s"], keep["s"])
        for k, t in again.items():
            v[k].copy_(t)
        for i in range(T):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(parent, want[i][0]) and torch.equal(v["token"], want[i][1]), f"replay {i}"
            assert torch.equal(v["scores"], want[i][2]), f"replay {i}"
            torch.randn(1000, device=dev).sum()
