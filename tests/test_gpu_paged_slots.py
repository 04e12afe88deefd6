"""Slots with latents in pages beside slots with their own: what is refused of the former runs on the latter as if there were no pages,
and a prompt's snapshot goes on in another slot that shares its pages."""

from __future__ import annotations

import pytest
import torch

from test_gpu_paged_serving import _setup
from test_gpu_runtime import REL_TOL, _i64, _np, _oracle_last, _rel

pytestmark = pytest.mark.gpu


def test_drafts_run_beside_paged_slots_and_not_on_them():
    from sophia_amd.runtime import pack_trees
    model, _, slots, pages, dev = _setup(21)
    ids = torch.randint(0, 512, (30,), generator=torch.Generator().manual_seed(22)).to(dev)
    tree = ([3, 4, 5], [-1, 0, 0])
    with torch.no_grad():
        s = slots.allocate(2)
        model.forward_step(prefill_ids=ids, prefill_lens=[30], prefill_slots=s[:1].contiguous())
        want = model.forward_tree(pack_trees(model, [tree], s[:1], [30])).logits.clone()
        paged = int(s[1])
        pages.reserve(paged, 40)
        model.forward_step(prefill_ids=ids, prefill_lens=[30], prefill_slots=s[1:].contiguous(), pages=pages)
        with pytest.raises(RuntimeError, match=rf"slots \[{paged}\] are in pages"):
            pack_trees(model, [tree, tree], s, [30, 30])
        trees = pack_trees(model, [tree], s[:1], [30])
        assert torch.equal(model.forward_tree(trees).logits, want)
        # captured while there are pages: the slots are not read
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            model.forward_tree(trees)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = model.forward_tree(trees).logits
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
        trees.slots.fill_(paged)
        with pytest.raises(RuntimeError, match="in pages"):
            model.forward_tree(trees)
        pages.release([paged])
        model.forward_tree(trees)


def test_a_prompts_snapshot_goes_on_where_its_pages_are_shared():
    model, params, slots, pages, dev = _setup(23)
    gen = torch.Generator().manual_seed(24)
    prompt, nxt = torch.randint(0, 512, (53,), generator=gen), torch.randint(0, 512, (1,), generator=gen)
    with torch.no_grad():
        s = slots.allocate(3)
        one, two, own = s.tolist()
        pages.reserve(one, 60)
        model.forward_step(prefill_ids=torch.cat([prompt, prompt[:20]]).to(dev), prefill_lens=[53, 20], prefill_slots=s[[0, 2]].contiguous(),
                           pages=pages)
        with pytest.raises(RuntimeError, match="in pages"):
            model.cache_dump(slots=s[:1])
        snap = model.cache_dump(slots=s[:1], latents=False)
        # the first slot goes on; another one takes the prompt up where it was
        model.forward_step(decode_ids=prompt[:1].to(dev), decode_slots=s[:1].contiguous(), decode_pos=_i64([53], dev), max_decode_len=54,
                           pages=pages)
        pages.share(one, two, 53)
        pages.reserve(two, 54)
        model.cache_load(snap, slots=s[1:2])
        out = model.forward_step(decode_ids=nxt.to(dev), decode_slots=s[1:2].contiguous(), decode_pos=_i64([53], dev), max_decode_len=54,
                                 pages=pages)
        assert _rel(_np(out[0]), _oracle_last(params, torch.cat([prompt, nxt]).numpy())) < REL_TOL
        # a slot without pages has its own latents in its snapshot
        assert model.cache_dump(slots=s[2:], cache_pos=20).layers[3].latent.shape[1] == 20
