"""Host side of ``runtime.beam_search`` (CPU, no kernel): which tokens it gives to the model, with the step, the choice and the fork
replaced by functions of the test."""

from __future__ import annotations

import pytest
import torch

VOCAB = 64


class Search:
    """A model, slots and pages on the CPU.  ``choose(t)`` -> (scores, parents, tokens) of the t-th choice, or None: token t + 1 and on."""

    def __init__(self, monkeypatch, choose=None):
        from sophia_amd import ops
        from sophia_amd.config import ModelArgs
        from sophia_amd.decoder import Transformer
        from sophia_amd.runtime import PagedLatents, SlotAllocator
        torch.manual_seed(0)
        self.model = Transformer(ModelArgs(vocab_size=VOCAB, n_layers=4, ffn_hidden=64, mla_q_rank=64, mla_kv_rank=32, dim=128,
                                           num_heads=1, max_seq_len=64, max_batch_size=8))
        self.slots, self.pages = SlotAllocator(self.model), PagedLatents(self.model, 40, page_size=16)
        self.fed, self.choices, self.choose = [], 0, choose

        def step(*, prefill_ids=None, decode_ids=None, prefill_lens=(), **kw):
            self.fed.append(prefill_ids if prefill_ids is not None else decode_ids)
            return torch.zeros(len(prefill_lens) or decode_ids.numel(), VOCAB)

        def select(logits, scores, beams, *, keep, ended, pad_token):
            groups = logits.size(0) // beams
            best = None if self.choose is None else self.choose(self.choices)
            self.choices += 1
            if best is None:
                best = torch.zeros(groups, keep), torch.zeros(groups, keep).int(), torch.arange(keep).expand(groups, keep) + self.choices
            score, parent, token = best
            if ended is not None:
                token = torch.where(torch.gather(ended.view(groups, beams), 1, parent.long().clamp(min=0)), pad_token, token)
            return score, parent, token.clone()
        monkeypatch.setattr(self.model, "forward_step", step)
        monkeypatch.setattr(self.model, "fork_slots", lambda *a, **kw: None)
        monkeypatch.setattr(ops, "beam_select", select)

    def __call__(self, prompts, **kw):
        from sophia_amd.runtime import beam_search
        return beam_search(self.model, self.slots, self.pages, prompts, **kw)


@pytest.mark.parametrize("pad", [VOCAB, VOCAB + 7, 1 << 40, -3, 0, 9])
def test_a_pad_token_is_for_the_output_alone(pad, monkeypatch):
    """Any number, such as one that no token has: the model is given tokens of its vocabulary."""
    end = 5
    ids = [torch.tensor([[end, 8]]), torch.tensor([[3, end]]), torch.tensor([[2, 1]])]
    search = Search(monkeypatch, lambda t: (torch.zeros(1, 2), torch.tensor([[0, 1]]).int(), ids[t]))
    got = search([[1, 2, 3]], beams=2, max_new=3, end_token=end, pad_token=pad)
    assert got.tokens.tolist() == [[[end, pad, pad], [8, end, pad]]] and got.ended.tolist() == [[True, True]]
    assert len(search.fed) == 3
    for ids in search.fed:
        assert int(ids.min()) >= 0 and int(ids.max()) < VOCAB


def test_places_without_a_beam_are_fed_a_token_of_the_vocabulary(monkeypatch):
    none = torch.tensor([[0.0, -torch.inf]]), torch.tensor([[0, -1]]).int(), torch.tensor([[4, -1]])
    search = Search(monkeypatch, lambda t: none)
    got = search([[1]], beams=2, max_new=3)
    assert got.tokens.tolist() == [[[4, 4, 4], [-1, -1, -1]]]
    assert all(int(ids.min()) >= 0 for ids in search.fed)


@pytest.mark.parametrize("prompt", [[VOCAB], [1, -1, 2], [3, 1 << 40]])
def test_prompts_outside_the_vocabulary_are_refused(prompt, monkeypatch):
    search = Search(monkeypatch)
    with pytest.raises(ValueError, match="vocabulary"):
        search([[1, 2], prompt], beams=2, max_new=2)
    assert not search.fed and search.slots.in_use == 0 and search.pages.pages_free == 40


@pytest.mark.parametrize("change", [lambda x: torch.cat([x, x], -1), lambda x: x[:, :8], lambda x: x[:1], lambda x: x[None]])
def test_adjusted_logits_of_another_shape_are_refused(change, monkeypatch):
    """Wider ones would be tokens that the model does not have."""
    search = Search(monkeypatch)
    with pytest.raises(ValueError, match="adjust"):
        search([[1, 2], [3]], beams=2, max_new=3, adjust=lambda logits, tokens: change(logits))
    assert search.choices == 0 and search.slots.in_use == 0 and search.pages.pages_free == 40
