"""Host bookkeeping of ``runtime.PagedLatents`` (CPU tensors, no kernel launch)."""

from __future__ import annotations

import pytest
import torch


def _pages(n=12, **over):
    from sophia_amd.config import ModelArgs
    from sophia_amd.decoder import Transformer
    from sophia_amd.runtime import PagedLatents
    torch.manual_seed(0)
    model = Transformer(ModelArgs(vocab_size=64, n_layers=4, ffn_hidden=64, mla_q_rank=64, mla_kv_rank=32, dim=128, num_heads=1,
                                  max_seq_len=64, max_batch_size=2))
    return PagedLatents(model, n, **{**dict(page_size=16), **over})


def test_reserve_share_release():
    p = _pages()
    assert p.max_len == 64 and list(p.table.shape) == [2, 4] and len(p.pools) == 1 and p.pages_free == 12
    p.reserve(0, 33)
    assert p.held(0) == [0, 1, 2] and p.table[0].tolist() == [0, 1, 2, -1]
    p.reserve(0, 20)                                  # fewer: as it was
    p.reserve(0, 49)
    assert p.held(0) == [0, 1, 2, 3] and p.pages_free == 8
    p.share(0, 5, 32)                                 # whole pages: none is copied; a row that was not there
    assert p.table[5].tolist() == [0, 1, -1, -1] and p.pages_free == 8 and p.table.size(0) == 6
    p.reserve(5, 40)
    assert p.held(5) == [0, 1, 4]
    p.release([0])
    assert p.pages_free == 9 and p.table[0].tolist() == [-1] * 4 and p.held(0) == []
    p.release(torch.tensor([5, 1]))                   # (slot 1 holds nothing)
    assert p.pages_free == 12 and int(p.table.max()) == -1
    p.reserve(1, 64, first=20)
    assert p.table[1].tolist() == [-1, 0, 1, 2]
    p.reserve(1, 0)
    p.reserve(1, 16)
    assert p.table[1].tolist() == [3, 0, 1, 2]


def test_nothing_is_taken_where_there_is_not_enough():
    p = _pages(3)
    p.reserve(0, 32)
    with pytest.raises(RuntimeError, match="2 pages needed, 1 free"):
        p.reserve(1, 17)
    assert p.held(1) == [] and p.pages_free == 1
    p.reserve(1, 1)
    with pytest.raises(RuntimeError, match="1 page needed"):
        p.share(0, 3, 20)
    assert p.held(3) == [] and p._holders == [1, 1, 1]


@pytest.mark.parametrize("call,word", [
    (lambda p: p.reserve(0, 65), "at most 64"), (lambda p: p.reserve(0, -1), "at most"), (lambda p: p.reserve(-1, 5), "slots"),
    (lambda p: p.reserve(0, 5, first=-1), "first"), (lambda p: p.share(0, 1, 20), "fewer"), (lambda p: p.share(0, 1, 99), "at most"),
    (lambda p: p.release([1, 1]), "twice")])
def test_refusals(call, word):
    p = _pages()
    with pytest.raises(ValueError, match=word):
        call(p)
    p.reserve(1, 5)
    p.reserve(0, 64)
    with pytest.raises(ValueError, match="holds pages"):
        p.share(0, 1, 20)


def test_a_slot_whose_pages_a_fork_has_changed_is_not_shared():
    p = _pages()
    p.reserve(0, 40)
    p.reserve(1, 40)
    p.table[0, 1] = p.table[1, 1]                     # (as a fork does on the device)
    p.share(0, 2, 16)
    with pytest.raises(ValueError, match="fork"):
        p.share(0, 3, 32)
    assert p.held(3) == [] and p.pages_free == 6


def test_a_fork_under_a_remembered_mask_is_refused():
    from sophia_amd.config import ModelArgs
    from sophia_amd.decoder import Transformer
    model = Transformer(ModelArgs(vocab_size=64, n_layers=4, ffn_hidden=64, mla_q_rank=64, mla_kv_rank=32, dim=128, num_heads=1,
                                  max_seq_len=64, max_batch_size=2))
    model.layers[3].attn._prompt_mask = torch.ones(1, 8, dtype=torch.bool)
    i32 = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="padded"):
        model.fork_slots(i32, i32, torch.zeros(1, dtype=torch.int64))


def test_construction_refuses():
    for bad in (dict(n=0), dict(page_size=0), dict(page_size=24), dict(page_size=1 << 17), dict(max_len=0)):
        with pytest.raises(ValueError):
            _pages(**bad)


def test_compact_of_pages_in_their_places_moves_nothing():
    p = _pages()
    p.reserve(0, 40)
    assert p.compact() == 3 and p.held(0) == [0, 1, 2]
