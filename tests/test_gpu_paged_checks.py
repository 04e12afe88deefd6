"""What the operators on paged latents, beams and cache moves refuse of device tensors, before any launch, and their calls on
another stream, in a captured graph, and on a table whose pools are elsewhere."""

from __future__ import annotations

import pytest
import torch

import paged_ref as ref
from test_gpu_paged_ops import BF, F32, SCALE

pytestmark = pytest.mark.gpu


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _i64(*v):
    return torch.tensor(v, dtype=torch.int64, device="cuda")


def _z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


# Each builds its arguments on the GPU: 3 rows of 2 sequences, 4 heads of rank 32, 6 pages of 16, a table of 2 x 3.
def _attn_args():
    return dict(qa=_z(3, 4, 32), pages=_z(6, 16, 32), table=_i32(0, 1, 2, 3, 4, 5).view(2, 3), cu_seqlens=_i32(0, 1, 3), kv_len=_i64(5, 20),
                scale=0.1, max_new=2)


def _norm_args():
    return dict(q_lat=_z(3, 64), kv_lat=_z(3, 32), q_norm_weight=_z(64, dtype=F32), q_eps=1e-5, kv_norm_weight=_z(32, dtype=F32), kv_eps=1e-5,
                pages=_z(6, 16, 32), table=_i32(0, 1, 2, 3, 4, 5).view(2, 3), cu_seqlens=_i32(0, 1, 3), kv_len=_i64(5, 20))


def _beam_args():
    return dict(logits=_z(4, 50), scores=_z(4, dtype=F32), beams=2)


def _fork_args():
    return dict(src=_i32(0, 1), dst=_i32(1, 0), kda=[(_z(2, 12, 3, dtype=F32), _z(2, 1, 8, 8, dtype=F32)) for _ in range(2)],
                mla=[_z(2, 40, 32, dtype=F32) for _ in range(2)], pools=[_z(6, 16, 32) for _ in range(2)],
                table=_i32(0, 1, 2, 3, 4, 5).view(2, 3), cached=_i64(5, 20))


PAGES = [
    (dict(pages=lambda a: a["pages"].cpu()), "pages"), (dict(pages=lambda a: a["pages"].float()), "dtype"),
    (dict(pages=lambda a: a["pages"].transpose(0, 1)), "dense"), (dict(pages=lambda a: a["pages"][..., :16]), "dense"),
    (dict(pages=lambda a: _z(6, 12, 32)), "page_size"), (dict(pages=lambda a: _z(6, 16, 64)), "rank"), (dict(pages=lambda a: a["pages"][0]), "pages"),
    (dict(table=lambda a: a["table"].long()), "table"), (dict(table=lambda a: a["table"].cpu()), "table"),
    (dict(table=lambda a: a["table"].t()), "table"), (dict(table=lambda a: a["table"][0]), "table"), (dict(table=lambda a: a["table"][:1]), "rows"),
    (dict(cu_seqlens=lambda a: a["cu_seqlens"].long()), "cu_seqlens"), (dict(cu_seqlens=lambda a: a["cu_seqlens"].cpu()), "cu_seqlens"),
    (dict(cu_seqlens=lambda a: a["cu_seqlens"][:0]), "cu_seqlens"), (dict(cu_seqlens=lambda a: a["cu_seqlens"][:2]), "kv_len"),
    (dict(kv_len=lambda a: a["kv_len"].int()), "kv_len"), (dict(kv_len=lambda a: a["kv_len"].cpu()), "kv_len"),
    (dict(kv_len=lambda a: a["kv_len"].repeat_interleave(2)[::2]), "kv_len"),
    (dict(slots=lambda a: _i64(0, 1)), "slots"), (dict(slots=lambda a: _i32(0)), "slots"), (dict(slots=lambda a: _i32(0, 1).cpu()), "slots")]


def _refused(fn, args, change, word):
    args.update({k: v(args) for k, v in change.items()})
    before = {k: t.clone() for k, t in args.items() if isinstance(t, torch.Tensor) and t.is_cuda}
    with pytest.raises((RuntimeError, ValueError), match=word):
        fn(**args)
    for k, t in before.items():
        assert torch.equal(args[k], t), k


@pytest.mark.parametrize("change,word", PAGES + [
    (dict(qa=lambda a: a["qa"].half()), "dtype"), (dict(qa=lambda a: a["qa"][0]), "qa"), (dict(qa=lambda a: a["qa"].transpose(1, 2)), "qa"),
    (dict(qa=lambda a: a["qa"].transpose(0, 1)), "qa"), (dict(qa=lambda a: _z(3, 4, 48), pages=lambda a: _z(6, 16, 48)), "rank"),
    (dict(qa=lambda a: _z(3, 129, 32)), "heads"), (dict(qa=lambda a: _z(3, 128 + 4)[:, 4:].view(3, 4, 32)), "strides|aligned"),
    (dict(out=lambda a: a["qa"].float()), "out"), (dict(out=lambda a: _z(2, 4, 32)), "out"), (dict(out=lambda a: a["qa"].cpu()), "out"),
    (dict(max_new=lambda a: 0), "max_new"), (dict(scale=lambda a: float("inf")), "scale"), (dict(splits=lambda a: -1), "splits")])
def test_attention_refuses(change, word):
    from sophia_amd import ops
    _refused(ops.mla_paged_attn, _attn_args(), change, word)


@pytest.mark.parametrize("change,word", PAGES + [
    (dict(q_lat=lambda a: a["q_lat"].float()), "dtype"), (dict(kv_lat=lambda a: a["kv_lat"][:2]), "rows"),
    (dict(q_lat=lambda a: a["q_lat"].t()), "q_lat|rows"), (dict(kv_lat=lambda a: a["kv_lat"].cpu()), "kv_lat"),
    (dict(q_norm_weight=lambda a: a["q_norm_weight"][:60]), "q_norm_weight"), (dict(kv_norm_weight=lambda a: a["q_norm_weight"]), "kv_norm_weight")])
def test_norms_refuse(change, word):
    from sophia_amd import ops
    _refused(ops.mla_latent_norms_paged, _norm_args(), change, word)


@pytest.mark.parametrize("change,word", [
    (dict(logits=lambda a: a["logits"][0]), "logits"), (dict(logits=lambda a: a["logits"].half()), "bfloat16"),
    (dict(logits=lambda a: a["logits"].t()), "logits|rows"), (dict(logits=lambda a: a["logits"][:3]), "groups"), (dict(beams=lambda a: 0), "beams"),
    (dict(beams=lambda a: 65), "beams"), (dict(keep=lambda a: 0), "keep"), (dict(keep=lambda a: 65), "keep"),
    (dict(scores=lambda a: a["scores"].double()), "scores"), (dict(scores=lambda a: a["scores"][:3]), "scores"),
    (dict(scores=lambda a: a["scores"].cpu()), "scores"), (dict(ended=lambda a: _i32(0, 0, 0, 0)), "ended"),
    (dict(ended=lambda a: _z(3, dtype=torch.bool)), "ended")])
def test_beams_refuse(change, word):
    from sophia_amd import ops
    _refused(ops.beam_select, _beam_args(), change, word)


@pytest.mark.parametrize("change,word", [
    (dict(src=lambda a: a["src"].long()), "src"), (dict(dst=lambda a: a["dst"].cpu()), "dst"), (dict(dst=lambda a: a["dst"][:1]), "entries"),
    (dict(src=lambda a: _i32(*[0] * 4097), dst=lambda a: _i32(*[0] * 4097)), "4096"),
    (dict(kda=lambda a: [(a["kda"][0][0], a["kda"][0][1].to(BF))]), "state"), (dict(kda=lambda a: [a["kda"][0], (None, a["kda"][1][1])]), "conv_state"),
    (dict(kda=lambda a: [(a["kda"][0][0], _z(3, 1, 8, 8, dtype=F32))]), "slots"), (dict(kda=lambda a: [(None, _z(2, 1, 5, 5, dtype=F32))]), "multiples"),
    (dict(kda=lambda a: [a["kda"][0], a["kda"][0]]), "of its own"), (dict(mla=lambda a: [a["mla"][0]] * 2), "of its own"),
    (dict(pools=lambda a: [a["pools"][0]] * 2), "of its own"), (dict(mla=lambda a: [a["mla"][0], a["mla"][1][:, :30]]), "latent_cache"),
    (dict(mla=lambda a: [t.to(BF) for t in a["mla"]]), "latent"), (dict(mla=lambda a: [_z(3, 40, 32, dtype=F32)]), "slots"),
    (dict(mla=lambda a: [_z(2, 40, 64, dtype=F32)]), "rank"), (dict(pools=lambda a: [a["pools"][0], a["pools"][1][:5]]), "pool 1"),
    (dict(pools=lambda a: [a["pools"][0], a["pools"][1].cpu()]), "pools"), (dict(pools=lambda a: [_z(6, 12, 32)]), "page_size"),
    (dict(pools=lambda a: []), "page_size"), (dict(page_size=lambda a: 32), "page_size"),
    (dict(pools=lambda a: [], page_size=lambda a: 12), "page_size"), (dict(table=lambda a: None), "table"),
    (dict(pools=lambda a: [], table=lambda a: None, page_size=lambda a: 16), "table"), (dict(table=lambda a: a["table"][:1]), "row"),
    (dict(table=lambda a: a["table"].long()), "table"), (dict(cached=lambda a: None), "cached"), (dict(cached=lambda a: _i64(5)), "cached"),
    (dict(cached=lambda a: _i32(5, 20)), "cached")])
def test_fork_refuses(change, word):
    from sophia_amd import ops
    _refused(ops.cache_fork, _fork_args(), change, word)


@pytest.mark.parametrize("change,word", [
    (dict(src=lambda a: a["src"].long()), "src"), (dict(dst=lambda a: a["dst"][:1]), "entries"), (dict(pools=lambda a: [a["pools"][0]] * 2), "of its own"),
    (dict(pools=lambda a: [a["pools"][0], a["pools"][1].float()]), "pool 1"), (dict(pools=lambda a: [a["pools"][0].half()]), "bfloat16"),
    (dict(pools=lambda a: [_z(6, 1, 36)]), "multiples"), (dict(pools=lambda a: [a["pools"][0].transpose(0, 1)]), "dense")])
def test_page_copy_refuses(change, word):
    from sophia_amd import ops
    args = {k: v for k, v in _fork_args().items() if k in ("src", "dst", "pools")}
    _refused(ops.page_copy, args, change, word)


@pytest.mark.parametrize("n", [1, 3, 70, 600])
def test_fork_of_a_table_whose_pools_are_elsewhere(n):
    """The ids of full pages become shared as they do beside pools; the pool's page sizes only say how many."""
    from sophia_amd import ops
    gen = torch.Generator().manual_seed(n)
    slots, width = n + 4, 9
    src, dst = torch.randint(slots, (n,), generator=gen).int(), torch.randperm(slots, generator=gen)[:n].int()
    table = torch.randperm(slots * width, generator=gen).view(slots, width).int()
    state, cached = torch.randn(slots, 1, 8, 8, generator=gen), torch.randint(0, 400, (n,), generator=gen)
    dt, ds = table.cuda(), state.cuda()
    ops.cache_fork(src.cuda(), dst.cuda(), kda=[(None, ds)], table=dt, cached=cached.cuda(), page_size=32)
    want, _ = ref.fork_pages(table, [torch.zeros(1, 32, 8)], src.tolist(), dst.tolist(), cached, slots)
    assert torch.equal(dt.cpu(), want) and torch.equal(ds.cpu(), ref.moved(state, src.tolist(), dst.tolist()))


# ------------------------------------------------------------------ streams and graphs
def _step(c, qa, q, kv, w, pages, table, cu, kv_len, slots, state, src, dst, cached, logits, scores):
    """Norms into the pages, attention, beams, a fork: in the order of a step."""
    from sophia_amd import ops
    ops.mla_latent_norms_paged(q, kv, w[0], 1e-5, w[1], 1e-5, pages, table, cu, kv_len, slots=slots)
    out = ops.mla_paged_attn(qa, pages, table, cu, kv_len, SCALE, max_new=max(c.news), slots=slots)
    best = ops.beam_select(logits, scores, 4)
    ops.cache_fork(src, dst, kda=[(None, state)], pools=[pages], table=table, cached=cached)
    return (out, *best)


def _inputs(c):
    gen = torch.Generator().manual_seed(11)
    q, kv = (torch.randn(c.rows, n, generator=gen).to(c.qa.dtype) for n in (384, 128))
    w = [torch.rand(n, generator=gen) + 0.5 for n in (384, 128)]
    pages = torch.nan_to_num(c.pages)
    slots = c.table.size(0)
    state = torch.randn(slots, 2, 128, 128, generator=gen)
    # two slots of sequences change places, at counts within their pages
    src, dst = c.slots[[0, 1]], c.slots[[1, 0]]
    cached = torch.tensor([min(c.lens[0], c.lens[1]) - 1] * 2)
    logits, scores = torch.randn(8, 1000, generator=gen), -torch.rand(8, generator=gen)
    return [c.qa, q, kv, w, pages, c.table, c.cu, c.kv_len, c.slots, state, src, dst, cached, logits, scores]


def _cuda(x):
    return [t.cuda() for t in x] if isinstance(x, list) else x.cuda()


def _case():
    return ref.Paged([1, 5, 40, 1], [700, 690, 100, 9], seed=4)


def test_steps_on_two_streams_at_once_are_those_of_one():
    c = _case()
    want_in = [_cuda(t) for t in _inputs(c)]
    want = [t.cpu() for t in _step(c, *want_in)]
    want_in = [want_in[i].cpu() for i in (1, 2, 4, 5, 9)]
    batches = [[_cuda(t) for t in _inputs(c)] for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in batches]
    outs = []
    for s, b in zip(streams, batches):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(_step(c, *b))
    torch.cuda.synchronize()
    for out, b in zip(outs, batches):
        assert all(torch.equal(o.cpu(), w) for o, w in zip(out, want))
        assert all(torch.equal(b[i].cpu(), w) for i, w in zip((1, 2, 4, 5, 9), want_in))


def test_two_captured_steps_replayed_in_turn_are_the_eager_ones():
    """Each graph has workspaces of its own; eager work and other graphs between the replays change nothing."""
    cases = [_case(), ref.Paged([1, 1, 1], [4000, 2100, 64], seed=5)]
    fresh = [[_cuda(t) for t in _inputs(c)] for c in cases]
    want = []
    for c in cases:
        dev = [_cuda(t) for t in _inputs(c)]
        out = _step(c, *dev)
        want.append([t.clone() for t in out] + [dev[i].clone() for i in (1, 2, 4, 5, 9)])
    live = [[[u.clone() for u in t] if isinstance(t, list) else t.clone() for t in f] for f in fresh]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for c, b in zip(cases, live):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            g.capture_begin()
            outs.append(_step(c, *b))
            g.capture_end()
        graphs.append(g)
    torch.cuda.current_stream().wait_stream(side)
    for turn in range(4):
        for g, b, f in zip(graphs, live, fresh):
            for t, u in zip(b, f):
                for x, y in zip(t, u) if isinstance(t, list) else [(t, u)]:
                    x.copy_(y)
            g.replay()
        if turn % 2:
            torch.cuda.synchronize()
            _step(cases[0], *[_cuda(t) for t in _inputs(cases[0])])      # eager work between
        for out, b, w in zip(outs, live, want):
            got = list(out) + [b[i] for i in (1, 2, 4, 5, 9)]
            assert all(torch.equal(x, y) for x, y in zip(got, w)), turn
