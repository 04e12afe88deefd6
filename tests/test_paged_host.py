"""Host side of the operators on paged latents, beams and cache moves (CPU): what their entry points refuse before any launch,
size queries, and constants that the binding shares with include/sophia_pages.h."""

from __future__ import annotations

import ctypes
import os
import re

import pytest
import torch

from test_tree_host import P, _call, nat  # noqa: F401  (nat: fixture)

HEADER = open(os.path.join(os.path.dirname(__file__), "..", "include", "sophia_pages.h")).read()


def test_header_constants_match_the_binding():
    from sophia_amd import _abi
    for name in ("BEAMS", "MOVES"):
        assert int(re.search(rf"#define SOPHIA_{name} (\d+)", HEADER).group(1)) == getattr(_abi, name)


PAGES = "pages ps np size table ts tr mp slots cu kv n"
ATTN = "qa qs dt pages ps np size table ts tr mp slots cu kv n rows new len scale out os heads rank splits ws wsb st"
PAGES_OK = dict(pages=P, ps=64 * 128, np=40, size=64, table=P, ts=9, tr=4, mp=8, slots=P, cu=P, kv=P, n=3)
ATTN_OK = dict(PAGES_OK, qa=P, qs=2048, dt=1, rows=9, new=4, len=500, scale=0.1, out=P, os=2048, heads=16, rank=128, splits=1, ws=None,
               wsb=0, st=None)
BAD_PAGES = [
    (dict(size=0), "page_size"), (dict(size=48), "page_size"), (dict(size=1 << 17), "page_size"), (dict(np=-1), "n_pages"),
    (dict(ps=64 * 128 - 8), "page_stride"), (dict(ps=64 * 128 + 4), "page_stride"), (dict(ts=7), "table"), (dict(mp=-1), "table"),
    (dict(mp=1 << 24, ts=1 << 24), "table"), (dict(tr=-1), "table"), (dict(n=-1), "n_seqs"), (dict(n=70000), "n_seqs"),
    (dict(rows=-1), "rows"), (dict(rows=1 << 29), "rows"), (dict(cu=None), "NULL"), (dict(kv=None), "NULL"), (dict(table=None), "NULL"),
    (dict(pages=None), "NULL"), (dict(pages=P + 8), "aligned")]


@pytest.mark.parametrize("change,word", BAD_PAGES + [
    (dict(dt=2), "dtype"), (dict(rank=96), "rank"), (dict(heads=0), "heads"), (dict(heads=129), "heads"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(new=0), "max_new"), (dict(splits=-1), "splits"), (dict(splits=1025), "splits"),
    (dict(qs=2040), "strides"), (dict(qs=2052), "strides"), (dict(os=100), "strides"), (dict(qa=None), "NULL"), (dict(out=None), "NULL"),
    (dict(qa=P + 8), "aligned"), (dict(out=P + 2), "aligned"), (dict(splits=2), "workspace"), (dict(splits=2, ws=P, wsb=64), "workspace"),
    (dict(splits=2, ws=P + 8, wsb=1 << 30), "workspace"), (dict(rows=1 << 27, heads=128, qs=1 << 14, os=1 << 14), "rows")])
def test_attention_refuses(nat, change, word):  # noqa: F811
    rc, msg = _call(nat, "sophia_mla_paged_attn", ATTN_OK, ATTN, **change)
    assert rc == nat.SOPHIA_ERR_INVALID and word in msg, msg


def test_attention_of_nothing(nat):  # noqa: F811
    for empty in (dict(n=0), dict(rows=0)):
        assert _call(nat, "sophia_mla_paged_attn", ATTN_OK, ATTN, cu=None, qa=None, **empty)[0] == nat.SOPHIA_OK


def test_attention_workspace(nat):  # noqa: F811
    size = nat.lib().sophia_mla_paged_workspace_size
    part = 64 * (4 * 8 + 2) * 4                                    # 16 columns of rank 128
    assert size(3, 3, 1, 500, 16, 128, 1, 1) == 0
    assert size(3, 3, 1, 500, 16, 128, 1, 2) == 3 * 2 * part
    assert size(3, 3, 1, 100, 16, 128, 1, 9) == 0                  # one tile of keys
    assert size(0, 3, 1, 500, 16, 128, 1, 0) == size(3, 0, 1, 500, 16, 128, 1, 0) == 0
    # max_new past the rows is the rows
    assert size(1, 5, 5, 4000, 16, 128, 1, 4) == size(1, 5, 1 << 20, 4000, 16, 128, 1, 4) > 0
    # bounded by what fills the chip, not by the lengths
    assert size(200, 200, 1, 1 << 29, 16, 128, 1, 0) < 64 << 20 and size(4, 4000, 1000, 1 << 29, 16, 128, 1, 0) < 256 << 20


NORMS = f"q qs kvl ks rows qr kr dt qw qe kw ke {PAGES} st"
NORMS_OK = dict(PAGES_OK, q=P, qs=384, kvl=P, ks=128, rows=9, qr=384, kr=128, dt=1, qw=P, qe=1e-5, kw=P, ke=1e-5, st=None)


@pytest.mark.parametrize("change,word", BAD_PAGES + [
    (dict(dt=3), "dtype"), (dict(qr=385, qs=392), "ranks"), (dict(qr=392, qs=392), "ranks"), (dict(kr=0), "ranks"), (dict(qs=380), "strides"),
    (dict(ks=132), "strides"), (dict(q=None), "NULL"), (dict(kw=None), "NULL"), (dict(q=P + 4), "aligned"), (dict(qw=P + 4), "aligned")])
def test_norms_refuse(nat, change, word):  # noqa: F811
    rc, msg = _call(nat, "sophia_mla_latent_norms_paged", NORMS_OK, NORMS, **change)
    assert rc == nat.SOPHIA_ERR_INVALID and word in msg, msg


BEAM = "x xs dt rows vocab scores ended pad beams keep os op ot ws wsb st"
BEAM_OK = dict(x=P, xs=1000, dt=1, rows=8, vocab=1000, scores=P, ended=P, pad=0, beams=4, keep=8, os=P, op=P, ot=P, ws=P, wsb=1 << 20, st=None)


@pytest.mark.parametrize("change,word", [
    (dict(dt=2), "dtype"), (dict(vocab=0), "vocab"), (dict(vocab=1 << 29, xs=1 << 30), "vocab"), (dict(beams=0), "beams"),
    (dict(beams=65), "beams"), (dict(keep=0), "keep"), (dict(keep=65), "keep"), (dict(rows=9), "rows"), (dict(rows=-4), "rows"),
    (dict(rows=65536), "rows"), (dict(xs=999), "stride"), (dict(x=None), "NULL"), (dict(scores=None), "NULL"), (dict(ot=None), "NULL"),
    (dict(ws=None), "workspace"), (dict(wsb=16), "workspace"), (dict(ws=P + 4), "workspace")])
def test_beams_refuse(nat, change, word):  # noqa: F811
    rc, msg = _call(nat, "sophia_beam_select", BEAM_OK, BEAM, **change)
    assert rc == nat.SOPHIA_ERR_INVALID and word in msg, msg


def test_beams_of_nothing(nat):  # noqa: F811
    assert _call(nat, "sophia_beam_select", BEAM_OK, BEAM, rows=0, x=None, ws=None)[0] == nat.SOPHIA_OK
    assert nat.lib().sophia_beam_select_workspace_size(0, 1000, 8) == 0


FORK = "src dst cached n slots states se convs ce nk mla ss seq nm pools ps np size npl table ts mp rank dt ws wsb st"


def _list(*addresses):
    return (ctypes.c_void_p * max(len(addresses), 1))(*addresses)


FORK_OK = dict(src=P, dst=P, cached=P, n=3, slots=5, states=_list(P, P), se=16384, convs=_list(P, P), ce=1152, nk=2, mla=_list(P), ss=6400,
               seq=50, nm=1, pools=_list(P), ps=1024, np=9, size=8, npl=1, table=P, ts=4, mp=4, rank=128, dt=1, ws=P, wsb=1 << 20, st=None)


@pytest.mark.parametrize("change,word", [
    (dict(n=-1), "moves"), (dict(n=4097), "moves"), (dict(slots=-1), "slots"), (dict(nk=49), "KDA"), (dict(nm=25), "MLA"),
    (dict(npl=25), "pools"), (dict(se=6), "multiples"), (dict(ce=9), "multiples"), (dict(rank=126, ss=6300), "rank"), (dict(ss=100), "stride"),
    (dict(table=None), "table"), (dict(dt=5), "dtype"), (dict(size=12), "page_size"), (dict(ts=3), "table"), (dict(np=-1), "table"),
    (dict(ps=1000), "page stride"), (dict(ps=1028), "page stride"), (dict(rank=132, ss=6600, ps=1056), "rank"), (dict(cached=None), "cached"),
    (dict(src=None), "NULL"), (dict(states=None), "NULL"), (dict(mla=None), "NULL"), (dict(pools=None), "NULL"), (dict(ws=None), "workspace"),
    (dict(wsb=32), "workspace"), (dict(states=_list(P, None)), "tensors"), (dict(convs=_list(P, P + 4)), "aligned"),
    (dict(pools=_list(P + 8)), "aligned")])
def test_fork_refuses(nat, change, word):  # noqa: F811
    rc, msg = _call(nat, "sophia_cache_fork", FORK_OK, FORK, **change)
    assert rc == nat.SOPHIA_ERR_INVALID and word in msg, msg


COPY = "src dst n pools npl ps pe np dt ws wsb st"
COPY_OK = dict(src=P, dst=P, n=3, pools=_list(P), npl=1, ps=1024, pe=1024, np=9, dt=1, ws=P, wsb=1 << 20, st=None)


@pytest.mark.parametrize("change,word", [
    (dict(dt=7), "dtype"), (dict(n=-1), "moves"), (dict(n=4097), "moves"), (dict(npl=25), "pools"), (dict(pe=1020), "multiples"),
    (dict(ps=1000), "multiples"), (dict(np=1 << 31), "multiples"), (dict(src=None), "NULL"), (dict(pools=None), "NULL"),
    (dict(pools=_list(None)), "pool"), (dict(pools=_list(P + 8)), "aligned"), (dict(ws=None), "workspace"), (dict(wsb=64), "workspace")])
def test_page_copy_refuses(nat, change, word):  # noqa: F811
    rc, msg = _call(nat, "sophia_page_copy", COPY_OK, COPY, **change)
    assert rc == nat.SOPHIA_ERR_INVALID and word in msg, msg


def test_moves_of_nothing(nat):  # noqa: F811
    assert _call(nat, "sophia_cache_fork", FORK_OK, FORK, n=0, src=None, cached=None, ws=None)[0] == nat.SOPHIA_OK
    assert _call(nat, "sophia_page_copy", COPY_OK, COPY, n=0, src=None, ws=None)[0] == nat.SOPHIA_OK
    size = nat.lib().sophia_move_workspace_size
    assert size(0) == size(4097) == 0 and size(4096) - size(1) == 4095 * 32


def test_no_cpu_tensors():
    from sophia_amd import ops
    i32, i64 = torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    x, pages, table = torch.zeros(1, 2, 32), torch.zeros(4, 16, 32), torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ops.mla_paged_attn(x, pages, table, i32, i64, 0.1, max_new=1)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ops.mla_latent_norms_paged(x[0], x[0], x, 1e-5, x, 1e-5, pages, table, i32, i64)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ops.beam_select(x[0], torch.zeros(2), 2)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ops.cache_fork(i32, i32)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ops.page_copy(i32, i32, [pages])
