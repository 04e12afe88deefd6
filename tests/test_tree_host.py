"""Host side of the drafted-token operators (CPU): what their entry points refuse before any launch, size queries, and the
structures that the binding shares with include/sophia_draft.h."""

from __future__ import annotations

import ctypes
import os
import re

import pytest
import torch


@pytest.fixture(scope="module")
def nat():
    from sophia_amd import _native
    if not os.path.exists(_native.LIB_PATH):
        pytest.skip("HIP library not built (run `python -m sophia_amd.build`)")
    return _native


HEADER = open(os.path.join(os.path.dirname(__file__), "..", "include", "sophia_draft.h")).read()


def test_header_constants_and_structures_match_the_binding():
    from sophia_amd import _abi
    assert int(re.search(r"#define SOPHIA_TREE_NODES (\d+)", HEADER).group(1)) == _abi.TREE_NODES
    for name, struct in (("sophia_commit_kda", _abi.CommitKda), ("sophia_commit_mla", _abi.CommitMla)):
        body = re.search(r"typedef struct \{([^}]*)\} " + name, HEADER).group(1)
        fields = re.findall(r"^\s*(.+?)(\w+);", body, re.M)
        assert [f for _, f in fields] == [f for f, _ in struct._fields_]
        for (ctype, _), (_, ptype) in zip(fields, struct._fields_):
            assert ptype is (ctypes.c_void_p if "*" in ctype else ctypes.c_int64)


# Addresses that no call here looks at: each returns at a check.
P = 1 << 12


def _call(nat, name, args, order, **change):
    values = dict(args, **change)
    rc = getattr(nat.lib(), name)(*[values[k] for k in order.split()])
    return rc, nat.last_error()


ATTN = "qa qs latent ls dt cache ss slots_n seq slots cached cu par n rows nodes scale out os heads rank splits sk ws wsb st"
ATTN_OK = dict(qa=P, qs=2048, latent=P, ls=128, dt=1, cache=P, ss=1024 * 128, slots_n=4, seq=1024, slots=P, cached=P, cu=P,
               par=P, n=2, rows=9, nodes=5, scale=0.1, out=P, os=2048, heads=16, rank=128, splits=1, sk=64, ws=None, wsb=0, st=None)


@pytest.mark.parametrize("change,word", [
    (dict(dt=2), "dtype"), (dict(rank=96), "rank"), (dict(heads=17), "heads"), (dict(heads=0), "heads"),
    (dict(nodes=65), "max_nodes"), (dict(nodes=0), "max_nodes"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(ss=100), "slot stride"), (dict(qs=2047), "strides"), (dict(qs=2052), "strides"),
    (dict(ls=127), "strides"), (dict(ls=132), "strides"), (dict(os=100), "strides"), (dict(qa=P + 8), "aligned"),
    (dict(cache=P + 4), "aligned"), (dict(out=P + 2), "aligned"), (dict(cached=None), "NULL"), (dict(par=None), "NULL"),
    (dict(splits=2), "workspace"), (dict(splits=2, ws=P, wsb=16), "workspace"), (dict(splits=0), "splits"),
    (dict(sk=0), "split_keys"), (dict(sk=96), "split_keys"),
    (dict(n=-1), "n_trees"), (dict(n=70000), "n_trees"), (dict(rows=-1), "rows"), (dict(seq=-1), "slot stride")])
def test_tree_attention_refuses(nat, change, word):
    rc, msg = _call(nat, "sophia_mla_tree_attn", ATTN_OK, ATTN, **change)
    assert rc == nat.SOPHIA_ERR_INVALID and word in msg, msg


STEP = ("xq xk xv xs xdt w hist taps g gs gdt beta bs bdt alog dtb scale lb flags state slots_n slots cu par n rows nodes heads "
        "hd o os tape st")
STEP_OK = dict(xq=P, xk=P, xv=P, xs=6144, xdt=1, w=P, hist=P, taps=4, g=P, gs=2048, gdt=1, beta=P, bs=16, bdt=1, alog=P, dtb=P,
               scale=0.1, lb=-5.0, flags=7, state=P, slots_n=4, slots=P, cu=P, par=P, n=2, rows=9, nodes=5, heads=16, hd=128,
               o=P, os=2048, tape=P, st=None)


@pytest.mark.parametrize("change,word", [
    (dict(hd=64), "head_dim"), (dict(taps=5), "kernel_size"), (dict(taps=0), "kernel_size"), (dict(n=-2), "n_trees"),
    (dict(heads=0), "num_heads"), (dict(nodes=65), "max_nodes"), (dict(xdt=3), "dtype"), (dict(gdt=3), "dtype"),
    (dict(bdt=-1), "dtype"), (dict(slots_n=-1), "n_slots"), (dict(xs=2000), "stride"), (dict(gs=2000), "stride"),
    (dict(bs=15), "stride"), (dict(os=2044), "stride"), (dict(xs=6148), "multiples"), (dict(hist=None), "NULL"),
    (dict(tape=None), "NULL"), (dict(alog=None), "A_log"), (dict(dtb=None), "A_log"), (dict(xq=P + 2), "aligned"),
    (dict(state=P + 8), "aligned"), (dict(o=P + 8), "aligned"), (dict(g=P + 8), "aligned"),
    (dict(dtb=P + 4), "aligned")])
def test_tree_step_refuses(nat, change, word):
    rc, msg = _call(nat, "sophia_kda_tree_step", STEP_OK, STEP, **change)
    assert rc == nat.SOPHIA_ERR_INVALID and word in msg, msg


COMMIT = "path ps count width cu n rows slots slots_n kda nk heads hd taps xdt mla nm cached seq rank ldt st"
COMMIT_OK = dict(path=P, ps=8, count=P, width=8, cu=P, n=2, rows=9, slots=P, slots_n=4, kda=None, nk=0, heads=16, hd=128, taps=4,
                 xdt=1, mla=None, nm=0, cached=P, seq=64, rank=128, ldt=1, st=None)


def test_commit_refuses(nat):
    def bad(word, kda=None, mla=None, **change):
        if kda is not None:
            change.update(kda=(nat.CommitKda * 1)(nat.CommitKda(*kda)), nk=change.get("nk", 1))
        if mla is not None:
            change.update(mla=(nat.CommitMla * 1)(nat.CommitMla(*mla)), nm=change.get("nm", 1))
        rc, msg = _call(nat, "sophia_tree_commit", COMMIT_OK, COMMIT, **change)
        assert rc == nat.SOPHIA_ERR_INVALID and word in msg, msg
    kda, mla = (P, P, 6144, P, P), (P, 128, P, 64 * 128)
    bad("n_trees", n=-1)
    bad("max_path", width=65, ps=65)
    bad("max_path", ps=7)
    bad("layer list", nk=2)
    bad("layer list", nm=2)
    bad("head_dim", kda=kda, hd=64)
    bad("num_heads", kda=kda, heads=0)
    bad("kernel_size", kda=kda, taps=5)
    bad("x fp32", kda=kda, xdt=7)
    bad("rank", mla=mla, rank=6)
    bad("max_seq", mla=mla, seq=-1)
    bad("NULL", kda=kda, count=None)
    bad("NULL", mla=mla, cached=None)
    bad("NULL pointer in KDA layer 0", kda=(None, P, 6144, P, P))
    bad("NULL pointer in KDA layer 0", kda=(P, P, 6144, None, P))
    bad("stride", kda=(P, P, 6143, P, P))
    bad("aligned", kda=(P, P, 6144, P, P + 4))
    bad("NULL pointer in MLA layer 0", mla=(None, 128, P, 64 * 128))
    bad("strides in MLA layer 0", mla=(P, 127, P, 64 * 128))
    bad("strides in MLA layer 0", mla=(P, 128, P, 63 * 128))
    bad("aligned in MLA layer 0", mla=(P + 4, 128, P, 64 * 128))


ADJUST = ("x xs y ys dt rows vocab hist hs hl pl hmax rep pres freq ids bias nb allowed masks arows cu par tok n nodes st")
ADJUST_OK = dict(x=P, xs=1000, y=P, ys=1000, dt=1, rows=9, vocab=1000, hist=P, hs=50, hl=P, pl=P, hmax=50, rep=P, pres=P, freq=P,
                 ids=P, bias=P, nb=4, allowed=P, masks=2, arows=P, cu=P, par=P, tok=P, n=2, nodes=5, st=None)


@pytest.mark.parametrize("change,word", [
    (dict(dt=2), "dtype"), (dict(rows=-1), "rows"), (dict(vocab=-1), "vocab"), (dict(n=70000), "n_seqs"),
    (dict(nodes=0), "max_nodes"), (dict(nodes=65), "max_nodes"), (dict(cu=None), "a row is a sequence"),
    (dict(xs=999), "stride"), (dict(ys=10), "stride"), (dict(hs=49), "history"), (dict(hmax=-1, hs=0), "history"),
    (dict(nb=-1), "counts"), (dict(masks=-1), "counts"), (dict(x=None), "NULL"), (dict(par=None), "parents"),
    (dict(tok=None), "tokens"), (dict(hl=None), "history_len"), (dict(bias=None), "biases"), (dict(arows=None), "mask per row")])
def test_adjust_refuses(nat, change, word):
    rc, msg = _call(nat, "sophia_adjust_logits", ADJUST_OK, ADJUST, **change)
    assert rc == nat.SOPHIA_ERR_INVALID and word in msg, msg


ACCEPT = "x xs dt rows vocab tok cu par n nodes path ps count next chosen ws wsb st"
ACCEPT_OK = dict(x=P, xs=1000, dt=1, rows=9, vocab=1000, tok=P, cu=P, par=P, n=2, nodes=5, path=P, ps=5, count=P, next=P, chosen=P,
                 ws=P, wsb=1 << 20, st=None)


@pytest.mark.parametrize("change,word", [
    (dict(dt=9), "dtype"), (dict(rows=-1), "rows"), (dict(vocab=0), "vocab"), (dict(n=-1), "n_trees"), (dict(nodes=65), "max_nodes"),
    (dict(ps=4), "path rows"), (dict(xs=999), "stride"), (dict(tok=None), "NULL"), (dict(path=None), "NULL"),
    (dict(ws=None), "workspace"), (dict(wsb=8), "workspace"), (dict(ws=P + 4), "workspace")])
def test_accept_refuses(nat, change, word):
    rc, msg = _call(nat, "sophia_tree_accept", ACCEPT_OK, ACCEPT, **change)
    assert rc == nat.SOPHIA_ERR_INVALID and word in msg, msg


def test_sizes_and_empty_calls(nat):
    lib = nat.lib()
    assert lib.sophia_tree_accept_workspace_size(-1, 5) == 0 and lib.sophia_tree_accept_workspace_size(0, 5) == 0
    assert lib.sophia_tree_accept_workspace_size(3, 5) >= 3 * 8
    # nothing to do: no pointer is needed
    null = dict(qa=None, latent=None, cache=None, cached=None, cu=None, par=None, out=None)
    for empty in (dict(n=0), dict(rows=0)):
        assert _call(nat, "sophia_mla_tree_attn", ATTN_OK, ATTN, **null, **empty)[0] == nat.SOPHIA_OK
        assert _call(nat, "sophia_kda_tree_step", STEP_OK, STEP, xq=None, tape=None, cu=None, **empty)[0] == nat.SOPHIA_OK
        assert _call(nat, "sophia_tree_commit", COMMIT_OK, COMMIT, path=None, cu=None, **empty)[0] == nat.SOPHIA_OK
    assert _call(nat, "sophia_adjust_logits", ADJUST_OK, ADJUST, x=None, rows=0)[0] == nat.SOPHIA_OK
    assert _call(nat, "sophia_tree_accept", ACCEPT_OK, ACCEPT, x=None, path=None, rows=0, n=0)[0] == nat.SOPHIA_OK
    assert _call(nat, "sophia_tree_accept", ACCEPT_OK, ACCEPT, x=None, n=0)[0] == nat.SOPHIA_ERR_INVALID   # (rows of no tree)


def test_operators_reject_cpu_tensors():
    from sophia_amd import ops
    f, i32, i64 = torch.zeros, torch.int32, torch.int64
    cu, par = torch.tensor([0, 4], dtype=i32), f(4, dtype=i32)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ops.mla_tree_attn(f(4, 2, 32), f(4, 32), f(1, 8, 32), cu, par, f(1, dtype=i32), f(1, dtype=i64), 0.1, max_nodes=4)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ops.kda_tree_step(f(4, 768), f(768, 4), f(1, 768, 3), f(4, 2, 128), f(4, 2), f(1, 2, 128, 128), cu, par, max_nodes=4,
                          A_log=f(2), dt_bias=f(256))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ops.tree_commit(f(1, 4, dtype=i32), f(1, dtype=i32), cu, None)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ops.adjust_logits(f(4, 10))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ops.tree_accept(f(4, 10), f(4, dtype=i64), cu, par, max_nodes=4)


def test_tree_attention_splits_rule(nat):
    from sophia_amd import ops
    for length in (0, 1, 255, 257, 4096, 10 ** 5, 2 ** 31 - 1):
        s = ops.mla_tree_splits(length)
        assert 1 <= s <= 128
        assert s <= -(-length // 64) + 1    # no range without keys at the longest length
    size = nat.lib().sophia_mla_tree_workspace_size
    part = 4 * 64 * (128 // 2 + 2) * 4      # of 8 nodes in bf16
    assert size(1, 7, 128, nat.DTYPE_BF16, 5) == 5 * part and size(1, 9, 128, nat.DTYPE_BF16, 5) == 10 * part
    assert size(65535, 64, 128, nat.DTYPE_BF16, 128) == 1024 * part
    assert size(3, 64, 256, nat.DTYPE_F32, 1) == size(0, 64, 256, nat.DTYPE_F32, 4) == size(-1, 64, 256, nat.DTYPE_F32, 4) == 0
    assert size(2, 5, 128, nat.DTYPE_F32, 4) == 16 * 4 * 64 * (128 // 4 + 2) * 4
