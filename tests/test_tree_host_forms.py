"""Host side of the drafted-token entry points that take one argument more than their first forms (CPU): the same refusals, and
those of the argument."""

from __future__ import annotations

import pytest

import test_tree_host as host
from test_tree_host import nat  # noqa: F401  (fixture)

COMMIT = host.COMMIT.replace(" rows ", " rows nodes ")
COMMIT_OK = dict(host.COMMIT_OK, nodes=64)


@pytest.mark.parametrize("change,word", [
    (dict(nodes=0), "max_nodes"), (dict(nodes=65), "max_nodes"), (dict(nodes=-1), "max_nodes"), (dict(width=65, ps=65), "max_path"),
    (dict(n=-1), "n_trees"), (dict(rows=-1), "rows"), (dict(nk=2), "layer list"), (dict(count=None), "NULL")])
def test_commit_within_refuses(nat, change, word):  # noqa: F811
    rc, msg = host._call(nat, "sophia_tree_commit_within", COMMIT_OK, COMMIT, **change)
    assert rc == nat.SOPHIA_ERR_INVALID and word in msg, msg


def test_commit_within_of_nothing(nat):  # noqa: F811
    for empty in (dict(n=0), dict(rows=0)):
        assert host._call(nat, "sophia_tree_commit_within", COMMIT_OK, COMMIT, path=None, cu=None, **empty)[0] == nat.SOPHIA_OK


@pytest.mark.parametrize("change,word", [
    (dict(dt=9), "dtype"), (dict(vocab=0), "vocab"), (dict(nodes=65), "max_nodes"), (dict(ps=4), "path rows"), (dict(xs=999), "stride"),
    (dict(tok=None), "NULL"), (dict(ws=None), "workspace"), (dict(wsb=8), "workspace")])
def test_strict_accept_refuses(nat, change, word):  # noqa: F811
    rc, msg = host._call(nat, "sophia_tree_accept_strict", host.ACCEPT_OK, host.ACCEPT, **change)
    assert rc == nat.SOPHIA_ERR_INVALID and word in msg, msg


def test_layer_lists_are_the_structures_of_the_header():
    """What tree_commit hands over: field by field the words it was made of, none left."""
    import ctypes
    from sophia_amd import _abi
    for struct in (_abi.CommitKda, _abi.CommitMla):
        fields = [f for f, _ in struct._fields_]
        assert ctypes.sizeof(struct) == 8 * len(fields)
        words = [(1 << 40) + 3 * i for i in range(7 * len(fields))]
        made = _abi.packed(struct, words)
        assert len(made) == 7 and made._type_ is struct
        assert [getattr(layer, f) for layer in made for f in fields] == words
        assert _abi.packed(struct, []) is None
    nulls = _abi.packed(_abi.CommitKda, [1, 2, 3, 0, 5])
    assert nulls[0].conv_state is None and nulls[0].state == 5
