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
