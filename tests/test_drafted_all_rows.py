"""ptoamd_draft_tree_all refuses what ptoamd_draft_tree refuses, under its own name."""
import pytest

import __graft_entry__ as ge
from test_drafted_refusals import AT, TREE


def call(**change):
    pa = ge.load_package()
    good = dict(tree=AT, words=1, parents=AT, tokens=2, sequences=2, cu=None, most=1, stream=None)
    assert not set(change) - set(good)
    good.update(change)
    return pa.lib().ptoamd_draft_tree_all(*good.values()), pa.lib().ptoamd_last_error().decode()


@pytest.mark.parametrize("change,code,text", TREE + [
    (dict(tree=None), -1, "null"), (dict(parents=None), -1, "null"), (dict(parents=AT + 2), -3, "aligned"), (dict(tokens=-1), -1, "negative"),
    (dict(sequences=0), -1, "positive"), (dict(most=-1), -1, "negative"), (dict(tokens=3), -1, "sequences * max_tokens"),
    (dict(parents=AT + 8), -1, "overlap"), (dict(parents=AT + 64, cu=AT - 8), -1, "overlap"), (dict(cu=AT + 64, most=0, words=0), -1, "words"),
    (dict(cu=AT + 64, most=0, tree=None), -1, "null")])
def test_refusals(change, code, text):
    rc, error = call(**change)
    assert rc == code and text in error and error.startswith("ptoamd_draft_tree_all:"), error
    assert call(tokens=0, most=0)[0] == 0
