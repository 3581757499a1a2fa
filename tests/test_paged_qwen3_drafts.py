"""PagedQwen3Cache around drafts that go wrong (CPU: the operators are replaced by
their bookkeeping)."""
import pytest
import torch

from tests.test_paged_tokens_host import _forward, _qwen


def _halfway(c, n):
    """A forward that fails behind the first layer."""
    x = torch.zeros(c.batch * n, 2, 64)
    c.append(0, n, n, c.packed(n), x, x)


@pytest.mark.parametrize("when", ["before", "halfway", "after"])
def test_a_tree_can_be_given_up(monkeypatch, when):
    c, calls = _qwen(monkeypatch)
    c.drop_tree()  # none: nothing
    parents = torch.tensor([[-1, 0, 0, 1]] * 2)
    _forward(c, 5)
    c.draft_tree(parents)
    if when == "halfway":
        _halfway(c, 4)
        assert c.held == [9, 5]
        with pytest.raises(RuntimeError):
            c.accept([[0]] * 2)
    elif when == "after":
        _forward(c, 4)
    c.drop_tree()
    assert c.tree is None and c.held == c.seen == [5, 5] and (c.seq_lens == 5).all()
    c.draft_tree(parents)  # and on
    _forward(c, 4)
    c.accept([[0, 1]] * 2)
    assert c.held == c.seen == [7, 7] and (c.seq_lens == 7).all()
    c.crop(6)
    assert c.held == [6, 6]


def test_a_tree_that_evicted_can_be_given_up(monkeypatch):
    c, calls = _qwen(monkeypatch, keep_tokens=10, recent_tokens=3)
    _forward(c, 16)
    c.draft_tree(torch.tensor([[-1, 0, 0, 1]] * 2))
    _halfway(c, 4)
    assert c.held == [14, 16]
    c.drop_tree()
    assert c.held == [10, 16] and c.seen == [16, 16] and c.seq_lens[:, 0].tolist() == [10, 16]
    _forward(c, 1)
    assert c.held == [11, 17] and c.seen == [17, 17]


def test_accepted_places_continue_the_text(monkeypatch):
    """Places whose positions skip or repeat are no branch."""
    c, calls = _qwen(monkeypatch)
    parents = torch.tensor([[-1, 0, 0, 1, 7, 3], [-1, 0, 1, -5, 3, 4]])
    _forward(c, 5)
    c.draft_tree(parents)
    parents.zero_()  # the cache has its own
    _forward(c, 6)
    for bad in ([[1], [0]], [[0], [1]], [[0, 3], [0, 1]], [[0, 4], [0, 1]], [[0, 1, 2], [0, 1, 2]], [[0, 1], [0, 3]]):
        with pytest.raises(ValueError, match="branch"):
            c.accept(bad)
    assert c.tree is not None and c.seen == [11, 11] and not any(x[0] == "keep" for x in calls)
    c.accept([[0, 1, 3], [3, 4, 5]])
    assert calls[-1] == ("keep", [[0, 1, 3], [3, 4, 5]], False) and c.seen == [8, 8]
