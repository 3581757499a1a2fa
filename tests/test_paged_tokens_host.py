"""Refusals of the paged cache's tree, eviction and keep operators: bad arguments
end before any launch (CPU); and PagedQwen3Cache's bookkeeping around them."""
import types

import pytest
import torch

from spatten_b200 import _native as N
from tests.test_paged_host import BAD_CACHE, _attend, _cache

P = 1 << 20  # stands for a pointer


def _fill(a, kw):
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _tree(**kw):
    a = N.PagedTreeArgs()
    a.B, a.T, a.max_tokens, a.tree_words, a.tree_stride = 3, 60, 40, 2, 2
    a.cu_tokens = a.seq_lens = a.parents = a.tree = a.positions = P
    return _fill(a, kw)


def _ext(cache=(), attend=(), **kw):
    a = N.PagedAttendExtArgs()
    a.attend = _attend(cache=cache, **dict(attend))
    a.tree, a.tree_words, a.tree_stride = P, 1, 1
    a.weight = a.position = a.positions = P
    return _fill(a, kw)


def _evict(cache=(), **kw):
    a = N.PagedEvictArgs()
    _cache(a.cache, **dict(cache))
    a.B, a.keep, a.recent, a.per_head = 3, 10, 2, 0
    a.seq_lens = a.new_lens = a.weight = a.position = P
    return _fill(a, kw)


def _keep(cache=(), **kw):
    a = N.PagedKeepArgs()
    _cache(a.cache, **dict(cache))
    a.B, a.n_accepted, a.accepted_stride = 3, 5, 5
    a.cu_tokens = a.seq_lens = a.accepted = a.weight = a.position = P
    a.new_lens = 2 * P
    return _fill(a, kw)


def _run(kind, a):
    if kind == "ext":
        return N.lib.spatten_paged_attend_ext(a, None, 0, None)
    if kind == "evict":
        return N.lib.spatten_paged_evict(a, None, 0, None)
    return {"tree": N.lib.spatten_paged_tree, "keep": N.lib.spatten_paged_keep}[kind](a, None)


MAKE = {"tree": _tree, "ext": _ext, "evict": _evict, "keep": _keep}


@pytest.mark.parametrize("kind", ["ext", "evict", "keep"])
@pytest.mark.parametrize("field,value,code", BAD_CACHE)
def test_bad_cache(kind, field, value, code):
    kw = {field: value}
    if field == "max_pages" and value > 4:
        kw["table_stride"] = value
    assert _run(kind, MAKE[kind](cache=kw.items())) == code
    assert N.lib.spatten_last_error().decode().startswith("paged_")


@pytest.mark.parametrize("kind,field,value,code", [
    ("tree", "B", -1, N.ERR_INVALID), ("tree", "B", 70000, N.ERR_UNSUPPORTED), ("tree", "T", -1, N.ERR_INVALID),
    ("tree", "max_tokens", -1, N.ERR_INVALID), ("tree", "cu_tokens", 0, N.ERR_INVALID),
    ("tree", "seq_lens", P + 2, N.ERR_INVALID), ("tree", "parents", 0, N.ERR_INVALID),
    ("tree", "parents", P + 1, N.ERR_INVALID), ("tree", "tree", 0, N.ERR_INVALID), ("tree", "tree", P + 2, N.ERR_INVALID),
    ("tree", "tree_words", 1, N.ERR_INVALID), ("tree", "tree_words", 0, N.ERR_INVALID),
    ("tree", "tree_stride", 1, N.ERR_INVALID), ("tree", "tree_stride", -2, N.ERR_INVALID),
    ("tree", "positions", P + 2, N.ERR_INVALID),
    ("ext", "tree", P + 2, N.ERR_INVALID), ("ext", "tree_words", 0, N.ERR_INVALID),
    ("ext", "tree_stride", -1, N.ERR_INVALID), ("ext", "weight", 0, N.ERR_INVALID), ("ext", "position", 0, N.ERR_INVALID),
    ("ext", "weight", P + 4, N.ERR_INVALID), ("ext", "position", P + 8, N.ERR_INVALID),
    ("ext", "positions", P + 2, N.ERR_INVALID),
    ("evict", "B", -1, N.ERR_INVALID), ("evict", "B", 70000, N.ERR_UNSUPPORTED), ("evict", "keep", 0, N.ERR_INVALID),
    ("evict", "keep", -5, N.ERR_INVALID), ("evict", "recent", -1, N.ERR_INVALID), ("evict", "weight", 0, N.ERR_INVALID),
    ("evict", "position", 0, N.ERR_INVALID), ("evict", "weight", P + 4, N.ERR_INVALID),
    ("evict", "seq_lens", 0, N.ERR_INVALID), ("evict", "new_lens", 0, N.ERR_INVALID),
    ("evict", "new_lens", P + 1, N.ERR_INVALID),
    ("keep", "B", -1, N.ERR_INVALID), ("keep", "B", 70000, N.ERR_UNSUPPORTED), ("keep", "n_accepted", -1, N.ERR_INVALID),
    ("keep", "accepted", 0, N.ERR_INVALID), ("keep", "accepted", P + 2, N.ERR_INVALID),
    ("keep", "accepted_stride", -5, N.ERR_INVALID), ("keep", "weight", 0, N.ERR_INVALID),
    ("keep", "position", 0, N.ERR_INVALID), ("keep", "cu_tokens", 0, N.ERR_INVALID), ("keep", "seq_lens", 0, N.ERR_INVALID),
    ("keep", "new_lens", 0, N.ERR_INVALID), ("keep", "new_lens", P, N.ERR_INVALID),
    ("keep", "new_lens", P + 8, N.ERR_INVALID), ("keep", "new_lens", P - 8, N.ERR_INVALID),
])
def test_bad_arguments(kind, field, value, code):
    a = MAKE[kind](**{field: value})
    assert _run(kind, a) == code
    err = N.lib.spatten_last_error().decode()
    assert err.startswith("paged_") and "workspace of" not in err


@pytest.mark.parametrize("field,value", [("H", 7), ("q", 0), ("out", P + 8), ("q_st", 1020), ("sm_scale", float("nan")),
                                         ("o_sh", 64), ("T", -2), ("dtype", N.DTYPE_F32)])
def test_bad_attention_beside(field, value):
    """What the causal form refuses is refused with a tree and weights too."""
    a = _ext(attend={field: value}.items())
    assert _run("ext", a) in (N.ERR_INVALID, N.ERR_UNSUPPORTED)
    assert "workspace of" not in N.lib.spatten_last_error().decode()


def test_sizes_refused():
    assert _run("tree", _tree(max_tokens=1025, T=2000, tree_words=64, tree_stride=64)) == N.ERR_UNSUPPORTED
    wide = dict(max_pages=1 << 15, table_stride=1 << 15, page_size=64).items()  # 2^21 slots
    assert _run("evict", _evict(cache=wide)) == N.ERR_UNSUPPORTED
    assert N.lib.spatten_paged_evict_workspace_size(_evict(cache=wide)) == 0
    shared = dict(table_stride=0).items()
    for kind in ("evict", "keep"):
        assert _run(kind, MAKE[kind](cache=shared)) == N.ERR_INVALID and b"stride" in N.lib.spatten_last_error()
    for kind in MAKE:
        assert _run(kind, None) == N.ERR_INVALID


def test_what_is_missing_is_the_workspace():
    """Good arguments reach the check of the workspace; its size is that which is asked for."""
    for kind, size in (("ext", N.lib.spatten_paged_attend_ext_workspace_size),
                       ("evict", N.lib.spatten_paged_evict_workspace_size)):
        a = MAKE[kind]()
        n = size(a)
        assert n > 0 and n % 256 == 0 and _run(kind, a) == N.ERR_INVALID
        assert f"workspace of {n} bytes" in N.lib.spatten_last_error().decode()
    plain = N.lib.spatten_paged_attend_workspace_size(_attend())
    assert N.lib.spatten_paged_attend_ext_workspace_size(_ext(weight=0, position=0, positions=0)) == plain
    # scores are kept in a bounded workspace only
    big = dict(max_pages=1 << 13, table_stride=1 << 13, page_size=128).items()
    n = N.lib.spatten_paged_attend_ext_workspace_size(_ext(cache=big, attend=dict(B=256, T=256).items(), tree=0))
    assert 0 < n < 3 << 30


def test_no_work_is_ok():
    assert _run("tree", _tree(B=0, parents=0, tree=0)) == N.OK and _run("tree", _tree(max_tokens=0)) == N.OK
    assert _run("tree", _tree(T=0, tree=0, parents=0)) == N.OK
    assert _run("ext", _ext(attend=dict(T=0, q=0, out=0).items())) == N.OK
    assert _run("ext", _ext(attend=dict(B=0).items())) == N.OK
    none = dict(page_table=0, max_pages=0, table_stride=0).items()
    assert _run("evict", _evict(cache=none, B=0, seq_lens=0, new_lens=0)) == N.OK
    assert _run("keep", _keep(cache=none, B=0, seq_lens=0, new_lens=0, accepted=0)) == N.OK


def test_python_refuses_cpu_tensors():
    from spatten_b200 import paged
    c = paged.new_paged_cache(4, 2, 64, page_size=16, device="cpu")
    w = paged.new_paged_weights(c)
    assert w.weight.shape == w.position.shape == (4, 2, 16) and w.weight.dtype == torch.float32
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="no CPU path"):
        paged.paged_tree(i, i, i[:1], 1)
    with pytest.raises(ValueError, match="no CPU path"):
        paged.paged_evict(c, w, i[None], i[:1], 1)
    with pytest.raises(ValueError, match="no CPU path"):
        paged.paged_keep(c, i[None], i, i[:1], i[None])


# ------------------------------------------------------------------ PagedQwen3Cache

def _qwen(monkeypatch, batch=2, room=18, **kw):
    """A cache on the CPU whose operators are replaced by their bookkeeping."""
    from spatten_b200 import paged
    from spatten_b200.qwen3 import PagedQwen3Cache
    cfg = types.SimpleNamespace(num_hidden_layers=2, num_key_value_heads=2, head_dim=64)
    calls = []
    monkeypatch.setattr(paged, "paged_append", lambda *a, **k: calls.append("append"))

    def evict(cache, weights, table, lens, keep, recent=0):
        calls.append(("evict", keep, recent))
        return lens.clamp(max=keep)

    def tree(parents, cu, lens, n):
        calls.append(("tree", parents.tolist(), lens.tolist(), n))
        return torch.zeros(parents.shape[0], 1, dtype=torch.int32), torch.arange(parents.shape[0], dtype=torch.int32)

    def keep(cache, table, cu, lens, accepted, weights=None):
        calls.append(("keep", accepted.tolist(), weights is not None))
        return lens - (cu[1] - cu[0]) + accepted.shape[1]
    monkeypatch.setattr(paged, "paged_evict", evict)
    monkeypatch.setattr(paged, "paged_tree", tree)
    monkeypatch.setattr(paged, "paged_keep", keep)
    return PagedQwen3Cache(cfg, batch, room, page_size=4, device="cpu", **kw), calls


def _forward(c, n):
    x = torch.zeros(c.batch * n, 2, 64)
    for i in range(2):
        c.append(i, n, n, c.packed(n), x, x)


def test_a_full_cache_evicts(monkeypatch):
    c, calls = _qwen(monkeypatch, keep_tokens=10, recent_tokens=3)
    _forward(c, 16)
    _forward(c, 2)
    assert calls == ["append"] * 4 and c.held == [18] * 2
    _forward(c, 1)
    assert calls[4:] == [("evict", 10, 3), "append"] * 2
    assert c.held == [11] * 2 and (c.seq_lens == 11).all() and c.seen == [19] * 2 and c.pruned == [18] * 2
    c.crop(18)
    assert c.held == [10] * 2
    with pytest.raises(NotImplementedError):
        c.crop(17)
    with pytest.raises(ValueError, match="room"):  # more than an eviction makes room for: nothing changes
        _forward(c, 9)
    assert c.held == [10] * 2 and len(calls) == 8
    c.crop(0)
    assert c.held == c.pruned == [0] * 2


def test_arguments_of_a_bounded_cache(monkeypatch):
    for kw in (dict(keep_tokens=0), dict(keep_tokens=18), dict(keep_tokens=5, recent_tokens=6), dict(recent_tokens=1),
               dict(keep_tokens=5, recent_tokens=-1)):
        with pytest.raises(ValueError):
            _qwen(monkeypatch, **kw)
    c, _ = _qwen(monkeypatch)
    _forward(c, 18)
    with pytest.raises(ValueError, match="room"):
        _forward(c, 1)


def test_store_starts_the_accounts(monkeypatch):
    c, _ = _qwen(monkeypatch, keep_tokens=10)
    k = torch.zeros(2, 6, 2, 64)
    imp = torch.arange(12, dtype=torch.float32).view(2, 6)
    pos = torch.tensor([[0, 2, 3, 5, 7, 8], [1, 2, 3, 4, 5, 9]])
    c.store(0, k, k, 10, importance=imp, positions=pos)
    c.store(1, k, k, 6)
    for layer, (w, p) in enumerate(((imp, pos), (torch.zeros(2, 6), torch.arange(6).expand(2, 6)))):
        for b in range(2):
            for s in range(6):
                at = int(c.page_table[b, s // 4]), slice(None), s % 4
                assert (c.weights[layer].weight[at] == w[b, s] / 2).all()
                assert (c.weights[layer].position[at] == p[b, s]).all()
    assert c.positions(0, 3).tolist() == [10, 11, 12] * 2


def test_drafted_tree_bookkeeping(monkeypatch):
    c, calls = _qwen(monkeypatch)
    parents = torch.tensor([[-1, 0, 0, 1]] * 2)
    with pytest.raises(ValueError):
        c.draft_tree(parents)  # no prompt yet
    _forward(c, 5)
    for bad in (parents[:1], parents[:, :0]):
        with pytest.raises(ValueError):
            c.draft_tree(bad)
    pos = c.draft_tree(parents)
    assert pos.shape == (2, 4) and pos.dtype == torch.int64
    assert calls[-1] == ("tree", [-1, 0, 0, 1] * 2, [9, 9], 4)
    for call in (lambda: c.draft_tree(parents), lambda: c.accept([[0]] * 2), lambda: c.crop(3),
                 lambda: c.reorder_cache(torch.tensor([1, 0])), lambda: c.batch_repeat_interleave(2)):
        with pytest.raises(RuntimeError):
            call()
    _forward(c, 4)
    for bad in ([[0]], [[0], [0, 1]], [[1, 0]] * 2, [[0, 4]] * 2, [[-1, 0]] * 2, [[0, 0]] * 2):
        with pytest.raises(ValueError):
            c.accept(bad)
    c.accept(torch.tensor([[0, 1, 3], [0, 2, 3]]))
    assert calls[-2:] == [("keep", [[0, 1, 3], [0, 2, 3]], False)] * 2
    assert c.held == c.seen == [8, 8] and (c.seq_lens == 8).all() and c.tree is None
    c.draft_tree(parents)
    _forward(c, 4)
    c.accept([[], []])  # none of them
    assert c.held == [8, 8] and c.tree is None
    c.draft_tree(parents)
    c.reset()
    assert c.tree is None and c.seen == [0, 0]
