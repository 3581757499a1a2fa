"""PagedQwen3Cache's bookkeeping on the CPU: HF's operations on a cache (crop,
reorder_cache, batch_repeat_interleave, batch_select_indices) change what the
paged pools hold, or are refused before anything changes."""
import types

import pytest
import torch

I8, E4 = torch.int8, torch.float8_e4m3fn


def _cache(batch=2, held=(10, 10), seen=(10, 10), kv=I8, page=4, room=18):
    """Two layers whose slots hold values of their own, counted as ``held``
    slots of ``seen`` positions (fewer where a prompt was pruned)."""
    from spatten_b200.qwen3 import PagedQwen3Cache
    cfg = types.SimpleNamespace(num_hidden_layers=2, num_key_value_heads=2, head_dim=64)
    c = PagedQwen3Cache(cfg, batch, room, page_size=page, kv_dtype=kv, device="cpu")
    g = torch.Generator().manual_seed(0)
    for pool, h in zip(c.pools, held):
        for t in pool[:2]:
            t.view(I8).copy_(torch.randint(-100, 100, t.shape, generator=g, dtype=I8))
        for t in pool[2:]:
            t.copy_(torch.rand(t.shape, generator=g))
    c.held, c.seen = list(held), list(seen)
    c.pruned = [s if h < s else 0 for h, s in zip(held, seen)]
    c.seq_lens.copy_(torch.tensor(held, dtype=torch.int32)[:, None].expand(-1, batch))
    return c


def _slots(c, layer, b):
    """The codes and scales of what sequence b holds in a layer."""
    pool, n = c.pools[layer], int(c.seq_lens[layer, b])
    page = pool.k.shape[2]
    at = [(int(c.page_table[b, s // page]), s % page) for s in range(n)]
    return [torch.stack([t.view(I8)[p, :, r] for p, r in at]) for t in pool[:2]] + \
        [torch.stack([t[p] for p, _ in at]) for t in pool[2:]]


def _same(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("to,left", [(5, 5), (-3, 7), (10, 10), (12, 10), (0, 0), (-10, 0)])
def test_crop(to, left):
    c = _cache()
    was = [[_slots(c, i, b) for b in range(2)] for i in range(2)]
    c.crop(to)
    assert c.get_seq_length() == c.get_seq_length(1) == left and c.held == [left] * 2
    assert (c.seq_lens == left).all() and c.get_mask_sizes(1, 0) == (left + 1, 0)
    if left:
        for i in range(2):
            for b in range(2):
                assert _same(_slots(c, i, b), [t[:left] for t in was[i][b]])


def test_crop_of_a_pruned_prompt():
    """Layer 1 holds 4 of the prompt's 10 positions and 3 later ones: these can
    go, the prompt's only all together (which of the kept ones they were is not
    on the host)."""
    c = _cache(held=(13, 7), seen=(13, 13))
    c.pruned[1] = 10
    c.crop(11)
    assert c.held == [11, 5] and c.seen == [11, 11] and c.seq_lens.tolist() == [[11, 11], [5, 5]]
    c.crop(10)
    assert c.held == [10, 4] and c.seen == [10, 10]
    with pytest.raises(NotImplementedError, match="pruned"):
        c.crop(9)
    with pytest.raises(NotImplementedError, match="pruned"):
        c.crop(-1)
    assert c.held == [10, 4] and c.seen == [10, 10] and c.seq_lens.tolist() == [[10, 10], [4, 4]]
    c.crop(0)
    assert c.held == [0, 0] and c.pruned == [0, 0] and (c.seq_lens == 0).all()


def test_crop_after_layers_went_apart():
    """A forward that failed between two layers: both end at the same count."""
    c = _cache(held=(12, 10), seen=(12, 10))
    c.crop(10)
    assert c.held == c.seen == [10, 10] and (c.seq_lens == 10).all()


@pytest.mark.parametrize("kv", [I8, E4])
@pytest.mark.parametrize("beams", [[0, 1, 2], [2, 0, 1], [1, 1, 1], [0, 0, 2]])
def test_reorder(kv, beams):
    c = _cache(batch=3, held=(10, 6), seen=(10, 10), kv=kv)
    was = [[_slots(c, i, b) for b in range(3)] for i in range(2)]
    where = [t.data_ptr() for p in c.pools for t in p] + [c.seq_lens.data_ptr(), c.page_table.data_ptr()]
    c.reorder_cache(torch.tensor(beams))
    for i in range(2):
        for b, src in enumerate(beams):
            assert _same(_slots(c, i, b), was[i][src])
    # sequences keep pages of their own, at the addresses that a captured step reads
    assert c.page_table.unique().numel() == c.page_table.numel()
    assert where == [t.data_ptr() for p in c.pools for t in p] + [c.seq_lens.data_ptr(), c.page_table.data_ptr()]
    assert c.held == [10, 6] and c.seen == [10, 10] and c.pruned == [0, 10]


@pytest.mark.parametrize("kv", [I8, E4])
@pytest.mark.parametrize("op,arg,rows", [
    ("batch_repeat_interleave", 2, [0, 0, 1, 1, 2, 2]),
    ("batch_repeat_interleave", 1, [0, 1, 2]),
    ("batch_select_indices", torch.tensor([2, 0]), [2, 0]),
    ("batch_select_indices", torch.tensor([1, 1, 1, 0]), [1, 1, 1, 0]),
    ("batch_select_indices", torch.tensor([True, False, True]), [0, 2]),
])
def test_batch_changes(kv, op, arg, rows):
    c = _cache(batch=3, held=(10, 6), seen=(10, 10), kv=kv)
    was = [[_slots(c, i, b) for b in range(3)] for i in range(2)]
    getattr(c, op)(arg)
    assert c.batch == c.max_batch_size == len(rows) and c.page_table.unique().numel() == c.page_table.numel()
    assert c.packed(2).tolist() == list(range(0, 2 * len(rows) + 1, 2))
    for i in range(2):
        assert c.pools[i].k.shape[0] == c.page_table.numel() and c.pools[i].k.dtype == kv
        for b, src in enumerate(rows):
            assert _same(_slots(c, i, b), was[i][src])


def test_refused_rows():
    c = _cache(batch=2)
    was = [_slots(c, i, b) for i in range(2) for b in range(2)]
    for op, bad in (("reorder_cache", torch.tensor([0])), ("reorder_cache", torch.tensor([0, 1, 1])),
                    ("reorder_cache", torch.tensor([0, 2])), ("reorder_cache", torch.tensor([0, -1])),
                    ("batch_select_indices", torch.tensor([3])), ("batch_select_indices", torch.tensor([True])),
                    ("batch_repeat_interleave", 0)):
        with pytest.raises((ValueError, IndexError)):
            getattr(c, op)(bad)
    assert c.batch == 2 and _same(was[0] + was[3], _slots(c, 0, 0) + _slots(c, 1, 1))


def test_sizes_that_hf_asks_for():
    c = _cache(batch=2, room=18)
    assert c.max_batch_size == 2 and c.max_cache_len == 18 and c.get_max_cache_shape() == 18
    c.reset()
    assert c.get_seq_length() == 0 and c.held == [0, 0] and c.pruned == [0, 0] and (c.seq_lens == 0).all()


def test_a_refused_append_counts_nothing(monkeypatch):
    """An append that refuses its arguments (here: a cache without a GPU, rows of
    another type) leaves the counts as they were, on the host and beside the
    pools; and so does a forward that finds no room."""
    from spatten_b200 import paged
    c = _cache(held=(10, 6), seen=(10, 10))
    was = list(c.held), list(c.seen), list(c.pruned), c.seq_lens.clone()
    x = torch.zeros(2, 3, 2, 64, dtype=torch.float16)
    for k, seen in ((x, 3), (x, 5), (x.float(), 3), (torch.zeros(2, 9, 2, 64, dtype=torch.float16), 9)):
        for layer in range(2):
            with pytest.raises((ValueError, TypeError)):
                c.store(layer, k, k, seen)
            assert (c.held, c.seen, c.pruned) == was[:3] and torch.equal(c.seq_lens, was[3])
    # the call itself finds the new lengths
    calls = []
    monkeypatch.setattr(paged, "paged_append", lambda *a, **kw: calls.append((a[5].tolist(), a[6])))
    c.store(1, x, x, 5)
    assert calls == [([9, 9], 3)] and c.held == [10, 9] and c.seen == [10, 15] and c.pruned == [0, 15]


def test_lengths_given_as_tensors_and_empty_caches():
    c = _cache()
    c.crop(torch.tensor(4))
    assert c.held == c.seen == [4, 4] and all(type(n) is int for n in c.held + c.seen)
    c.reset()
    c.reorder_cache(torch.tensor([1, 1]))
    c.batch_repeat_interleave(2)
    assert c.batch == 4 and c.held == [0, 0] and c.seq_lens.shape == (2, 4)
