"""Qwen3 over a paged cache that forgets: eviction by accumulated attention when
a layer is full, and trees of drafted tokens in one forward. Every call that the
model makes of the cache's operators is checked against the float64 oracle."""
import pytest
import torch

from oracle import paged_tokens as OT
from tests.test_gpu_paged import BF16, E4, I8, _cpu, _cum
from tests.test_gpu_paged_tokens import _check, _check_moved

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


@pytest.fixture()
def lm(qwen3_model):
    from transformers import Qwen3ForCausalLM
    from spatten_b200.qwen3 import patch_qwen3
    torch.manual_seed(0)
    return patch_qwen3(Qwen3ForCausalLM(qwen3_model.config).to("cuda", BF16).eval())


@pytest.fixture()
def checked(monkeypatch):
    """The operators, each call checked; returns the counts of their calls."""
    from spatten_b200 import paged
    calls = {"attention": 0, "evict": 0, "keep": 0, "sees": None}
    attention, evict, keep = paged.paged_attention, paged.paged_evict, paged.paged_keep

    def _attention(q, cache, table, cu, lens, n, sm_scale=None, tree=None, weights=None, positions=None):
        before = weights and paged.PagedWeights(*(t.clone() for t in weights))
        out = attention(q, cache, table, cu, lens, n, sm_scale=sm_scale, tree=tree, weights=weights, positions=positions)
        _check(out, q, cache, table.cpu(), cu.tolist(), lens.tolist(), sm_scale, calls["sees"] if tree is not None else None,
               before, weights, None if positions is None else positions.tolist())
        calls["attention"] += 1
        return out

    def _evict(cache, weights, table, lens, k, **kw):
        before, w, p = _cpu(cache), weights.weight.cpu(), weights.position.cpu()
        new = evict(cache, weights, table, lens, k, **kw)
        moves, want = OT.evict(before, w, p, table.cpu(), lens.tolist(), k, **kw)
        assert new.tolist() == want and any(m[0] for m in moves)
        _check_moved(cache, before, table.cpu(), moves, want)
        calls["evict"] += 1
        return new

    def _keep(cache, table, cu, lens, accepted, weights=None):
        before = _cpu(cache)
        new = keep(cache, table, cu, lens, accepted, weights=weights)
        moves, want = OT.keep(before, table.cpu(), cu.tolist(), lens.tolist(), accepted.tolist())
        assert new.tolist() == want
        _check_moved(cache, before, table.cpu(), moves, want)
        calls["keep"] += 1
        return new
    monkeypatch.setattr(paged, "paged_attention", _attention)
    monkeypatch.setattr(paged, "paged_evict", _evict)
    monkeypatch.setattr(paged, "paged_keep", _keep)
    return calls


def _generate(lm, ids, cache, n):
    return lm.generate(ids, attention_mask=torch.ones_like(ids), past_key_values=cache, max_new_tokens=n, min_new_tokens=n,
                       do_sample=False, eos_token_id=None, pad_token_id=0)


@pytest.mark.parametrize("kv,B,prune", [(I8, 2, False), (E4, 1, True)])
def test_generation_past_the_caches_room(lm, checked, kv, B, prune):
    """Every layer evicts whenever it is full; the recent tokens and those that
    the oracle's weights name stay."""
    from spatten_b200.qwen3 import PagedQwen3Cache
    for layer in lm.model.layers:
        layer.self_attn.enable_token_prune, layer.self_attn.token_keep_ratio = prune, 0.9
    ids = torch.randint(0, 1000, (B, 40), generator=torch.Generator().manual_seed(3)).cuda()
    cache = PagedQwen3Cache(lm.config, B, 48, page_size=16, kv_dtype=kv, keep_tokens=33, recent_tokens=6)
    out = _generate(lm, ids, cache, 45)
    L = lm.config.num_hidden_layers
    assert out.shape == (B, 85) and checked["evict"] >= 2 * L and checked["attention"] == 44 * L
    assert max(cache.held) <= 48 and cache.get_seq_length() == 84
    for i in range(L):
        assert (cache.seq_lens[i] == cache.held[i]).all()
        n = cache.held[i]
        pos = cache.weights[i].position.view(B, -1, *cache.weights[i].position.shape[1:]).transpose(2, 3).flatten(1, 2)
        for b in range(B):
            held = pos[b, :n, 0].tolist()
            assert len(set(held)) == n and set(held) >= set(range(78, 84))  # distinct, the newest among them
    with pytest.raises(NotImplementedError):
        cache.crop(20)


def test_room_enough_changes_nothing(lm):
    """Without an eviction the tokens are those of a cache without accounts."""
    from spatten_b200.qwen3 import PagedQwen3Cache
    ids = torch.randint(0, 1000, (2, 30), generator=torch.Generator().manual_seed(4)).cuda()
    a = _generate(lm, ids, PagedQwen3Cache(lm.config, 2, 64), 20)
    cache = PagedQwen3Cache(lm.config, 2, 64, keep_tokens=40, recent_tokens=8)
    assert torch.equal(a, _generate(lm, ids, cache, 20))
    # each token's rows give a weight of 1 per query head: a layer's weights add up to them
    H = lm.config.num_attention_heads
    for w, n in zip(cache.weights, cache.held):
        total = w.weight.view(2, -1).double().sum(1)
        assert n == 49 and torch.allclose(total, torch.full_like(total, 49.0 * H), rtol=1e-3)


def test_beams_and_batches_take_the_weights_along(lm):
    from spatten_b200.qwen3 import PagedQwen3Cache
    ids = torch.randint(0, 1000, (1, 20), generator=torch.Generator().manual_seed(5)).cuda()
    cache = PagedQwen3Cache(lm.config, 3, 32, page_size=16, keep_tokens=20)
    out = lm.generate(ids, attention_mask=torch.ones_like(ids), past_key_values=cache, max_new_tokens=25, min_new_tokens=25,
                      num_beams=3, do_sample=False, eos_token_id=None, pad_token_id=0)
    assert out.shape == (1, 45) and max(cache.held) <= 32
    rows = [t.view(3, -1, *t.shape[1:]).clone() for t in cache.weights[1]]
    cache.reorder_cache(torch.tensor([2, 0, 0]))
    n = -(-cache.held[1] // 16)
    for t, was in zip(cache.weights[1], rows):
        assert torch.equal(t.view(3, -1, *t.shape[1:])[:, :n], was[[2, 0, 0]][:, :n])
    cache.batch_repeat_interleave(2)
    cache.batch_select_indices(torch.tensor([1, 5]))
    assert cache.batch == 2 and cache.weights[0].weight.shape[0] == cache.pools[0].k.shape[0]


@pytest.mark.parametrize("B,keep", [(1, None), (2, 60)])
def test_drafted_trees(lm, checked, B, keep):
    """Trees in one forward, their accepted branches kept, the text going on."""
    from spatten_b200.qwen3 import PagedQwen3Cache
    g = torch.Generator().manual_seed(6)
    cache = PagedQwen3Cache(lm.config, B, 72, page_size=16, keep_tokens=keep, recent_tokens=8 if keep else 0)
    ids = torch.randint(0, 1000, (B, 45), generator=g).cuda()
    with torch.no_grad():
        lm(input_ids=ids, past_key_values=cache, use_cache=True)
        parents = torch.tensor([[-1, 0, 0, 1, 1, 2, 5, 6, -1]] * B)
        parents[-1, 3] = 2
        seen, L = 45, lm.config.num_hidden_layers
        for step, path in enumerate(([0, 2, 5, 6], [0, 1, 4], [8], [0, 2, 5])):
            pos = cache.draft_tree(parents.cuda())
            assert pos[0].tolist() == [seen + d for d in (0, 1, 1, 2, 2, 2, 3, 4, 0)]
            cu = _cum([9] * B)
            checked["sees"] = OT.tree(parents.flatten().tolist(), cu, [seen + 9] * B, 9)[0]
            tokens = torch.randint(0, 1000, (B, 9), generator=g).cuda()
            out = lm(input_ids=tokens, position_ids=pos, past_key_values=cache, use_cache=True)
            assert out.logits.shape[:2] == (B, 9) and torch.isfinite(out.logits).all()
            with pytest.raises(RuntimeError):
                lm(input_ids=tokens, position_ids=pos, past_key_values=cache, use_cache=True)
            with pytest.raises(RuntimeError):
                cache.crop(3)
            cache.accept([path] * B)
            seen += len(path)
            assert cache.get_seq_length() == seen and cache.tree is None
            assert all((n == h).all() for n, h in zip(cache.seq_lens, cache.held))
        lm(input_ids=tokens[:, :1], past_key_values=cache, use_cache=True)
    assert checked["keep"] == 4 * L and checked["attention"] == 5 * L
    for bad in ([[0]] * (B + 1), [[2, 1]] * B, [[0, 9]] * B):
        cache.draft_tree(parents)
        with pytest.raises(RuntimeError):  # no forward yet
            cache.accept(bad)
        cache.tree = None


def test_operators_under_torch_ops():
    from spatten_b200 import paged
    import spatten_b200.torch_ops  # noqa: F401
    from tests.test_gpu_paged import _filled, _i32, _table
    from tests.test_gpu_paged_tokens import _weights
    g = torch.Generator().manual_seed(8)
    a, b = [_filled(I8, 8, 2, 16, 64, torch.Generator().manual_seed(9)) for _ in range(2)]
    table, cu, lens = _table(2, 4, 8, g).cuda(), _i32([0, 3, 6]), _i32([40, 50])
    wa = _weights(a, g)
    wb = paged.PagedWeights(*(t.clone() for t in wa))
    q, ops = torch.randn(6, 4, 64, generator=g).to(BF16).cuda(), torch.ops.spatten
    tree, pos = ops.paged_tree(_i32([-1, 0, 0, -1, 0, 1]), cu, lens, 3)
    assert pos.tolist() == [37, 38, 38, 47, 48, 49]
    assert torch.equal(ops.paged_tree_attention(q, *a, table, cu, lens, tree, 3, 0.125),
                       paged.paged_attention(q, b, table, cu, lens, 3, sm_scale=0.125, tree=tree))
    assert torch.equal(ops.paged_weighing_attention(q, *a, *wa, table, cu, lens, pos, 3, 0.125),
                       paged.paged_attention(q, b, table, cu, lens, 3, sm_scale=0.125, weights=wb, positions=pos))
    kept = ops.paged_keep(*a, table, cu, lens, _i32([[0, 2], [1, -1]]))
    assert torch.equal(kept, paged.paged_keep(b, table, cu, lens, _i32([[0, 2], [1, -1]])))
    assert torch.equal(ops.paged_evict(*a, *wa, table, kept, 20, 3, False),
                       paged.paged_evict(b, wb, table, kept, 20, recent=3))
    for x, y in zip((*a, *wa), (*b, *wb)):
        assert torch.equal(x, y)
