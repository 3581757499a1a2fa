"""What PagedQwen3Cache(keep_tokens=...) counts while tokens are drafted: the attention
weights of the text's tokens and no others, to the bounds of
tests/test_gpu_paged_tokens.py where a call is compared with the oracle."""
import pytest
import torch

from oracle import paged_tokens as OT
from tests.test_gpu_paged import BF16, E4, I8, U, _cpu

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


def _ids(B, n, seed):
    return torch.randint(0, 1000, (B, n), generator=torch.Generator().manual_seed(seed)).cuda()


def _totals(cache, lm, tokens):
    """Each token of the text gives a weight of 1 per query head, in every layer: a layer's
    weights add up to them (fp32 sums of at most 2^8 rounded terms each, 2^-16)."""
    H = lm.config.num_attention_heads
    for w, n in zip(cache.weights, cache.held):
        by_seq = w.weight.view(cache.batch, -1, *w.weight.shape[1:]).transpose(2, 3).flatten(1, 2)[:, :n]
        total = by_seq.double().sum((1, 2))
        assert torch.allclose(total, torch.full_like(total, tokens * H), rtol=2.0 ** -12), (total.tolist(), tokens * H)


PARENTS = [-1, 0, 0, 1, 1, 2, 5, 6, -1]


@pytest.mark.parametrize("kv,B", [(I8, 1), (E4, 2)])
def test_rejected_drafts_of_a_tree_do_not_count(lm, kv, B):
    """Over a text that a tree's accepted branch continued, each layer's weights are
    those of before and what the oracle gives for the accepted tokens' queries."""
    from spatten_b200.qwen3 import PagedQwen3Cache
    cache = PagedQwen3Cache(lm.config, B, 120, page_size=16, kv_dtype=kv, keep_tokens=60, recent_tokens=8)
    G, H, D = lm.config.num_key_value_heads, lm.config.num_attention_heads, lm.config.head_dim
    with torch.no_grad():
        lm(input_ids=_ids(B, 45, 1), past_key_values=cache, use_cache=True)
        seen = 45
        for step, path in enumerate(([0, 2, 5, 6], [], [8], [0, 1, 4], [0, 2, 5])):
            _totals(cache, lm, seen)
            pos = cache.draft_tree(torch.tensor([PARENTS] * B))
            lm(input_ids=_ids(B, 9, step + 2), position_ids=pos, past_key_values=cache, use_cache=True)
            before = [w.weight.double().cpu().clone() for w in cache.weights]
            queries = [q[:, path].float().cpu() for q, _ in cache.asked]
            cache.accept([path] * B)
            seen, n = seen + len(path), len(path)
            assert cache.held == [seen] * len(cache.held)
            table, cu = cache.page_table.cpu(), [b * n for b in range(B + 1)]
            for i, (w, q) in enumerate(zip(cache.weights, queries)):
                want = before[i].view(B, -1, G, 16).transpose(2, 3).flatten(1, 2)[:, :seen - n]  # [B, slots, G]
                _, _, _, add, err = OT.attend(q.reshape(B * n, H, D), _cpu(cache.pools[i]), table, cu, [seen] * B, D ** -0.5)
                got = w.weight.double().cpu().view(B, -1, G, 16).transpose(2, 3).flatten(1, 2)[:, :seen]
                at = w.position.cpu().view(B, -1, G, 16).transpose(2, 3).flatten(1, 2)[:, :seen]
                assert (at == torch.arange(seen)[None, :, None]).all()
                for b in range(B):
                    total = torch.cat([want[b], torch.zeros(n, G).double()]) + (add[b].T if n else 0)
                    tol = 2 * D * U * (err[b].T if n else 0) + total * (3 * 2.0 ** -16) + 1e-37
                    assert ((got[b] - total).abs() <= tol).all()
        _totals(cache, lm, seen)


def test_a_text_continued_by_trees_weighs_its_tokens(lm):
    from spatten_b200.qwen3 import PagedQwen3Cache
    cache = PagedQwen3Cache(lm.config, 2, 120, page_size=16, keep_tokens=60, recent_tokens=8)
    with torch.no_grad():
        lm(input_ids=_ids(2, 30, 1), past_key_values=cache, use_cache=True)
        for step in range(3):
            pos = cache.draft_tree(torch.tensor([PARENTS] * 2))
            lm(input_ids=_ids(2, 9, step + 2), position_ids=pos, past_key_values=cache, use_cache=True)
            cache.accept([[0, 1, 3], [0, 2, 5]])
            lm(input_ids=_ids(2, 1, step + 9), past_key_values=cache, use_cache=True)
    _totals(cache, lm, 42)


@pytest.mark.parametrize("kv,B,n,stay", [(I8, 1, 6, 2), (E4, 2, 6, 5), (I8, 2, 1, 0), (E4, 1, 64, 1), (I8, 1, 90, 40)])
def test_cropped_drafts_do_not_count(lm, kv, B, n, stay):
    """n drafted tokens of which the last are cropped: each layer's weights are those of
    before and what the oracle gives for the queries that stay. What was added and taken
    back again leaves its rounding twice."""
    from spatten_b200.qwen3 import PagedQwen3Cache
    cache = PagedQwen3Cache(lm.config, B, 200, page_size=16, kv_dtype=kv, keep_tokens=150)
    G, H, D, old = lm.config.num_key_value_heads, lm.config.num_attention_heads, lm.config.head_dim, 45
    flat = lambda w: w.double().cpu().view(B, -1, G, 16).transpose(2, 3).flatten(1, 2)  # noqa: E731  [B, slots, G]
    with torch.no_grad():
        lm(input_ids=_ids(B, old, 1), past_key_values=cache, use_cache=True)
        before = [flat(w.weight) for w in cache.weights]
        lm(input_ids=_ids(B, n, 2), past_key_values=cache, use_cache=True)
        queries = [q.float().cpu() for q, _ in cache.asked]
        m = queries[0].shape[1]
        assert m == min(n, 64) and n - stay <= m
        cache.crop(stay - n if n == 6 else old + stay)  # (a negative length: that many of the last)
        assert cache.get_seq_length() == old + stay
    _totals(cache, lm, old + stay)
    table, held = cache.page_table.cpu(), old + n
    for i, (w, q) in enumerate(zip(cache.weights, queries)):
        cu = [b * m for b in range(B + 1)]
        args = _cpu(cache.pools[i]), table, cu
        _, _, _, all_of, err = OT.attend(q.reshape(B * m, H, D), *args, [held] * B, D ** -0.5)
        gone = q[:, m - (n - stay):].reshape(-1, H, D)
        _, _, _, out_of, _ = OT.attend(gone, *args[:2], [b * (n - stay) for b in range(B + 1)], [held] * B, D ** -0.5)
        got = flat(w.weight)[:, :old]
        for b in range(B if n <= 64 else 0):  # (of more, the first ones' queries are not at hand: the totals)
            want = before[i][b, :old] + (all_of[b] - out_of[b])[:, :old].T
            most = before[i][b, :old] + all_of[b][:, :old].T
            tol = 4 * D * U * err[b][:, :old].T + most * (6 * 2.0 ** -16) + 1e-37
            assert ((got[b] - want).abs() <= tol).all()


@pytest.mark.parametrize("quant", [False, True])
def test_drafts_of_generate_do_not_count(lm, quant):
    """HF's drafted tokens, the first ones in the prompt's own forward."""
    from spatten_b200.qwen3 import PagedQwen3Cache
    for layer in lm.model.layers:
        layer.self_attn.enable_prog_quant = quant
    ids = torch.randint(0, 50, (1, 10), generator=torch.Generator().manual_seed(1)).repeat(1, 4).cuda()
    cache, dropped = PagedQwen3Cache(lm.config, 1, 128, page_size=16, keep_tokens=100), []
    crop = cache.crop

    def counted(length):
        dropped.append(cache.get_seq_length() - length)
        crop(length)
        _totals(cache, lm, length)
    cache.crop = counted
    lm.generate(ids, attention_mask=torch.ones_like(ids), past_key_values=cache, max_new_tokens=30, min_new_tokens=30,
                do_sample=False, eos_token_id=999, pad_token_id=0, prompt_lookup_num_tokens=4)
    assert dropped[0] > 0 and sum(d > 0 for d in dropped) > 3


def test_noted_queries_follow_their_sequences(lm):
    """A crop after the batch was reordered and selected from; a second one takes what is left."""
    from spatten_b200.qwen3 import PagedQwen3Cache
    cache = PagedQwen3Cache(lm.config, 3, 64, page_size=16, keep_tokens=60)
    with torch.no_grad():
        lm(input_ids=_ids(3, 20, 1), past_key_values=cache, use_cache=True)
        lm(input_ids=_ids(3, 6, 2), past_key_values=cache, use_cache=True)
        cache.reorder_cache(torch.tensor([2, 0, 0]))
        cache.batch_select_indices(torch.tensor([0, 2]))
        cache.batch_repeat_interleave(2)
        for n in (24, 21, 20):
            cache.crop(n)
            _totals(cache, lm, n)
        assert cache.asked == [None] * len(cache.asked)
        lm(input_ids=_ids(4, 5, 3), past_key_values=cache, use_cache=True)
    _totals(cache, lm, 25)


def test_a_tree_given_up_leaves_the_accounts(lm):
    """After its forward, or when a layer raises."""
    from spatten_b200.qwen3 import PagedQwen3Cache
    cache = PagedQwen3Cache(lm.config, 1, 120, page_size=16, keep_tokens=60)
    attn = lm.model.layers[1].self_attn
    with torch.no_grad():
        lm(input_ids=_ids(1, 30, 1), past_key_values=cache, use_cache=True)
        before = [[t.clone() for t in w] for w in cache.weights]
        for fails in (False, True):
            pos = cache.draft_tree(torch.tensor([PARENTS]))
            o_proj = attn.o_proj
            attn.o_proj = None if fails else o_proj  # (no module)
            try:
                lm(input_ids=_ids(1, 9, 2), position_ids=pos, past_key_values=cache, use_cache=True)
                assert not fails
            except TypeError:
                assert fails and cache.seen == [39, 39, 30]
            attn.o_proj = o_proj
            cache.drop_tree()
            assert cache.held == cache.seen == [30] * 3
            for w, was in zip(cache.weights, before):
                assert all(torch.equal(a, b) for a, b in zip(w, was))
        lm(input_ids=_ids(1, 3, 3), past_key_values=cache, use_cache=True)
    _totals(cache, lm, 33)


def test_a_refused_append_forgets_nothing(lm):
    """A full cache evicts only for tokens that it can take."""
    from spatten_b200.qwen3 import PagedQwen3Cache
    cache = PagedQwen3Cache(lm.config, 1, 48, page_size=16, keep_tokens=30)
    G, D = lm.config.num_key_value_heads, lm.config.head_dim
    with torch.no_grad():
        lm(input_ids=_ids(1, 48, 1), past_key_values=cache, use_cache=True)
    was = [t.clone().view(I8) for i in range(3) for t in (*cache.pools[i], *cache.weights[i])]
    good = torch.zeros(2, G, D, dtype=BF16, device="cuda")
    shifted = torch.zeros(2 * G * D + 1, dtype=BF16, device="cuda")[1:].view(2, G, D)  # not 16-byte aligned
    cos = torch.zeros(2, D, dtype=BF16, device="cuda")
    for k, kw in ((good.float(), {}), (good[:1], {}), (good[..., :64], {}), (good.cpu(), {}), (shifted, {}),
                  (good, dict(cos=cos)), (good, dict(cos=cos, sin=cos.float())), (good, dict(q_norm_w=cos[0])),
                  (good, dict(k_norm_w=good[0, 0], eps=-1.0))):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            cache.append(0, 2, 2, cache.packed(2), k, good, **kw)
    assert cache.held == cache.seen == [48] * 3 and cache.pruned == [0] * 3 and (cache.seq_lens == 48).all()
    for t, old in zip([t.view(I8) for i in range(3) for t in (*cache.pools[i], *cache.weights[i])], was):
        assert torch.equal(t, old)
    cache.append(0, 2, 2, cache.packed(2), good, good)
    assert cache.held == [32, 48, 48] and cache.pruned[0] == 48


@pytest.mark.parametrize("quant", [False, True])
def test_a_prompts_weights_are_the_layers_own(lm, quant):
    """Whatever the layers before gathered, to the bit; and the cascade's sums are those of a
    model without such a cache."""
    from spatten_b200.qwen3 import PagedQwen3Cache
    attn = lm.model.layers[1].self_attn
    attn.enable_prog_quant = quant
    S, hidden = 40, lm.config.hidden_size
    g = torch.Generator().manual_seed(9)
    x = torch.randn(1, S, hidden, generator=g).to(BF16).cuda()
    rope = lm.model.rotary_emb(x, torch.arange(S, device="cuda")[None])
    past = torch.exp(4 * torch.randn(1, S, generator=g)).cuda() * 1e4
    want, sums = None, None
    for cumulative, cached in ((None, True), (past, True), (past, False)):
        attn.cascade.positions = torch.arange(S, device="cuda")[None]
        attn.cascade.cumulative = cumulative
        cache = PagedQwen3Cache(lm.config, 1, 64, page_size=16, keep_tokens=40) if cached else None
        attn(x, rope, past_key_values=cache)
        if cached:
            got = cache.weights[1].weight.clone()
            assert want is None or torch.equal(got, want)
            want = got
        if cumulative is not None:
            assert sums is None or torch.equal(attn.token_importance, sums)
            sums = attn.token_importance
