"""Generation with the Qwen3 drop-in over the paged 8-bit cache: every layer's
extension step against the float64 oracle, fed the layer's own projections.
The tolerances are those of tests/test_gpu_paged.py; q and k come out of an
RMS norm, so their rotation's roundings are relative to the row's largest
element."""
import pytest
import torch

from oracle import paged as O
from tests.test_gpu_paged import _check_append, _check_attend, _cpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


@pytest.fixture()
def patched(qwen3_model):
    import copy
    from spatten_b200.qwen3 import patch_qwen3

    def make(**knobs):
        return patch_qwen3(copy.deepcopy(qwen3_model).to("cuda", torch.bfloat16), **knobs)
    return make


@pytest.mark.parametrize("knobs,kv,pieces", [
    ({}, torch.int8, [1, 1]),
    ({"enable_token_prune": True, "token_keep_ratio": 0.6, "enable_prog_quant": True}, torch.int8, [1, 3, 1]),
    ({"enable_token_prune": True, "token_keep_ratio": 0.8}, torch.float8_e4m3fn, [40, 1]),
])
def test_generation_steps_match_oracle(patched, monkeypatch, knobs, kv, pieces):
    from spatten_b200 import paged, qwen3
    model = patched(**knobs)
    cfg, B, S = model.config, 2, 70
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(0, 1000, (B, S + sum(pieces)), generator=g).cuda()
    cache = qwen3.PagedQwen3Cache(cfg, B, 200, page_size=32, kv_dtype=kv)
    model(input_ids=ids[:, :S], past_key_values=cache, use_cache=True)
    kept = model.layers[0].self_attn.cascade.kept_per_layer
    assert cache.get_seq_length() == S and cache.held == kept and cache.seq_lens[:, 0].tolist() == kept
    at, seen = S, []
    append, attend = paged.paged_append, paged.paged_attention

    def check_append(pool, k, v, table, cu, lens, mx, **kw):
        before = _cpu(pool)
        out = append(pool, k, v, table, cu, lens, mx, **kw)
        pos = kw["positions"].tolist()
        want = O.append(before, k.cpu(), v.cpu(), table.cpu(), cu.tolist(), lens.tolist(), q=kw["q"].cpu(),
                        cos=kw["cos"].cpu(), sin=kw["sin"].cpu(), positions=pos, wq=kw["q_norm_w"].cpu(),
                        wk=kw["k_norm_w"].cpu(), eps=kw["eps"])
        _check_append(pool, before, want, out)
        # the tables' rows are the tokens' positions in the text, not their slots
        n = len(pos) // B
        cos, _ = model.rotary_emb(k, torch.arange(at, at + n, device="cuda")[None])
        assert torch.equal(kw["cos"][kw["positions"].long()].view(B, n, -1), cos.expand(B, -1, -1))
        return out

    def check_attend(q, pool, table, cu, lens, mx, sm_scale=None):
        out = attend(q, pool, table, cu, lens, mx, sm_scale=sm_scale)
        _check_attend(out, q, pool, table.cpu(), cu.tolist(), lens.tolist(), sm_scale)
        seen.append(lens.tolist())
        return out

    monkeypatch.setattr(paged, "paged_append", check_append)
    monkeypatch.setattr(paged, "paged_attention", check_attend)
    for n in pieces:
        out = model(input_ids=ids[:, at:at + n], past_key_values=cache, use_cache=True).last_hidden_state
        assert out.shape == (B, n, cfg.hidden_size) and torch.isfinite(out).all()
        at += n
        assert cache.get_seq_length() == at and cache.get_mask_sizes(1) == (at + 1, 0)
        assert seen[-len(kept):] == [[k + at - S] * B for k in kept]
    assert len(seen) == len(pieces) * len(kept)


def test_cache_refusals_and_reset(patched):
    from transformers import DynamicCache
    from spatten_b200 import qwen3
    model = patched()
    ids = torch.arange(12, device="cuda")[None] % 7
    cache = qwen3.PagedQwen3Cache(model.config, 1, 14, page_size=16)
    model(input_ids=ids, past_key_values=cache, use_cache=True)
    first = model(input_ids=ids[:, :2], past_key_values=cache, use_cache=True).last_hidden_state
    with pytest.raises(ValueError, match="room for 14"):
        model(input_ids=ids[:, :1], past_key_values=cache, use_cache=True)
    with pytest.raises(NotImplementedError, match="SpattenQwen3Attention only"):
        cache.update(torch.zeros(1), torch.zeros(1), 0)
    cache.reset()
    assert cache.get_seq_length() == 0
    model(input_ids=ids, past_key_values=cache, use_cache=True)
    assert torch.equal(model(input_ids=ids[:, :2], past_key_values=cache, use_cache=True).last_hidden_state, first)
    with pytest.raises(ValueError, match="made for 1"):
        model(input_ids=ids[:, :1].repeat(2, 1), past_key_values=cache, use_cache=True)
    dense = DynamicCache(config=model.config)
    model(input_ids=ids, past_key_values=dense, use_cache=True)
    with pytest.raises(NotImplementedError, match="PagedQwen3Cache"):
        model(input_ids=ids[:, :1], past_key_values=dense, use_cache=True)


def test_torch_ops_match_python():
    import spatten_b200.torch_ops  # noqa: F401
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(1)
    c = [paged.new_paged_cache(6, 2, 64, page_size=16) for _ in range(2)]
    k, v, q = (torch.randn(20, n, 64, generator=g).half().cuda() for n in (2, 2, 4))
    t, cu, ln = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([[4, 1]], [0, 20], [20]))
    idx = torch.tensor([[3, 19, 40]], device="cuda")
    torch.ops.spatten.paged_append(*c[0], k, v, t, cu, ln, 20)
    paged.paged_append(c[1], k, v, t, cu, ln, 20)
    assert all(torch.equal(a, b) for a, b in zip(*c))
    assert torch.equal(torch.ops.spatten.paged_attention(q, *c[0], t, cu, ln, 20, 0.1),
                       paged.paged_attention(q, c[1], t, cu, ln, 20, sm_scale=0.1))
    for a, b in zip(torch.ops.spatten.paged_read(*c[0], t, ln, idx), paged.paged_read(c[1], t, ln, idx=idx)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("knobs", [{}, {"enable_token_prune": True, "token_keep_ratio": 0.7}])
def test_generate(qwen3_model, knobs):
    """HF's generate over the paged cache: the tokens that a loop of forwards
    over another paged cache picks."""
    from transformers import Qwen3ForCausalLM
    from spatten_b200.qwen3 import PagedQwen3Cache, patch_qwen3
    torch.manual_seed(0)
    lm = patch_qwen3(Qwen3ForCausalLM(qwen3_model.config).to("cuda", torch.bfloat16).eval(), **knobs)
    cfg = lm.config
    ids = torch.randint(0, cfg.vocab_size, (2, 33), device="cuda")
    cache = PagedQwen3Cache(cfg, 2, 64, page_size=16)
    out = lm.generate(ids, attention_mask=torch.ones_like(ids), past_key_values=cache, max_new_tokens=9, do_sample=False,
                      eos_token_id=None, pad_token_id=0)
    assert out.shape == (2, 42) and torch.equal(out[:, :33], ids) and cache.get_seq_length() == 41
    want, new, cache = ids, ids, PagedQwen3Cache(cfg, 2, 64, page_size=16)
    with torch.no_grad():
        for _ in range(9):
            logits = lm(input_ids=new, past_key_values=cache, use_cache=True, logits_to_keep=1).logits
            new = logits[:, -1:].argmax(-1)
            want = torch.cat([want, new], 1)
    assert torch.equal(out, want)
