"""HF's generation modes that change a cache, over the paged 8-bit cache: with
drafted tokens the rejected ones leave it (crop), with beams each sequence goes
on from its parent's keys (reorder_cache)."""
import pytest
import torch

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
    return patch_qwen3(Qwen3ForCausalLM(qwen3_model.config).to("cuda", torch.bfloat16).eval())


def _held(cache, layer):
    from spatten_b200 import paged
    return paged.paged_read(cache.pools[layer], cache.page_table, cache.seq_lens[layer],
                            n_tokens=cache.held[layer])


def test_drafted_tokens(lm, monkeypatch):
    """The first layer's keys depend on the tokens alone: after generation with
    drafts that were rejected, its slots hold those of the text, as a cache that
    was given the text at once does, to the roundings of their pages' scales: half
    a step when they are rounded and half for each time that a later token of the
    page raises the scale."""
    from spatten_b200.qwen3 import PagedQwen3Cache
    page, S, n = 16, 40, 30
    ids = torch.randint(0, 50, (1, 10), generator=torch.Generator().manual_seed(1)).repeat(1, S // 10).cuda()
    cache, dropped = PagedQwen3Cache(lm.config, 1, 128, page_size=page), []
    crop = cache.crop

    def recorded(length):
        dropped.append(cache.get_seq_length() - length)
        crop(length)
        assert cache.get_seq_length() == length and (cache.seq_lens == length).all()
    monkeypatch.setattr(cache, "crop", recorded)
    out = lm.generate(ids, attention_mask=torch.ones_like(ids), past_key_values=cache, max_new_tokens=n, min_new_tokens=n,
                      do_sample=False, eos_token_id=999, pad_token_id=0, prompt_lookup_num_tokens=4)
    assert out.shape == (1, S + n) and torch.equal(out[:, :S], ids)
    assert max(dropped) > 0  # some drafts were rejected
    held = cache.held[0]
    assert S + n - 5 <= held <= S + n and cache.held == [held] * len(cache.held)
    want = PagedQwen3Cache(lm.config, 1, 128, page_size=page)
    with torch.no_grad():
        lm(input_ids=out[:, :held], past_key_values=want, use_cache=True)
    for got, ref, scale in zip(_held(cache, 0), _held(want, 0), (cache.pools[0].k_scale, cache.pools[0].v_scale)):
        step = scale[:-(-held // page)].repeat_interleave(page, 0)[:held]  # a sequence's pages are in a row
        tol = (1 + (page + 4 * len(dropped)) / 2) * step[None, :, :, None] + 2.0 ** -7 * ref.abs()
        assert ((got - ref).abs() <= tol).all()
        # and no others' (where the neighbour is the same token, its value is the same too)
        other = ((got - ref.roll(1, 1)).abs() > tol).any(-1).all(-1)
        assert other[:, 1:][out[:, 1:held] != out[:, :held - 1]].all()


def test_beams(lm, monkeypatch):
    """Every reordering copies the parents' keys and values, of all layers;
    afterwards the beams write on pages of their own."""
    from spatten_b200.qwen3 import PagedQwen3Cache
    S, n, beams = 21, 12, 3
    ids = torch.randint(0, 1000, (1, S), generator=torch.Generator().manual_seed(2)).cuda()
    cache, moved = PagedQwen3Cache(lm.config, beams, 64, page_size=16, kv_dtype=torch.float8_e4m3fn), []
    reorder = cache.reorder_cache

    def checked(idx):
        before = [_held(cache, i) for i in range(len(cache.pools))]
        reorder(idx)
        moved.append(idx.tolist())
        for i, old in enumerate(before):
            assert all(torch.equal(a, b[idx]) for a, b in zip(_held(cache, i), old))
    monkeypatch.setattr(cache, "reorder_cache", checked)
    out = lm.generate(ids, attention_mask=torch.ones_like(ids), past_key_values=cache, max_new_tokens=n, min_new_tokens=n,
                      num_beams=beams, do_sample=False, eos_token_id=None, pad_token_id=0)
    assert out.shape == (1, S + n) and any(m != list(range(beams)) for m in moved)
    assert cache.page_table.unique().numel() == cache.page_table.numel()
