"""Tokens that move in the paged 8-bit KV cache (eviction, accepted tokens) where a
scale, a page table or a pool is far from the ordinary, against the oracle to the
bounds of tests/test_gpu_paged_tokens.py."""
import pytest
import torch

from oracle import paged as O
from oracle import paged_tokens as OT
from tests.test_gpu_paged import BF16, E4, I8, _cpu, _i32, _table
from tests.test_gpu_paged_tokens import _check_moved, _evicted

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


@pytest.mark.parametrize("kv", [I8, E4])
@pytest.mark.parametrize("op", ["evict", "keep"])
def test_zeros_between_scales_far_apart(kv, op):
    """A row of zeros out of a page whose scale is more than 2^128 times that of the page
    it comes to: zeros still, as 0 times any finite ratio, and the others as they were."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(61)
    G, D, page, n = 2, 64, 16, 32
    cache, table = paged.new_paged_cache(3, G, D, page_size=page, kv_dtype=kv), _table(1, 2, 3, g)
    x = torch.randn(n, 2 * G, D, generator=g)
    x[:page] *= 1e-37
    x[page:] *= 5000.0
    x[17] = 0
    x = x.to(BF16).cuda()
    paged.paged_append(cache, x[:, :G], x[:, G:], table.cuda(), _i32([0, n]), _i32([n]), n)
    tiny, large = (float(cache.k_scale[int(table[0, i])].max()) for i in range(2))
    assert large > 0 and tiny > 0 and large > tiny * 2.0 ** 64 * 2.0 ** 64
    if op == "evict":
        w = paged.new_paged_weights(cache)
        w.weight.fill_(1.0)
        w.weight[int(table[0, 0]), :, 15] = 0.0     # the zeros take the last place of the first page
        w.weight[int(table[0, 1])] = 0.0
        w.weight[int(table[0, 1]), :, 1] = 2.0
        assert _evicted(cache, w, table, [n], page) == [[[(15, 17)]] * G]
    else:
        before = _cpu(cache)
        got = paged.paged_keep(cache, table.cuda(), _i32([0, 18]), _i32([n]), _i32([[0, 3]]))  # slots 14 .. 31
        moves, new = OT.keep(before, table, [0, 18], [n], [[0, 3]])
        assert got.tolist() == new == [page] and moves == [[[(15, 17)]] * G]
        _check_moved(cache, before, table, moves, new)
    for codes, scale in zip(cache[:2], cache[2:]):
        page0 = O.code_values(_cpu([codes])[0])[int(table[0, 0])]
        assert (page0[:, 15] == 0).all() and (page0[:, :14] != 0).any(-1).all()
        assert float(scale[int(table[0, 0])].max()) < 1e-30
