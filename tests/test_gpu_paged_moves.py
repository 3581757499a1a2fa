"""Tokens that move in the paged 8-bit KV cache (eviction, accepted tokens) where a
scale, a page table or a pool is far from the ordinary, against the oracle to the
bounds of tests/test_gpu_paged_tokens.py."""
import pytest
import torch

from oracle import paged as O
from oracle import paged_tokens as OT
from tests.test_gpu_paged import BF16, E4, I8, _cpu, _filled, _i32, _table
from tests.test_gpu_paged_tokens import _check_moved, _evicted, _weights

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


@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("recent", [0, 9])
@pytest.mark.parametrize("kv,D,page,G,lens,keep", [
    (I8, 64, 16, 3, [300, 40, 129, 0, 500, 65, 64, 70], 64),
    (E4, 128, 64, 2, [700, 1000, 333], 256),
    (I8, 64, 32, 1, [9000, 5000], 3000),             # several CTAs a sequence
    (E4, 64, 128, 1, [60000, 1000, 45000], 40000),
])
def test_evict_with_tables_wider_than_the_pool(kv, D, page, G, lens, keep, recent, per_head):
    """Tables with many times the pool's slots: what a call keeps for them lies like the pool."""
    g = torch.Generator().manual_seed(keep)
    mp = max(lens) // page + 1
    need = [-(-n // page) for n in lens]
    P = sum(need) + 1
    cache = _filled(kv, P, G, page, D, g)
    table = torch.full((len(lens), min(max(20 * mp, 5000), (1 << 20) // page)), -1, dtype=torch.int32)
    perm = torch.randperm(P, generator=g).to(torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = perm[sum(need[:b]):sum(need[:b]) + n]
    _evicted(cache, _weights(cache, g), table, lens, keep, recent=recent, per_head=per_head)


def test_evict_of_sequences_that_share_a_prefix():
    """A page that all of them keep is common to them; a sequence that lacks a page is left alone."""
    g = torch.Generator().manual_seed(62)
    G, D, page, lens, keep = 2, 64, 16, [90, 70, 64, 33, 80], 32
    P = 30
    cache, table = _filled(I8, P, G, page, D, g), torch.full((5, 400), -1, dtype=torch.int32)
    table[:, 0] = 7
    free = iter(p for p in torch.randperm(P, generator=g).tolist() if p != 7)
    for b, n in enumerate(lens):
        for i in range(1, -(-n // page)):
            table[b, i] = next(free)
    table[4, 2] = -1
    w = _weights(cache, g)
    w.weight[7] += 1e6
    for _ in range(2):  # (the second finds nothing but that sequence to do)
        moves = _evicted(cache, w, table, lens, keep, recent=3)
        assert not any(to < page for m in moves for to, _ in m[0]) and not moves[4][0]
        lens = [min(n, keep) if b < 4 else n for b, n in enumerate(lens)]


def test_wide_tables_captured_and_replayed():
    """The places of the lists start over with every call."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(63)
    G, D, page, lens, keep = 2, 64, 16, [200, 150, 90], 64
    cache = _filled(E4, 40, G, page, D, g)
    table = torch.full((3, 900), -1, dtype=torch.int32)
    table[:, :13] = torch.randperm(39, generator=g).view(3, 13)
    w, table_d, lens_d = _weights(cache, g), table.cuda(), _i32(lens)
    was = [t.clone() for t in (*cache, *w)]
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        new = paged.paged_evict(cache, w, table_d, lens_d, keep, per_head=True)
    want = None
    for _ in range(4):
        for t, old in zip((*cache, *w), was):
            t.view(torch.uint8).copy_(old.view(torch.uint8))
        gr.replay()
        assert new.tolist() == [keep] * 3
        got = [t.clone().view(torch.uint8) for t in (*cache, *w)]
        assert want is None or all(torch.equal(a, b) for a, b in zip(got, want))
        want = got
