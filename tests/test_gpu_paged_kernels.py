"""Which of the paged attention's kernels a causal call takes goes by its query rows
alone; the kernel for pieces at the rows, values and tables where it takes over."""
import random

import pytest
import torch

from oracle import paged as O
from tests.test_gpu_paged import BF16, E4, F16, I8, _check_attend, _cum, _device_error, _filled, _i32, _table
from tests.test_gpu_paged_tokens import _check, _weights, _wide

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


@pytest.mark.parametrize("kv", [I8, E4])
@pytest.mark.parametrize("R,news", [(4, [24]), (4, [17]), (1, [65, 128]), (2, [40, 1, 33]), (16, [8]), (4, [16, 16]), (7, [9] * 3)])
def test_bits_do_not_change_with_the_tables_width(kv, R, news):
    """65 to 128 query rows per KV head, beside shorter sequences, and 49 to 64 where all
    have as many."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(R)
    G, D, page, B = 2, 128, 64, len(news)
    lens = [n + 700 - 100 * b for b, n in enumerate(news)]
    cu, mp = _cum(news), 13
    cache, table = _filled(kv, B * mp, G, page, D, g), _table(B, mp, B * mp, g)
    q = torch.randn(cu[-1], G * R, D, generator=g).to(BF16).cuda()
    big = [b for b, n in enumerate(news) if n * R > 64 or len(set(news)) == 1]
    call = lambda t: paged.paged_attention(q, cache, t.cuda(), _i32(cu), _i32(lens), max(news))  # noqa: E731
    out, wide = call(table), call(_wide(table, page))
    for b in big:  # (the few-row kernel splits its work by the launch, which the table's width bounds)
        assert torch.equal(out[cu[b]:cu[b + 1]], wide[cu[b]:cu[b + 1]])
    _check_attend(out, q, cache, table, cu, lens, D ** -0.5)
    assert _device_error() == 0


# ------------------------------------------------------------------ 49 to 64 rows, all sequences alike

@pytest.mark.parametrize("kv", [I8, E4])
@pytest.mark.parametrize("T", [25, 32])
@pytest.mark.parametrize("dt,outlier", [(BF16, 40.0), (F16, 60000.0)])
def test_outlier_channels(kv, T, dt, outlier):
    from tests.test_gpu_paged_numerics import test_outlier_channels as check
    check(kv, dt, outlier, T)


@pytest.mark.parametrize("kv", [I8, E4])
@pytest.mark.parametrize("D,R,T", [(64, 2, 25), (128, 4, 16), (128, 1, 64)])
def test_rows_of_all_kinds(kv, D, R, T):
    from tests.test_gpu_paged_numerics import test_rows_of_all_kinds_side_by_side as check
    check(kv, D, R, T)


@pytest.mark.parametrize("kv", [I8, E4])
@pytest.mark.parametrize("T", [13, 16])
@pytest.mark.parametrize("below", [18.0, 29.0])
def test_weak_keys_beside_a_strong_one(kv, T, below):
    from tests.test_gpu_paged_numerics import test_many_weak_keys_beside_a_strong_one as check
    check(kv, T, below)


@pytest.mark.parametrize("kv,D,page,G,R", [(I8, 128, 64, 2, 4), (E4, 64, 16, 1, 8), (I8, 64, 32, 2, 1), (E4, 128, 128, 1, 3)])
@pytest.mark.parametrize("rows", [48, 49, 56, 64])
@pytest.mark.parametrize("weigh,wide", [(False, False), (True, False), (True, True)])
def test_equal_pieces(kv, D, page, G, R, rows, weigh, wide):
    """Every sequence brings as many tokens, over contexts that end anywhere, one without any."""
    from spatten_b200 import paged
    g, rng = torch.Generator().manual_seed(rows), random.Random(R)
    n, B = -(-rows // R), 5
    lens = [n, n + 1] + [n + rng.randint(2, 500) for _ in range(B - 2)]
    cu, mp = _cum([n] * B), max(lens) // page + 2
    cache, table = _filled(kv, B * mp, G, page, D, g), _table(B, mp, B * mp, g)
    table[3, 1] = -1
    table = _wide(table, page) if wide else table
    q = torch.randn(cu[-1], G * R, D, generator=g).to(F16 if kv == E4 else BF16).cuda()
    w = _weights(cache, g) if weigh else None
    before = paged.PagedWeights(*(t.clone() for t in w)) if weigh else None
    out = paged.paged_attention(q, cache, table.cuda(), _i32(cu), _i32(lens), n, weights=w)
    _check(out, q, cache, table, cu, lens, D ** -0.5, None, before, w)
    assert _device_error() == 0


# ------------------------------------------------------------------ weights of many rows in many sequences

@pytest.mark.parametrize("B,G,R,news", [(600, 2, 16, (3, 4)), (1501, 1, 16, (0, 3, 5)), (8192, 1, 12, (3,)),
                                        (1500, 1, 40, (0, 1, 2))])
def test_weights_of_many_rows_in_many_sequences(B, G, R, news):
    """More than 32 query rows per KV head, sequences without tokens among them, batches of more
    pairs than the threads that number them; every slot against fp64."""
    from spatten_b200 import paged
    g, rng = torch.Generator().manual_seed(B), random.Random(B)
    D, page, cols = 64, 16, 4
    new = [rng.choice(news) for _ in range(B)]
    new[0] = new[-1] = max(news)
    lens = [n + rng.randint(0, 59) for n in new]
    cu, n_max, T = _cum(new), max(new), sum(new)
    cache = _filled(E4, cols * B, G, page, D, g)
    table = torch.randperm(cols * B, generator=g).to(torch.int32).view(B, cols)
    q = torch.randn(T, G * R, D, generator=g).to(BF16).cuda()
    w = _weights(cache, g)
    before = paged.PagedWeights(*(t.clone() for t in w))
    args = (q, cache, table.cuda(), _i32(cu), _i32(lens), n_max)
    out = paged.paged_attention(*args, weights=w)
    assert torch.equal(out, paged.paged_attention(*args)) and _device_error() == 0
    at = table.long().cuda()
    flat = lambda t: t[at].transpose(1, 2).reshape(B, G, cols * page)  # noqa: E731
    codes = O.code_values(cache.k.view(I8).cpu().view(E4)).cuda()
    k = (codes[at] * cache.k_scale[at].double()[..., None, None]).transpose(1, 2).reshape(B, G, cols * page, D)
    length, count = torch.tensor(lens).cuda(), torch.tensor(new).cuda()
    slot = torch.arange(cols * page, device="cuda")
    gained, err = torch.zeros(2, B, G, cols * page, dtype=torch.float64, device="cuda")
    for i in range(n_max):
        live = count > i
        row = (torch.tensor(cu[:-1]).cuda() + i).clamp(max=T - 1)
        x = q[row].double().view(B, G, R, D)
        seen = (slot < (length - count + i + 1)[:, None])[:, None, None] & live[:, None, None, None]
        s = (x @ k.transpose(2, 3) * D ** -0.5).masked_fill(~seen, float("-inf"))
        p = torch.softmax(s, -1).nan_to_num(0.0)
        S = (x.abs() @ k.abs().transpose(2, 3) * D ** -0.5).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
        gained += p.sum(2)
        err += (p * S).sum(2)
    old = (slot < (length - count)[:, None])[:, None]
    fresh = (slot < length[:, None])[:, None] & ~old & (count > 0)[:, None, None]
    was = flat(before.weight).double()
    want = torch.where(fresh, torch.zeros_like(was), was) + gained
    tol = 2 * D * 2.0 ** -24 * err + want * (3 * 2.0 ** -16) + 1e-37
    assert ((flat(w.weight).double() - want).abs() <= tol).all()
    assert torch.equal(flat(w.position), torch.where(fresh, slot.int().expand(B, G, -1), flat(before.position)))


@pytest.mark.parametrize("n,R", [(1, 2), (40, 2)])
def test_weights_past_2_32_bytes(n, R):
    """A pool of more than 2^30 rows, its last pages in use: weights and positions lie beyond
    2^32 bytes, codes beyond 2^36; then eviction and accepted tokens there."""
    from oracle import paged_tokens as OT
    from spatten_b200 import paged
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 100e9:
        pytest.skip("needs 77 GB of a GPU's memory")
    g = torch.Generator().manual_seed(81)
    G, D, page, L, mp = 1, 64, 128, 700, 7
    P = (1 << 30) // page + 100
    codes = torch.empty(P, G, page, D, dtype=I8, device="cuda")  # K and V alike: one pool for both
    scale = torch.ones(P, G, device="cuda")
    cache = paged.PagedKVCache(codes, codes, scale, scale)
    w = paged.new_paged_weights(cache)
    small = _filled(I8, mp, G, page, D, g)
    small = paged.PagedKVCache(small.k, small.k, small.k_scale, small.k_scale)
    ws = _weights(small, g)
    order = torch.randperm(mp, generator=g)
    table, near = (P - mp + order).to(torch.int32)[None], order.to(torch.int32)[None]
    codes[P - mp:], scale[P - mp:] = small.k, small.k_scale
    for big, part in zip(w, ws):
        big[P - mp:] = part
    q = torch.randn(n, G * R, D, generator=g).to(BF16).cuda()
    before = paged.PagedWeights(*(t.clone() for t in ws))
    out = paged.paged_attention(q, cache, table.cuda(), _i32([0, n]), _i32([L]), n, weights=w)
    after = paged.PagedWeights(*(t[P - mp:].clone() for t in w))
    _check(out, q, small, near, [0, n], [L], D ** -0.5, None, before, after)
    moves, new = OT.evict([t.cpu() for t in small], after.weight.cpu(), after.position.cpu(), near, [L], 300, recent=50)
    assert paged.paged_evict(cache, w, table.cuda(), _i32([L]), 300, recent=50).tolist() == new == [300]
    for got, t in zip(w, after):
        assert torch.equal(got[P - mp:].cpu(), OT.move_beside(t.cpu(), near, moves))
    after = paged.PagedWeights(*(t[P - mp:].clone() for t in w))
    moves, new = OT.keep([t.cpu() for t in small], near, [0, 40], [300], [[0, 7, 9, 30]])
    assert paged.paged_keep(cache, table.cuda(), _i32([0, 40]), _i32([300]), _i32([[0, 7, 9, 30]]), weights=w).tolist() == new
    for got, t in zip(w, after):
        assert torch.equal(got[P - mp:].cpu(), OT.move_beside(t.cpu(), near, moves))
    assert (w.weight[:P - mp] == 0).all() and (w.position[:P - mp] == 0).all()
    del codes, cache, w
    torch.cuda.empty_cache()
