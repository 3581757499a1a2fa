"""GPU parity of trees of drafted tokens and of eviction over the paged 8-bit
KV cache (spatten_b200.paged) against the float64 oracle (oracle/paged_tokens.py).

Tolerances (u = 2^-24): attention as in test_gpu_paged.py. A weight is a sum over
rows of p = exp(s - max) / l: each p carries the rounding of its score and of
those in l (D u S each, relative to p), 2^-16 for the exponentials and the fp32 sum l;
the sum over rows and the weight before it 2^-16 and u of the result (at most 2^8
rounded additions one after another, or fewer per partial sum). A moved token's
code is round(code * S_old / S), two roundings of a value of at most 127 (int8;
the scales of e4m3 are powers of two and exact), so within 127 * 4 u = 3.1e-5 of
the border's side that 64 bits take, up to twice.
"""
import itertools
import random

import pytest
import torch

from oracle import paged as O
from oracle import paged_tokens as OT
from tests.test_gpu_paged import BF16, E4, F16, I8, U, _cpu, _cum, _filled, _i32, _table

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _random_tree(n, rng, width=3):
    return [-1 if i == 0 or rng.random() < 0.05 else rng.randint(max(0, i - width), i - 1) for i in range(n)]


def _weights(cache, g):
    from spatten_b200 import paged
    w = paged.new_paged_weights(cache)
    x = torch.exp(2 * torch.randn(w.weight.shape, generator=g))
    w.weight.copy_(torch.where(torch.rand(x.shape, generator=g) < 0.1, torch.zeros(()), x))
    w.position.copy_(torch.randint(0, 1000, w.position.shape, generator=g))
    return w


def _wide(table, page):
    """The table with columns behind the sequences' (300000 slots: calls of more than a few
    query rows go to the tcgen05 kernel, which small work over a narrow table does not)."""
    return torch.cat([table, torch.full((table.shape[0], 300000 // page), -1, dtype=torch.int32)], 1)


def _check(out, q, cache, table, cu, lens, sm, sees, before=None, after=None, positions=None, max_tokens=None):
    """Outputs, and with the pools ``before`` and ``after`` the weights and positions."""
    c = _cpu(cache)
    want, A, S, weight, err = OT.attend(q.cpu(), c, table, cu, lens, sm, sees, max_tokens)
    D = q.shape[-1]
    tol = torch.finfo(out.dtype).eps / 2 * want.abs() + A * (2.0 ** -11 + 2 * D * U * S + 2.0 ** -16) + \
        max(lens) * U * A.amax(-1, keepdim=True) + torch.finfo(out.dtype).smallest_normal
    rows = [t for b in range(len(lens)) for t in range(cu[b], min(cu[b + 1], cu[b] + (max_tokens or 1 << 30)))]
    bad = ((out.cpu().double() - want).abs() > tol)[rows]
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())
    if before is None:
        return want
    P, G, page = before.weight.shape
    w, p, dw = before.weight.double().cpu().clone(), before.position.cpu().clone(), torch.zeros(P, G, page).double()
    for b in range(len(lens)):
        n = cu[b + 1] - cu[b]
        m = n if max_tokens is None else min(n, max_tokens)
        for s in range(min(lens[b] - n + m, lens[b]) if n else 0):
            pid = int(table[b, s // page]) if s // page < table.shape[1] else -1
            if not 0 <= pid < P:
                continue
            if s >= lens[b] - n:
                w[pid, :, s % page] = 0
                t = cu[b] + s - (lens[b] - n)
                p[pid, :, s % page] = s if positions is None else positions[t]
            w[pid, :, s % page] += weight[b][:, s]
            dw[pid, :, s % page] = err[b][:, s]
    tol = 2 * D * U * dw + w * (3 * 2.0 ** -16) + 1e-37
    bad = (after.weight.double().cpu() - w).abs() > tol
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())
    assert torch.equal(after.position.cpu(), p)
    return want


# ------------------------------------------------------------------ trees

@pytest.mark.parametrize("news", [[1], [26], [64, 1, 0, 33, 32, 31], [1024, 5], [200] * 40])
def test_tree(news):
    from spatten_b200 import paged
    rng = random.Random(sum(news))
    cu, lens = _cum(news), [n + rng.randint(0, 500) for n in news]
    parents = [p for n in news for p in _random_tree(n, rng, width=rng.choice([1, 3]))]
    tree, pos = paged.paged_tree(_i32(parents), _i32(cu), _i32(lens), max(news))
    sees, want = OT.tree(parents, cu, lens, max(news))
    assert torch.equal(tree.cpu(), OT.words(sees, cu[-1], -(-max(news) // 32)))
    assert pos.tolist() == [want[t] for t in range(cu[-1])]


def test_tree_rows_and_values_out_of_range():
    """A chain of 1024; parents that are no earlier token; rows behind max_tokens and
    behind the last sequence stay as they are; sequences whose bounds descend bring none."""
    from spatten_b200 import _native as N
    from spatten_b200 import paged
    n = 1024
    tree, pos = paged.paged_tree(_i32(list(range(-1, n - 1))), _i32([0, n]), _i32([n + 7]), n)
    assert pos.tolist() == list(range(7, n + 7))
    bits = (tree.cpu().long()[:, :, None] >> torch.arange(32)) & 1
    assert torch.equal(bits.view(n, n), torch.ones(n, n, dtype=torch.long).tril())
    # b0: 5 tokens of which 3 are laid out; b1's bounds descend; b2's leave the rows; b3: fewer held than rows
    parents = _i32([5, 0, 9, 1, 1, -7, 0, 0, 2 ** 31 - 1, 0])
    cu, lens = _i32([0, 5, 3, 20, 5, 8]), _i32([9, 9, 9, 9, 1])
    a = N.PagedTreeArgs()
    tree = torch.full((10, 2), 77, dtype=torch.int32, device="cuda")
    pos = torch.full((10,), 77, dtype=torch.int32, device="cuda")
    a.B, a.T, a.max_tokens, a.tree_words, a.tree_stride = 5, 10, 3, 1, 2
    a.cu_tokens, a.seq_lens, a.parents = cu.data_ptr(), lens.data_ptr(), parents.data_ptr()
    a.tree, a.positions = tree.data_ptr(), pos.data_ptr()
    N.check(N.lib.spatten_paged_tree(a, torch.cuda.current_stream().cuda_stream))
    want = [1, 3, 4, 77, 77, 1, 3, 5, 77, 77]
    assert tree[:, 0].tolist() == want and (tree[:, 1] == 77).all()
    assert pos.tolist() == [4, 5, 4, 77, 77, -2, -1, -1, 77, 77]


TREES = [
    (I8, BF16, 128, 64, 2, 4, [26], [777]),                     # tcgen05
    (I8, BF16, 128, 64, 2, 1, [26, 1, 8], [26, 40, 300]),        # few rows, empty context
    (E4, F16, 64, 16, 2, 3, [3, 17, 0, 9], [20, 17, 5, 129]),
    (E4, F16, 128, 32, 1, 2, [40, 2, 33], [333, 64, 35]),        # both kernels in one call
    (I8, F16, 64, 128, 1, 8, [64, 70], [200, 70]),
    (E4, BF16, 128, 16, 1, 5, [120, 13], [250, 300]),            # several row tiles
    (I8, BF16, 64, 32, 3, 1, [8, 5, 1], [31, 32, 33]),
    (I8, F16, 128, 16, 1, 16, [7], [50]),
]


@pytest.mark.parametrize("kv,dt,D,page,G,R,news,lens", TREES)
@pytest.mark.parametrize("weigh", [False, True])
@pytest.mark.parametrize("wide", [False, True])
def test_tree_attention(kv, dt, D, page, G, R, news, lens, weigh, wide):
    """Trees of paged_tree, over contexts that end anywhere in a page or tile."""
    from spatten_b200 import paged
    g, rng = torch.Generator().manual_seed(len(news) + D), random.Random(5)
    mp = max(lens) // page + 2
    B, cu = len(lens), _cum(news)
    P = B * mp + 2
    cache, table = _filled(kv, P, G, page, D, g), _table(B, mp, P, g)
    table = _wide(table, page) if wide else table
    parents = [p for n in news for p in _random_tree(n, rng)]
    tree, pos = paged.paged_tree(_i32(parents), _i32(cu), _i32(lens), max(news))
    sees, _ = OT.tree(parents, cu, lens, max(news))
    q = torch.randn(cu[-1], G * R, D, generator=g).to(dt).cuda()
    w = _weights(cache, g) if weigh else None
    before = paged.PagedWeights(*(t.clone() for t in w)) if weigh else None
    out = paged.paged_attention(q, cache, table.cuda(), _i32(cu), _i32(lens), max(news), tree=tree, weights=w,
                                positions=pos if weigh else None)
    _check(out, q, cache, table, cu, lens, D ** -0.5, sees, before, w, pos.tolist())


@pytest.mark.parametrize("R,n", [(1, 5), (4, 40)])
@pytest.mark.parametrize("far", [False, True])
def test_masks_of_any_bits(R, n, far):
    """Words that name later tokens, none at all (an empty row, over an empty context
    too), bits behind the sequence's tokens, wide strided words; pages without
    memory in the context and among the new tokens."""
    from spatten_b200 import paged
    g, rng = torch.Generator().manual_seed(n), random.Random(n)
    G, D, page, H = 2, 64, 16, 2 * R
    news, lens = [n, n, n - 2, n], [n, n + 50, n + 14, n + 3]
    cu = _cum(news)
    mp = max(lens) // page + 2
    cache, table = _filled(I8, 30, G, page, D, g), _table(4, mp, 30, g)
    table[1, 1], table[2, 0], table[3, (n + 2) // page] = -1, 99, -5
    table = _wide(table, page) if far else table
    sees = {t: frozenset(j for j in range(64) if rng.random() < 0.4) for t in range(cu[-1])}
    for t in (0, 2, cu[1], cu[2] + 1):
        sees[t] = frozenset()
    sees[1] = frozenset(range(n, 64))  # no new token of its sequence
    W = 3
    wide = torch.zeros(cu[-1] + 4, 9, dtype=torch.int32, device="cuda")
    wide[:cu[-1], 2:2 + W] = OT.words(sees, cu[-1], W).cuda()
    q = torch.randn(cu[-1] + 4, H, D, generator=g).to(F16).cuda()
    w = _weights(cache, g)
    before = paged.PagedWeights(*(t.clone() for t in w))
    out = torch.full_like(q, 3.0)
    paged.paged_attention(q, cache, table.cuda(), _i32(cu), _i32(lens), n, out=out, tree=wide[:, 2:2 + W], weights=w)
    _check(out, q, cache, table, cu, lens, D ** -0.5, sees, before, w)
    assert (out[cu[-1]:] == 3).all()
    assert (out[0] == 0).all() and (out[1] == 0).all()  # empty context, nothing seen


@pytest.mark.parametrize("news,R", [([4], 2), ([70, 3], 1), ([33, 1], 4)])
def test_chain_is_causal(news, R):
    """A tree without branches gives the causal call's result."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(7)
    G, D, page = 2, 128, 32
    lens = [n + 61 for n in news]
    cu, mp = _cum(news), max(lens) // page + 1
    cache, table = _filled(I8, 20, G, page, D, g), _table(len(news), mp, 20, g).cuda()
    q = torch.randn(cu[-1], G * R, D, generator=g).to(BF16).cuda()
    args = (table, _i32(cu), _i32(lens), max(news))
    tree, pos = paged.paged_tree(_i32([i - 1 for n in news for i in range(n)]), *args[1:])
    assert pos.tolist() == [61 + i for n in news for i in range(n)]
    a, b = paged.paged_attention(q, cache, *args), paged.paged_attention(q, cache, *args, tree=tree)
    assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -7, atol=2.0 ** -9)


@pytest.mark.parametrize("kv", [I8, E4])
@pytest.mark.parametrize("R,n", [(4, 12), (7, 7), (4, 16), (1, 65), (4, 32), (3, 43), (16, 5)])
@pytest.mark.parametrize("wide,weigh", [(False, False), (True, False), (True, True)])
def test_causal_on_either_side_of_the_kernels(kv, R, n, wide, weigh):
    """48 to 129 query rows per KV head, over narrow and wide page tables, beside shorter ones."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(R * n)
    G, D, page, news, lens = 2, 128, 32, [n, 1, n - 1, 0, n], [n, 100, n + 33, 70, 450]
    cu, mp, B = _cum(news), 15, 5
    cache, table = _filled(kv, B * mp, G, page, D, g), _table(B, mp, B * mp, g)
    table = _wide(table, page) if wide else table
    q = torch.randn(cu[-1], G * R, D, generator=g).to(BF16).cuda()
    w = _weights(cache, g) if weigh else None
    before = paged.PagedWeights(*(t.clone() for t in w)) if weigh else None
    out = paged.paged_attention(q, cache, table.cuda(), _i32(cu), _i32(lens), n, weights=w)
    sees = {cu[b] + i: frozenset(range(i + 1)) for b in range(B) for i in range(news[b])}
    _check(out, q, cache, table, cu, lens, D ** -0.5, sees, before, w)


# ------------------------------------------------------------------ weights

@pytest.mark.parametrize("kv,dt,D,page,G,R,news,lens", [
    (I8, BF16, 128, 64, 2, 4, [1] * 6, [1, 31, 32, 33, 64, 700]),
    (E4, F16, 128, 16, 1, 1, [1] * 5, [1, 15, 16, 17, 333]),
    (E4, BF16, 64, 32, 3, 3, [1, 1, 1], [2, 129, 65]),
    (I8, F16, 64, 128, 1, 8, [1, 1], [127, 2500]),
    (I8, F16, 128, 64, 1, 16, [1, 1], [200, 90]),
    (E4, F16, 64, 16, 1, 40, [1, 1], [50, 31]),
    (I8, BF16, 64, 16, 2, 128, [1], [77]),
    (I8, BF16, 128, 32, 2, 5, [2, 7, 1, 3, 0], [2, 40, 9, 129, 10]),
    (E4, F16, 64, 64, 2, 2, [4, 8], [100, 8]),
    (I8, F16, 128, 64, 1, 2, [130, 1, 64], [300, 64, 64]),
    (E4, BF16, 64, 16, 2, 1, [257, 33], [257, 100]),
    (E4, BF16, 128, 128, 1, 8, [70, 200], [300, 201]),
    (I8, BF16, 64, 64, 2, 1, [9, 1], [1500, 700]),
])
def test_weights(kv, dt, D, page, G, R, news, lens):
    """Two calls in a row, the second with positions; the output is that of the
    call without weights."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(11)
    mp = max(lens) // page + 2
    B, cu = len(lens), _cum(news)
    P = B * mp + 1
    cache, table = _filled(kv, P, G, page, D, g), _table(B, mp, P, g)
    w = _weights(cache, g)
    for positions in (None, _i32(torch.randint(0, 10 ** 6, (cu[-1],), generator=g).tolist())):
        q = (torch.randn(cu[-1], G * R, D, generator=g) * (4 if positions is None else 1)).to(dt).cuda()
        before = paged.PagedWeights(*(t.clone() for t in w))
        args = (q, cache, table.cuda(), _i32(cu), _i32(lens), max(news))
        out = paged.paged_attention(*args, weights=w, positions=positions)
        assert torch.equal(out, paged.paged_attention(*args))
        _check(out, q, cache, table, cu, lens, D ** -0.5, None, before, w,
               None if positions is None else positions.tolist())


@pytest.mark.parametrize("R,n", [(1, 4), (2, 3), (4, 50)])
def test_weights_of_odd_batches(R, n):
    """More rows than max_tokens, fewer tokens held than rows, a page table that is too
    short, pages without memory, bounds that descend: only the slots of rows that are
    served change."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(13)
    G, D, page = 2, 64, 16
    news, lens = [n + 5, n, n, n, n, 0], [n + 40, 90, n - 2, n + 60, n, 9]
    cu = _cum(news)
    mp = 5
    cache, table = _filled(E4, 40, G, page, D, g), _table(6, mp, 40, g)
    table[1, 2], table[3, 0] = -1, 40
    w = _weights(cache, g)
    before = paged.PagedWeights(*(t.clone() for t in w))
    q = torch.randn(cu[-1], G * R, D, generator=g).to(F16).cuda()
    out = paged.paged_attention(q, cache, table.cuda(), _i32(cu), _i32(lens), n, weights=w)
    _check(out, q, cache, table, cu, lens, D ** -0.5, None, before, w, max_tokens=n)
    # descending bounds: the first sequence is left out
    before = paged.PagedWeights(*(t.clone() for t in w))
    bad = [cu[1]] + cu[1:]
    bad[1] = 0
    paged.paged_attention(q[:cu[1]], cache, table[:1].cuda(), _i32(bad[:2]), _i32(lens[:1]), n, weights=w)
    assert torch.equal(before.weight, w.weight) and torch.equal(before.position, w.position)


@pytest.mark.parametrize("n", [1, 40])
def test_weights_of_extreme_rows(n):
    """A NaN or an infinity in a query makes its head's weights NaN and no other's;
    queries of zeros spread evenly; scores far apart; codes and scales of zero."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(17)
    G, D, page, L = 4, 64, 16, 100
    cache, table = _filled(I8, 8, G, page, D, g), _table(1, 8, 8, g).cuda()
    cache.k_scale[:, 2] = 0
    q = torch.randn(n, 2 * G, D, generator=g).to(BF16)
    q[0, 0, 5] = float("nan")
    q[0, 3, 7] = float("inf")
    q[:, 6:] *= 1000.0
    w = paged.new_paged_weights(cache)
    paged.paged_attention(q.cuda(), cache, table, _i32([0, n]), _i32([L]), n, weights=w)
    got = w.weight[table[0].long()].transpose(0, 1).reshape(G, -1).cpu()
    first = L - n + 1  # slots that the odd row sees
    assert got[:2, :first].isnan().all() and not got[2:].isnan().any()
    assert (got[:, L:] == 0).all()
    even = sum(1.0 / (L - n + i + 1) for i in range(n)) * 2  # scores of 0
    assert torch.allclose(got[2, :first], torch.full((first,), even), rtol=1e-5)
    assert abs(float(got[3].sum()) - 2 * n) < 1e-3 * n


@pytest.mark.parametrize("n,R", [(1, 2), (3, 4), (80, 2)])
@pytest.mark.parametrize("scale", [None, 0.0, -0.25])
def test_weights_of_rows_far_apart(n, R, scale):
    """Query rows whose magnitudes lie 2^40 apart, some of zeros; a scale of 0 or below it."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(18)
    G, D, page, L = 2, 128, 32, 300
    cache, table = _filled(E4, 12, G, page, D, g), _table(1, 10, 12, g)
    q = torch.randn(n, G * R, D, generator=g)
    q *= 2.0 ** torch.randint(-35, 4, (n, G * R, 1), generator=g)
    q[n // 2, 0] = 0
    q = q.to(BF16).cuda()
    w = _weights(cache, g)
    before = paged.PagedWeights(*(t.clone() for t in w))
    args = (q, cache, table.cuda(), _i32([0, n]), _i32([L]), n)
    out = paged.paged_attention(*args, sm_scale=scale, weights=w)
    _check(out, q, cache, table, [0, n], [L], D ** -0.5 if scale is None else scale, None, before, w)


@pytest.mark.parametrize("news,R", [([1, 1, 1], 4), ([1, 1, 1], 1), ([3, 7, 1], 3), ([60, 1, 2], 2), ([90, 70, 130], 1)])
def test_weights_with_a_table_wider_than_the_pool(news, R):
    """Most of the page table has no memory: what a call keeps lies like the pool."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(21)
    G, D, page, lens = 2, 64, 16, [n + 70 for n in news]
    mp = max(lens) // page + 1
    cache = _filled(I8, 3 * mp, G, page, D, g)
    table = torch.cat([_table(3, mp, 3 * mp, g), torch.full((3, 500), -1, dtype=torch.int32)], 1)
    table[1, 2] = -1  # and a hole
    w, cu = _weights(cache, g), _cum(news)
    for _ in range(2):
        q = torch.randn(cu[-1], G * R, D, generator=g).to(BF16).cuda()
        before = paged.PagedWeights(*(t.clone() for t in w))
        out = paged.paged_attention(q, cache, table.cuda(), _i32(cu), _i32(lens), max(news), weights=w)
        _check(out, q, cache, table, cu, lens, D ** -0.5, None, before, w)


@pytest.mark.parametrize("B,R,G", [(5000, 16, 1), (8192, 2, 1), (3, 1, 12), (700, 9, 3)])
def test_weights_of_many_sequences_and_heads(B, R, G):
    """Each row gives a weight of 1 in all; the output is the plain call's."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(25)
    D, page = 64, 16
    lens = [rng % 61 + 1 for rng in torch.randint(0, 1 << 20, (B,), generator=g).tolist()]
    cache = _filled(E4, 4 * B, G, page, D, g)
    table = torch.arange(4 * B, dtype=torch.int32).view(B, 4).cuda()
    q = torch.randn(B, G * R, D, generator=g).to(BF16).cuda()
    w = _weights(cache, g)
    args = (q, cache, table, _i32(list(range(B + 1))), _i32(lens), 1)
    before = w.weight.clone()
    out = paged.paged_attention(*args, weights=w)
    assert torch.equal(out, paged.paged_attention(*args))
    slot = torch.arange(64, device="cuda")
    held = (slot < args[4][:, None]).view(B, 4, 1, page)
    old = (slot < args[4][:, None] - 1).view(B, 4, 1, page)
    now, was = w.weight.view(B, 4, G, page).double(), before.view(B, 4, G, page).double()
    gained = torch.where(held, now - torch.where(old, was, torch.zeros_like(was)), torch.zeros_like(now)).sum((1, 3))
    assert torch.allclose(gained, torch.full_like(gained, R), rtol=1e-3, atol=1e-3)  # (differences of rounded sums)
    assert torch.equal(now[~held.expand_as(now)], was[~held.expand_as(was)])


@pytest.mark.parametrize("n,R,L", [(600, 64, 700), (1100, 8, 2500)])
def test_weights_of_very_many_rows(n, R, L):
    """Chunks of thousands of rows."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(26)
    G, D, page = 1, 64, 64
    mp = -(-L // page)
    cache, table = _filled(I8, mp, G, page, D, g, spread=False), _table(1, mp, mp, g)
    q = torch.randn(n, R, D, generator=g).to(F16).cuda()
    w = paged.new_paged_weights(cache)
    paged.paged_attention(q, cache, table.cuda(), _i32([0, n]), _i32([L]), n, weights=w)
    at = table[0].long().cuda()
    k = (cache.k[at, 0].double() * cache.k_scale[at, 0, None, None].double()).reshape(-1, D)[:L]
    want = torch.zeros(L, dtype=torch.float64, device="cuda")
    late = torch.arange(L, device="cuda")[None] > torch.arange(n, device="cuda")[:, None] + L - n
    for h in range(R):
        want += torch.softmax((q[:, h].double() @ k.T * D ** -0.5).masked_fill(late, float("-inf")), -1).sum(0)
    got = w.weight[at, 0].view(-1)[:L].double()
    assert ((got - want).abs() <= want * 4 * 2.0 ** -16 + 1e-30).all()


@pytest.mark.parametrize("n,R", [(6, 1), (40, 4)])
def test_trees_of_odd_batches(n, R):
    """Fewer tokens held than rows, more rows than max_tokens, a table that is too short."""
    from spatten_b200 import paged
    g, rng = torch.Generator().manual_seed(27), random.Random(27)
    G, D, page = 2, 64, 16
    news, lens = [n, n + 3, n, 0], [n - 3, n + 20, n + 50, 7]
    cu = _cum(news)
    cache, table = _filled(I8, 30, G, page, D, g), _table(4, 5, 30, g)
    sees = {t: frozenset(j for j in range(64) if rng.random() < 0.5) for t in range(cu[-1])}
    tree = OT.words(sees, cu[-1], 2).cuda()
    q = torch.randn(cu[-1], G * R, D, generator=g).to(F16).cuda()
    w = _weights(cache, g)
    before = paged.PagedWeights(*(t.clone() for t in w))
    out = paged.paged_attention(q, cache, table.cuda(), _i32(cu), _i32(lens), n, tree=tree, weights=w)
    _check(out, q, cache, table, cu, lens, D ** -0.5, sees, before, w, max_tokens=n)


def test_expanded_words_and_lists():
    """One mask, one list of accepted tokens for all; limits beyond any length."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(20)
    G, D, page, n = 1, 64, 16, 4
    cu, lens = _cum([n] * 3), [n + 9, n + 30, n]
    cache, table = _filled(I8, 12, G, page, D, g), _table(3, 4, 12, g)
    q = torch.randn(cu[-1], 2, D, generator=g).to(F16).cuda()
    mask = _i32([[5]])  # tokens 0 and 2
    out = paged.paged_attention(q, cache, table.cuda(), _i32(cu), _i32(lens), n, tree=mask.expand(cu[-1], 1))
    _check(out, q, cache, table, cu, lens, D ** -0.5, {t: frozenset((0, 2)) for t in range(cu[-1])})
    before = _cpu(cache)
    got = paged.paged_keep(cache, table.cuda(), _i32(cu), _i32(lens), _i32([[0, 2, -1]]).expand(3, 3))
    moves, new = OT.keep(before, table, cu, lens, [[0, 2, -1]] * 3)
    assert got.tolist() == new
    _check_moved(cache, before, table, moves, new)
    w = _weights(cache, g)
    was = [t.clone() for t in (*cache, *w)]
    assert paged.paged_evict(cache, w, table.cuda(), got, 2 ** 40, recent=2 ** 40).tolist() == new
    assert all(torch.equal(a, b) for a, b in zip(was, (*cache, *w)))
    moves = _evicted(cache, w, table, new, 5, recent=2 ** 31 - 1)
    assert moves[1][0]
    tree, pos = paged.paged_tree(_i32([-1] * 5), _i32([0, 5]), _i32([5]), 1 << 28)
    assert tree.tolist() == [[1], [2], [4], [8], [16]] and pos.tolist() == [0] * 5


def test_weights_long_and_offsets_past_32_bits():
    """A pool whose codes and weights lie beyond 2^32 bytes, pages at its end."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(19)
    G, D, page, R, L = 8, 128, 128, 1, 70000
    P = (1 << 30) // (G * page) + 600  # weights past 2^32 bytes, codes past 2^37
    P = min(P, 40000)                  # (what a GPU beside other tests has room for: codes past 2^32)
    cache = paged.new_paged_cache(P, G, D, page_size=page)
    mp = -(-L // page)
    table = torch.arange(P - mp, P, dtype=torch.int32)[torch.randperm(mp, generator=g)][None]
    small = _filled(I8, mp, G, page, D, g, spread=False)
    at = table[0].long().cuda()
    for big, part in zip(cache, small):
        big[at] = part
    w = paged.new_paged_weights(cache)
    q = torch.randn(1, G * R, D, generator=g).to(BF16).cuda()
    out = paged.paged_attention(q, cache, table.cuda(), _i32([0, 1]), _i32([L]), 1, weights=w)
    k, v = [(small[t].float() * small[2 + t][..., None, None]).transpose(0, 1).reshape(G, -1, D)[:, :L].double()
            for t in range(2)]
    p = torch.softmax(torch.einsum("gd,gnd->gn", q[0].double(), k) * D ** -0.5, -1)
    assert torch.allclose(out[0].double(), torch.einsum("gn,gnd->gd", p, v), rtol=2.0 ** -8, atol=1e-3)
    got = w.weight[at].transpose(0, 1).reshape(G, -1).double()
    assert torch.allclose(got[:, :L], p, rtol=1e-4, atol=1e-12) and (got[:, L:] == 0).all()
    kept = paged.paged_evict(cache, w, table.cuda(), _i32([L]), 1000)
    assert kept.tolist() == [1000]
    want = torch.topk(got.sum(0), 1000).values.sort().values
    now = w.weight[at].transpose(0, 1).reshape(G, -1).double()[:, :1000].sum(0).sort().values
    assert torch.allclose(now, want, rtol=1e-6)


# ------------------------------------------------------------------ eviction

def _check_moved(cache, before, table, moves, new_lens):
    kv = cache.k.dtype
    codes, scales, ys = OT.move(before, table, moves, new_lens)
    tol = 6.2e-5 if kv == I8 else 0.0
    for got, c, y in zip(_cpu(cache)[:2], codes, ys):
        got = O.code_values(got)
        assert ((got - y).abs() <= (c - y).abs() + tol).all()
    for got, s in zip(_cpu(cache)[2:], scales):
        assert torch.allclose(got.double(), s, rtol=4 * U, atol=0)


def _evicted(cache, w, table, lens, keep, **kw):
    """The call, checked against the oracle."""
    from spatten_b200 import paged
    before, wb, pb = _cpu(cache), w.weight.cpu(), w.position.cpu()
    got = paged.paged_evict(cache, w, table.cuda(), _i32(lens), keep, **kw)
    moves, new = OT.evict(before, wb, pb, table, lens, keep, **kw)
    assert got.tolist() == new
    _check_moved(cache, before, table, moves, new)
    assert torch.equal(w.weight.cpu().nan_to_num(-1), OT.move_beside(wb, table, moves).nan_to_num(-1))
    assert torch.equal(w.position.cpu(), OT.move_beside(pb, table, moves))
    return moves


@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("kv,D,page,G,lens,keep,recent", [
    (I8, 128, 64, 2, [300, 299, 64, 65, 0, 500], 256, 0),
    (E4, 64, 16, 3, [40, 17, 16, 33], 16, 5),
    (I8, 64, 128, 1, [1000, 129], 1, 0),
    (E4, 128, 32, 8, [700, 100], 99, 99),
    (I8, 64, 16, 2, [130, 200], 77, 1000),   # more recent ones than places
    (I8, 128, 128, 1, [900], 899, 3),
    (E4, 64, 64, 4, [50, 10], 100, 0),        # nothing to do
])
def test_evict(kv, D, page, G, lens, keep, recent, per_head):
    g = torch.Generator().manual_seed(keep)
    mp = max(lens) // page + 2
    P = len(lens) * mp + 2
    cache, table = _filled(kv, P, G, page, D, g), _table(len(lens), mp, P, g)
    _evicted(cache, _weights(cache, g), table, lens, keep, recent=recent, per_head=per_head)


@pytest.mark.parametrize("slots,lens,keep", [
    (4096, [4096, 4000], 2048), (6000, [6000, 5000], 4500), (10000, [9999, 10000], 700), (20000, [20000, 129], 11111),
    (140000, [131001], 65536),
])
@pytest.mark.parametrize("recent", [0, 300])
def test_evict_long(slots, lens, keep, recent):
    """Rows over every number of CTAs."""
    g = torch.Generator().manual_seed(keep)
    page, G, D = 64, 2, 64
    mp = -(-slots // page)
    P = len(lens) * mp
    cache, table = _filled(E4, P, G, page, D, g), _table(len(lens), mp, P, g)
    _evicted(cache, _weights(cache, g), table, lens, keep, recent=recent)


def test_evict_more_slots_than_shared_memory():
    """A table so wide that a CTA's keys do not fit its shared memory."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(2)
    page, G, D, L, keep = 128, 1, 64, 500_000, 123_456
    mp = 8192
    cache = paged.new_paged_cache(-(-L // page), G, D, page_size=page)
    table = torch.full((1, mp), -1, dtype=torch.int32)
    table[0, :-(-L // page)] = torch.randperm(-(-L // page), generator=g)
    w = paged.new_paged_weights(cache)
    w.weight.copy_(torch.exp(torch.randn(w.weight.shape, generator=g)))
    w.position.copy_(torch.randint(0, 10 ** 6, w.position.shape, generator=g))
    at = table[0, :-(-L // page)].long()
    wb = w.weight.cpu()[at, 0].view(-1)[:L]
    pb = w.position.cpu()[at, 0].view(-1)[:L]
    new = paged.paged_evict(cache, w, table.cuda(), _i32([L]), keep, recent=1000)
    assert new.tolist() == [keep]
    moves = OT.select(wb.tolist(), pb.tolist(), keep, 1000)
    want = wb.clone()
    to, fr = torch.tensor(moves).T
    want[to] = wb[fr]
    assert torch.equal(w.weight.cpu()[at, 0].view(-1)[:L], want)


def _weights_of(kind, shape, g):
    if kind == "equal":
        return torch.full(shape, 0.25)
    if kind == "zeros":
        return torch.zeros(shape)
    if kind == "few":  # many ties at the border
        return torch.randint(0, 3, shape, generator=g).float()
    if kind == "near":  # neighbours in fp32
        return 1 + torch.randint(0, 50, shape, generator=g) * 2.0 ** -23
    if kind == "tiny":  # subnormal and 0
        return torch.randint(0, 5, shape, generator=g) * 2.0 ** -149
    x = torch.exp(8 * torch.randn(shape, generator=g))
    x.view(-1)[::7] = float("nan")
    x.view(-1)[1::7] = float("inf")
    x.view(-1)[2::7] = -1.0
    x.view(-1)[3::7] = -0.0
    return x


@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("kind", ["equal", "zeros", "few", "near", "tiny", "odd"])
def test_evict_ties_and_odd_weights(kind, per_head):
    """Ties go to the lower slot; NaN and negative weights count as 0, infinities as
    the largest."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(23)
    page, G, D = 32, 1 if kind == "odd" and not per_head else 2, 64
    lens = [700, 333, 5000]
    mp = 5000 // page + 1
    P = 3 * mp
    cache, table = _filled(I8, P, G, page, D, g), _table(3, mp, P, g)
    w = paged.new_paged_weights(cache)
    w.weight.copy_(_weights_of(kind, w.weight.shape, g))
    w.position.copy_(torch.randint(-5, 2 ** 31 - 1, w.position.shape, generator=g) if kind == "odd"
                     else torch.randint(0, 100, w.position.shape, generator=g))
    for keep, recent in ((300, 0), (200, 7)):
        lens = [n if i == 2 else min(n, 600) for i, n in enumerate(lens)]
        _evicted(cache, w, table, lens, keep, recent=recent, per_head=per_head)


def test_evict_leaves_the_rest_alone():
    """Slots without memory, tables that are too short, negative lengths: such a
    sequence is left as it is, and its new length is its old one."""
    g = torch.Generator().manual_seed(29)
    page, G, D = 16, 2, 64
    lens = [80, 80, 90, -3, 80, 33]
    table = _table(6, 5, 40, g)
    table[0, 2], table[1, 4] = -1, 40
    cache = _filled(I8, 40, G, page, D, g)
    moves = _evicted(cache, _weights(cache, g), table, lens, 32)
    assert not any(m[0] for m in moves[:4]) and moves[4][0]


def test_evict_again_and_again():
    """A cache that is cut to half and filled up again, its scales spread over
    many octaves: appended, weighed, evicted, as a loop does it, against a cache that
    keeps every token apart."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(31)
    G, D, page, R, cap, keep = 2, 64, 16, 2, 96, 48
    cache = paged.new_paged_cache(2 * cap // page, G, D, page_size=page)
    w = paged.new_paged_weights(cache)
    table = torch.randperm(2 * cap // page, generator=g).view(2, -1).to(torch.int32)
    lens, seen = [0, 0], 0
    for step in range(14):
        n = 16 if step % 3 else 7
        if lens[0] + n > cap:
            _evicted(cache, w, table, lens, keep, recent=8, per_head=step % 2 == 0)
            lens = [keep, keep]
        cu = _cum([n, n])
        lens = [x + n for x in lens]
        x = (torch.randn(2 * n, G * R + 2 * G, D, generator=g) * 2.0 ** (step % 5 - 2)).to(BF16).cuda()
        pos = _i32([seen + i for _ in range(2) for i in range(n)])
        seen += n
        paged.paged_append(cache, x[:, :G], x[:, G:2 * G], table.cuda(), _i32(cu), _i32(lens), n)
        before = paged.PagedWeights(*(t.clone() for t in w))
        out = paged.paged_attention(x[:, 2 * G:], cache, table.cuda(), _i32(cu), _i32(lens), n, weights=w,
                                    positions=pos)
        _check(out, x[:, 2 * G:], cache, table, cu, lens, D ** -0.5, None, before, w, pos.tolist())


# ------------------------------------------------------------------ accepted tokens

@pytest.mark.parametrize("kv,D,page,G", [(I8, 128, 64, 2), (E4, 64, 16, 3), (I8, 64, 128, 1), (E4, 128, 32, 2)])
@pytest.mark.parametrize("weights", [False, True])
def test_keep(kv, D, page, G, weights):
    from spatten_b200 import paged
    g, rng = torch.Generator().manual_seed(37), random.Random(37)
    news = [26, 64, 1, 0, 100, 33, 9, 40, 5]
    olds = [1000, 0, 15, 7, 63, 64, 129, 3, 31]
    paths = [[0, 3, 17, 25], sorted(rng.sample(range(64), 30)), [0], [], list(range(100)), [], [8],
             [0, 1, 2, 39], [0, 2, 2, 4]]  # (a place twice ends the list)
    lens, cu = [a + n for a, n in zip(olds, news)], _cum(news)
    acc = torch.full((9, 101), -1, dtype=torch.int32)
    for b, p in enumerate(paths):
        acc[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
    acc[5, 0], acc[5, 1] = 33, 40   # no new tokens
    acc[2, 1] = 2 ** 31 - 1
    mp = max(lens) // page + 1
    P = 9 * mp + 1
    cache, table = _filled(kv, P, G, page, D, g), _table(9, mp, P, g)
    w = _weights(cache, g) if weights else None
    before = _cpu(cache)
    wb, pb = (w.weight.cpu(), w.position.cpu()) if weights else (None, None)
    got = paged.paged_keep(cache, table.cuda(), _i32(cu), _i32(lens), acc.cuda(), weights=w)
    moves, new = OT.keep(before, table, cu, lens, acc.tolist())
    assert got.tolist() == new
    _check_moved(cache, before, table, moves, new)
    if weights:
        assert torch.equal(w.weight.cpu(), OT.move_beside(wb, table, moves))
        assert torch.equal(w.position.cpu(), OT.move_beside(pb, table, moves))


def test_keep_odd_lists():
    """Fewer tokens held than rows, pages without memory, descending bounds, no columns,
    strided lists."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(41)
    G, D, page = 2, 64, 16
    news, lens = [20, 20, 20, 20], [10, 60, 60, 25]
    cu = _cum(news)
    table = _table(4, 4, 20, g)
    table[1, 3] = -1   # its tokens 8 .. 19
    table[2, 2] = 77   # its tokens 0 .. 7
    wide = torch.full((4, 20), -1, dtype=torch.int32, device="cuda")
    acc = wide[:, 3:9]
    acc.copy_(_i32([[11, 12, 15, 19, -1, -1], [0, 3, 6, 9, 12, 15], [9, 12, 15, -1, -1, -1], [1, 3, 5, 7, 9, 11]]))
    cache = _filled(E4, 20, G, page, D, g)
    before = _cpu(cache)
    got = paged.paged_keep(cache, table.cuda(), _i32(cu), _i32(lens), acc)
    moves, new = OT.keep(before, table, cu, lens, acc.tolist())
    assert got.tolist() == new
    _check_moved(cache, before, table, moves, new)
    before = _cpu(cache)
    assert paged.paged_keep(cache, table.cuda(), _i32(cu), _i32(lens), acc[:, :0]).tolist() == [0, 40, 40, 5]
    assert paged.paged_keep(cache, table[:1].cuda(), _i32([5, 2]), _i32([10]), acc[:1]).tolist() == [10]
    for a, b in zip(before, _cpu(cache)):
        assert torch.equal(a.view(I8) if a.dtype == E4 else a, b.view(I8) if b.dtype == E4 else b)


# ------------------------------------------------------------------ together

def _loop_step(paged, st, n, keep=40):
    """One step of a loop that drafts trees into a cache of bounded length."""
    tree, pos = paged.paged_tree(st["parents"], st["cu"], st["lens"], n)
    paged.paged_append(st["cache"], st["x"][:, :2], st["x"][:, 2:4], st["table"], st["cu"], st["lens"], n)
    out = paged.paged_attention(st["x"][:, 4:], st["cache"], st["table"], st["cu"], st["lens"], n, tree=tree,
                                weights=st["w"], positions=pos)
    lens = paged.paged_keep(st["cache"], st["table"], st["cu"], st["lens"], st["accepted"], weights=st["w"])
    lens = paged.paged_evict(st["cache"], st["w"], st["table"], lens, keep, recent=4)
    return out, lens


def _loop_state(seed):
    from spatten_b200 import paged
    g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    news, old = [9, 6, 9], [30, 41, 0]
    cu = _cum(news)
    cache = _filled(I8, 24, 2, 16, 64, g)
    return dict(cache=cache, w=_weights(cache, g), table=_table(3, 5, 24, g).cuda(), cu=_i32(cu),
                lens=_i32([a + n for a, n in zip(old, news)]), parents=_i32([p for n in news for p in _random_tree(n, rng)]),
                accepted=_i32([[0, 3, 4, 8], [0, 5, -1, -1], [0, 1, 2, -1]]),
                x=torch.randn(cu[-1], 12, 64, generator=g).to(BF16).cuda())


def _pools(st):
    return [t.view(I8) if t.dtype == E4 else t for t in (*st["cache"], *st["w"])]


def test_loop_captured_with_other_contents():
    """A captured step replayed over other trees, lists, lengths and contents gives
    what the plain calls give."""
    from spatten_b200 import paged
    st = _loop_state(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _loop_step(paged, st, 9)
    torch.cuda.current_stream().wait_stream(side)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out, lens = _loop_step(paged, st, 9)
    for seed in (2, 3):
        other = _loop_state(seed)
        for a, b in zip(_pools(st) + [st[k] for k in ("lens", "parents", "accepted", "x", "table")],
                        _pools(other) + [other[k] for k in ("lens", "parents", "accepted", "x", "table")]):
            a.copy_(b)
        gr.replay()
        torch.cuda.synchronize()
        want, want_lens = _loop_step(paged, other, 9)
        assert torch.equal(out, want) and torch.equal(lens, want_lens)
        for a, b in zip(_pools(st), _pools(other)):
            assert torch.equal(a, b)


def test_two_streams_at_once():
    """Two loops on streams of their own, repeatable to the bit."""
    from spatten_b200 import paged
    want = []
    for seed in (4, 5):
        st = _loop_state(seed)
        out, lens = _loop_step(paged, st, 9)
        want.append([out, lens] + _pools(st))
    torch.cuda.synchronize()
    for _ in range(5):
        states, streams = [_loop_state(seed) for seed in (4, 5)], [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = []
        for st, s in zip(states, streams):
            with torch.cuda.stream(s):
                got.append([*_loop_step(paged, st, 9)] + _pools(st))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for x, y in zip(a, b):
                assert torch.equal(x, y)


def test_refusals():
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(43)
    cache = _filled(I8, 8, 2, 16, 64, g)
    w, table = _weights(cache, g), _table(2, 4, 8, g).cuda()
    cu, lens = _i32([0, 3, 6]), _i32([20, 30])
    q = torch.zeros(6, 4, 64, dtype=F16, device="cuda")
    tree = torch.zeros(6, 1, dtype=torch.int32, device="cuda")
    call = lambda **kw: paged.paged_attention(q, cache, table, cu, lens, 3, **kw)  # noqa: E731
    with pytest.raises(ValueError, match="tree"):
        call(tree=tree[:5])
    with pytest.raises(ValueError, match="tree"):
        call(tree=tree.long())
    with pytest.raises(ValueError, match="0 words"):
        call(tree=tree[:, :0])
    with pytest.raises(ValueError, match="tree"):
        call(tree=tree.cpu())
    with pytest.raises(ValueError, match="positions without"):
        call(positions=_i32(range(6)))
    with pytest.raises(ValueError, match="positions"):
        call(weights=w, positions=_i32(range(5)))
    with pytest.raises(ValueError, match="weights.weight"):
        call(weights=paged.PagedWeights(w.weight[:7], w.position[:7]))
    with pytest.raises(ValueError, match="weights.position"):
        call(weights=paged.PagedWeights(w.weight, w.position.long()))
    with pytest.raises(ValueError, match="parents"):
        paged.paged_tree(_i32(range(6)).long(), cu, lens, 3)
    with pytest.raises(ValueError, match="no CPU path"):
        paged.paged_tree(_i32(range(6)).cpu(), cu, lens, 3)
    with pytest.raises(RuntimeError, match="at most 1024"):
        paged.paged_tree(_i32([0] * 2000), _i32([0, 2000]), _i32([2000]), 2000)
    for bad in (dict(keep=0), dict(keep=5, recent=-1)):
        with pytest.raises(RuntimeError, match="need >= 0"):
            paged.paged_evict(cache, w, table, lens, **bad)
    with pytest.raises(RuntimeError, match="page table of"):
        paged.paged_evict(cache, w, torch.zeros(2, 1 << 17, dtype=torch.int32, device="cuda"), lens, 5)
    with pytest.raises(RuntimeError, match="stride"):
        paged.paged_evict(cache, w, table[:1].expand(2, -1), lens, 5)
    with pytest.raises(ValueError, match="accepted"):
        paged.paged_keep(cache, table, cu, lens, _i32([[0, 1]]))
    with pytest.raises(ValueError, match="cu_tokens"):
        paged.paged_keep(cache, table, cu[:2], lens, _i32([[0], [1]]))


def test_no_sequences():
    from spatten_b200 import paged
    cache = paged.new_paged_cache(4, 2, 64, page_size=16)
    w = paged.new_paged_weights(cache)
    t, none = torch.zeros(0, 3, dtype=torch.int32, device="cuda"), _i32([])
    tree, pos = paged.paged_tree(none, _i32([0]), none, 0)
    assert tree.shape[0] == 0 and pos.shape == (0,)
    q = torch.zeros(0, 2, 64, dtype=F16, device="cuda")
    assert paged.paged_attention(q, cache, t, _i32([0]), none, 0, tree=tree, weights=w).shape == q.shape
    assert paged.paged_evict(cache, w, t, none, 5).shape == (0,)
    assert paged.paged_keep(cache, t, _i32([0]), none, torch.zeros(0, 4, dtype=torch.int32, device="cuda")).shape == (0,)
