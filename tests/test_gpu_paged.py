"""GPU parity of the paged 8-bit KV cache (spatten_b200.paged) against the
float64 oracle (oracle/paged.py).

Tolerances (u = 2^-24):
* append: a code's value y = x / S carries the roundings of the norm (a
  reciprocal root of 2 ulp and two products), of the rotation (two products
  and a sum, of halves of which |x1| + |x2| <= 2 sqrt(2) max|x'|) and of the
  scale: under 14 roundings of values up to 2 sqrt(2) * 127 (int8) or 448
  (e4m3), 14 u 2.83 * 127 < 3.1e-4 and < 1.1e-3. The code must be as near to y
  as the nearest one, up to twice that.
* attention, per output: half a step of the result, and of A = sum p |v|:
  the rounding of p to fp16 (2^-11) and of the scores, D u S each way with S =
  sum |q k| of the scores, into an exponent (times 2 for numerator and
  denominator), and 2^-16 for the fp32 sums over the keys. And of the row's
  largest A: a weight p v_scale is an fp16 relative to the row's largest, and
  one below fp16's normal range is off by up to half its smallest step, 2^-25 of
  that, times a code of at most 127; the largest weight meets a code of 64 or
  more in one of its key's dims (normal values, D >= 64), so n keys make at
  most n 2^-25 (127 / 64) < n 2^-24 of the row's largest A. It counts where an
  output's own terms are that much smaller than its row's: a dim in which the key
  with all the weight holds a 0.
"""
import itertools

import pytest
import torch

from oracle import paged as O

pytestmark = pytest.mark.gpu

I8, E4 = torch.int8, torch.float8_e4m3fn
F16, BF16 = torch.float16, torch.bfloat16
U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cum(news):
    return [0] + list(itertools.accumulate(news))


def _table(B, mp, P, g):
    """Every sequence's own pages, in a shuffled order."""
    return torch.randperm(P, generator=g)[:B * mp].view(B, mp).to(torch.int32)


def _tables(rows, D, dt=torch.float32):
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    return ang.cos().to(dt).cuda(), ang.sin().to(dt).cuda()


def _cpu(cache):
    return [t.view(I8).cpu().view(t.dtype) if t.dtype == E4 else t.cpu() for t in cache]


def _check_append(cache, before, want, q=None):
    qo, codes, scales, ys = want
    kv = cache.k.dtype
    tol = 6.2e-4 if kv == I8 else 2.2e-3
    for got, c, y in zip(_cpu(cache)[:2], codes, ys):
        got = O.code_values(got)
        assert torch.isfinite(got).all()
        assert ((got - y).abs() <= (c - y).abs() + tol).all()
    for got, s in zip(_cpu(cache)[2:], scales):
        assert torch.allclose(got.double(), s, rtol=3e-6, atol=0)  # 14 roundings of the maximum, and the division
    if q is not None:
        q = q.cpu()
        step = torch.finfo(q.dtype).eps / 2
        # a rotation's terms may cancel: its roundings are relative to them
        assert ((q.double() - qo).abs() <= step * qo.abs() + 14 * U * 2.83 * qo.abs().amax(-1, keepdim=True)
                + torch.finfo(q.dtype).smallest_normal).all()


@pytest.mark.parametrize("kv,dt,D,page,G,H,norm,rope,calls", [
    (I8, BF16, 128, 64, 2, 8, True, True, [[70, 0, 1, 63], [1, 1, 1, 1], [3, 0, 130, 1]]),
    (E4, F16, 64, 16, 3, 3, False, True, [[1, 15, 16, 17], [1, 1, 1, 1], [2, 33, 0, 5]]),
    (E4, BF16, 128, 128, 1, 5, True, True, [[129, 3], [1, 1], [1, 300]]),
    (I8, F16, 64, 32, 2, 4, True, False, [[31, 32, 33], [2, 2, 2]]),
    (I8, F16, 128, 16, 2, 0, False, False, [[40, 1], [1, 7]]),
    (E4, F16, 64, 64, 1, 16, False, True, [[5], [200], [1]]),
    (I8, BF16, 64, 128, 2, 2, False, True, [[100, 128], [40, 1]]),
])
def test_append(kv, dt, D, page, G, H, norm, rope, calls):
    """Several calls in a row: blocks that grow, and whose scale grows."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(3)
    B = len(calls[0])
    mp = max(sum(c[b] for c in calls) for b in range(B)) // page + 2
    P = B * mp + 3
    table = _table(B, mp, P, g)
    cache = paged.new_paged_cache(P, G, D, page_size=page, kv_dtype=kv)
    cache.k_scale.fill_(7.0)  # whatever an earlier user of the page left there
    cos, sin = _tables(mp * page, D) if rope else (None, None)
    wq, wk = ((1 + 0.3 * torch.randn(2, D, generator=g)).to(dt) if norm else (None, None))
    lens = [0] * B
    for step, new in enumerate(calls):
        cu = _cum(new)
        lens = [a + n for a, n in zip(lens, new)]
        x = (torch.randn(cu[-1], H + 2 * G + 1, D, generator=g) * 3.0 ** step).to(dt)
        xd = x.cuda()  # a fused projection's output: strided rows, and a head that is not the cache's
        q, k, v = xd[:, :H], xd[:, H:H + G], xd[:, H + G + 1:]
        before = _cpu(cache)
        got = paged.paged_append(cache, k, v, table.cuda(), _i32(cu), _i32(lens), max(new), q=q if H else None,
                                 cos=cos, sin=sin, q_norm_w=wq.cuda() if norm and H else None,
                                 k_norm_w=wk.cuda() if norm else None, eps=1e-5)
        want = O.append(before, x[:, H:H + G], x[:, H + G + 1:], table, cu, lens, q=x[:, :H] if H else None,
                        cos=None if cos is None else cos.cpu(), sin=None if sin is None else sin.cpu(), wq=wq, wk=wk,
                        eps=1e-5)
        _check_append(cache, before, want, got)


def test_append_head_major_in_place_positions_and_own_type_tables():
    """Head-major K, queries rotated in place, positions of a pruned prompt
    (some behind the tables), cos / sin in the rows' type and D wide."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(4)
    G, H, D, page, T = 2, 4, 64, 16, 50
    table = _table(1, 4, 6, g)
    cache = paged.new_paged_cache(6, G, D, page_size=page)
    k, v = torch.randn(2, G, T, D, generator=g).to(BF16)
    q = torch.randn(T, H, D, generator=g).to(BF16)
    pos = torch.randperm(90, generator=g)[:T].sort().values.to(torch.int32) - 3
    cos, sin = (torch.cat([t, t], 1) for t in _tables(60, D, BF16))
    before = _cpu(cache)
    qd = q.cuda()
    got = paged.paged_append(cache, k.cuda().transpose(0, 1), v.cuda().transpose(0, 1), table.cuda(), _i32([0, T]),
                             _i32([T]), T, q=qd, cos=cos, sin=sin, positions=pos.cuda(), q_out=qd)
    assert got is qd
    want = O.append(before, k.transpose(0, 1), v.transpose(0, 1), table, [0, T], [T], q=q, cos=cos.cpu(),
                    sin=sin.cpu(), positions=pos.tolist())
    _check_append(cache, before, want, got)


@pytest.mark.parametrize("kv", [I8, E4])
def test_append_odd_values(kv):
    """Infinities saturate and NaN becomes 0 without touching the block's
    scale; blocks of zeros; values at both ends of bf16's range."""
    from spatten_b200 import paged
    G, D, page = 1, 64, 16
    inf, nan = float("inf"), float("nan")
    x = torch.zeros(5 * page, G, D, dtype=BF16)
    x[3, 0, 1:6] = torch.tensor([1.0, -2.0, inf, -inf, nan])   # block 0
    x[page:2 * page] = 0                                          # block 1: zeros
    x[2 * page + 1, 0, :3] = torch.tensor([3e38, -1e38, 1e-38])   # block 2
    x[3 * page + 5, 0, :3] = torch.tensor([1e-39, -9e-40, 5e-40])  # block 3: subnormals
    x[4 * page + 2, 0, :2] = torch.tensor([inf, nan])             # block 4: nothing finite but 0
    T = x.shape[0]
    table = torch.arange(5, dtype=torch.int32)[None]
    cache = paged.new_paged_cache(5, G, D, page_size=page, kv_dtype=kv)
    before = _cpu(cache)
    paged.paged_append(cache, x.cuda(), x.cuda(), table.cuda(), _i32([0, T]), _i32([T]), T)
    codes = O.code_values(_cpu(cache)[0])[:, 0]
    top = 127 if kv == I8 else 448
    s = cache.k_scale[:, 0].double().cpu()
    want = O.append(before, x, x, table, [0, T], [T])
    # a subnormal scale holds its quotient to one part in a few hundred thousand
    assert torch.allclose(s, want[2][0][:, 0], rtol=1e-4, atol=0)
    assert torch.equal(codes[0, 3, 3:6], torch.tensor([top, -top, 0.0], dtype=torch.float64))
    assert (codes[1] == 0).all() and s[1] == 0 and s[4] == 0 and (codes[4] == 0).all()
    assert torch.isfinite(codes).all()
    assert torch.equal(codes[[0, 2]], want[1][0][[0, 2], 0])
    # half a code step: of e4m3 between 1/16 and 1/8, times the smallest scale
    assert ((codes[3] * s[3]).abs().max() - x[3 * page + 5, 0, 0].double()).abs() <= \
        (1e-4 * 1e-39 if kv == I8 else 2.0 ** -8 * 2.0 ** -126)
    k, _ = paged.paged_read(cache, table.cuda(), _i32([T]))
    assert torch.isfinite(k).all()


def test_append_leaves_the_rest_alone():
    """Sequences without tokens, pages without memory, a table that is too
    short, more tokens than slots, rows behind the last sequence and behind
    max_tokens: nothing else changes."""
    from spatten_b200 import paged
    G, H, D, page = 1, 2, 64, 16
    g = torch.Generator().manual_seed(5)
    # b0: 20 tokens, its second page has no memory; b1: none; b2: 4 tokens but only 2 slots held;
    # b3: runs past the table; b4: more tokens than max_tokens
    new, lens, cap = [20, 0, 4, 10, 30], [20, 5, 2, 40, 30], 25
    table = torch.tensor([[3, -1], [0, 1], [2, 99], [4, 5], [6, 7]], dtype=torch.int32)
    cu = _cum(new)
    T = cu[-1]
    x = torch.randn(T + 6, 2 * G + H, D, generator=g).to(F16)
    cache = paged.new_paged_cache(9, G, D, page_size=page)
    for t in cache[:2]:
        t.fill_(11)
    for t in cache[2:]:
        t.fill_(0.5)
    before = _cpu(cache)
    q_out = torch.full((T + 6, H, D), 9.0, dtype=F16, device="cuda")
    xd = x.cuda()
    paged.paged_append(cache, xd[:, :1], xd[:, 1:2], table.cuda(), _i32(cu), _i32(lens), cap, q=xd[:, 2:],
                       q_out=q_out)
    # the oracle's calls: the sequences as if only the rows that are processed were there
    want = [t.clone() for t in before]
    codes, scales, ys = [O.code_values(want[0]), O.code_values(want[1])], [want[2].double(), want[3].double()], None
    ys = [c.clone() for c in codes]
    for b in range(5):
        n = min(new[b], cap)
        end = lens[b] - new[b] + n
        part = x[cu[b]:cu[b] + n]
        r = O.append(before, part[:, :1], part[:, 1:2], table[b:b + 1], [0, n], [end])
        for pid in [int(p) for p in table[b] if 0 <= p < 9]:
            for w in range(2):
                codes[w][pid], ys[w][pid], scales[w][pid] = r[1][w][pid], r[3][w][pid], r[2][w][pid]
    _check_append(cache, before, (None, codes, scales, ys))
    q = q_out.cpu()
    live = torch.zeros(T + 6, dtype=torch.bool)
    for b in range(5):
        live[cu[b]:cu[b] + min(new[b], cap)] = True
    assert torch.equal(q[live], x[:, 2:][live])  # neither norm nor rotation: a copy
    assert (q[~live] == 9).all()


def _filled(kv, P, G, page, D, g, spread=True):
    """A pool of random blocks, scales over several octaves."""
    from spatten_b200 import paged
    cache = paged.new_paged_cache(P, G, D, page_size=page, kv_dtype=kv)
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = torch.randn(P, G, page, D, generator=g)
        amax = x.abs().amax((2, 3), keepdim=True)
        c = (x / amax * 127).round().to(I8) if kv == I8 else (x / amax * 448).to(E4)
        codes.view(I8).copy_(c.view(I8))
        scale.copy_((amax / (127 if kv == I8 else 448))[..., 0, 0] *
                    2.0 ** (torch.randint(-3, 3, (P, G), generator=g) if spread else 0))
    return cache


def _check_attend(out, q, cache, table, cu, lens, sm):
    want, A, S = O.attend(q.cpu(), _cpu(cache), table, cu, lens, sm)
    D = q.shape[-1]
    T = cu[-1]
    tol = torch.finfo(out.dtype).eps / 2 * want.abs() + A * (2.0 ** -11 + 2 * D * U * S + 2.0 ** -16) + \
        max(lens) * U * A.amax(-1, keepdim=True) + torch.finfo(out.dtype).smallest_normal
    bad = ((out.cpu().double() - want).abs() > tol)[:T]
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())
    return want


@pytest.mark.parametrize("kv,dt,D,page,G,R,news,lens", [
    # one token: every group size, ragged lengths around tile and page borders
    (I8, BF16, 128, 64, 2, 4, [1] * 6, [1, 31, 32, 33, 64, 700]),
    (E4, F16, 128, 16, 1, 1, [1] * 5, [1, 15, 16, 17, 333]),
    (E4, BF16, 64, 32, 3, 3, [1, 1, 1], [2, 129, 65]),
    (I8, F16, 64, 128, 1, 8, [1, 1], [127, 130]),
    (I8, F16, 128, 64, 1, 16, [1, 1], [200, 90]),
    (E4, F16, 64, 16, 1, 40, [1, 1], [50, 31]),
    (I8, BF16, 64, 16, 2, 128, [1], [77]),
    # drafted tokens
    (I8, BF16, 128, 32, 2, 5, [2, 7, 1, 3], [2, 40, 9, 129]),
    (E4, F16, 64, 64, 2, 2, [4, 8], [100, 8]),
    # pieces of prompts
    (I8, F16, 128, 64, 1, 2, [130, 1, 64], [300, 64, 64]),
    (E4, BF16, 64, 16, 2, 1, [257, 33], [257, 100]),
    (E4, BF16, 128, 128, 1, 8, [70, 200], [300, 201]),
])
def test_attention(kv, dt, D, page, G, R, news, lens):
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(6)
    B, H = len(news), G * R
    mp = max(lens) // page + 2
    P = B * mp + 2
    table, cu = _table(B, mp, P, g), _cum(news)
    cache = _filled(kv, P, G, page, D, g)
    q = torch.randn(cu[-1], H, D, generator=g).to(dt).cuda()
    out = paged.paged_attention(q, cache, table.cuda(), _i32(cu), _i32(lens), max(news))
    _check_attend(out, q, cache, table, cu, lens, D ** -0.5)


@pytest.mark.parametrize("kv,R", [(I8, 4), (E4, 12)])
def test_attention_masked_places(kv, R):
    """Sequences without slots or with fewer slots than queries (empty rows:
    0), pages without memory, garbage behind the last slot (e4m3 NaN codes,
    NaN scales of unused pages), rows behind the last sequence."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(7)
    G, D, page = 2, 64, 32
    news, lens = [1, 3, 0, 2, 5], [0, 2, 40, 90, 70]
    cu, B = _cum(news), 5
    table = _table(B, 4, 22, g)
    table[3, 1], table[4, 0], table[4, 1] = -1, 1000, -7
    cache = _filled(kv, 22, G, page, D, g)
    used = torch.zeros(22, dtype=torch.bool)
    for b in range(B):
        for s in range(lens[b]):
            if 0 <= table[b, s // page] < 22:
                used[table[b, s // page]] = True
        last = int(table[b, lens[b] // page])
        if 0 <= last < 22:  # the rows behind the sequence's last slot
            for t in cache[:2]:
                t.view(I8)[last, :, lens[b] % page:] = 0x7F
    for t in cache[2:]:
        t[(~used).cuda()] = float("nan")
    T = cu[-1] + 3
    q = torch.randn(T, G * R, D, generator=g).to(BF16).cuda()
    q[cu[-1]:] = float("nan")
    out = torch.full((T, G * R, D), 5.0, dtype=BF16, device="cuda")
    got = paged.paged_attention(q, cache, table.cuda(), _i32(cu), _i32(lens), max(news), out=out)
    assert got is out
    want = _check_attend(out, q, cache, table, cu, lens, D ** -0.5)
    assert (out[cu[-1]:] == 5).all()
    empty = [0, 1]  # sequence 0 holds nothing; sequence 1's first query would be slot -1
    assert (want[empty] == 0).all() and (out[empty] == 0).all()
    # the rows behind max_tokens are left alone as well
    out.fill_(5.0)
    paged.paged_attention(q, cache, table.cuda(), _i32(cu), _i32(lens), 2, out=out)
    keep = torch.tensor([i - cu[b] >= 2 for b in range(B) for i in range(cu[b], cu[b + 1])] + [True] * 3)
    assert (out.cpu()[keep] == 5).all()
    part = out[:cu[-1]].clone()
    part[keep[:cu[-1]].cuda()] = want.to(BF16)[:cu[-1]][keep[:cu[-1]]].cuda()
    _check_attend(part, q[:cu[-1]], cache, table, cu, lens, D ** -0.5)


def test_attention_extremes():
    """Blocks of zeros, scales 2^-100 to 2^100 side by side in one sequence,
    scores of thousands, strided queries and outputs."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(8)
    G, R, D, page, n = 1, 4, 128, 16, 200
    table = _table(1, 13, 15, g)
    cache = _filled(I8, 15, G, page, D, g, spread=False)
    cache.v_scale[:, 0] = 2.0 ** torch.linspace(-100, 100, 15)[torch.randperm(15, generator=g)].round().cuda()
    cache.v_scale[int(table[0, 2])] = 0.0
    cache.k_scale[int(table[0, 4])] = 0.0
    q = torch.randn(1, 2 * R, D, generator=g).to(BF16).cuda()[:, ::2]
    out = torch.zeros(1, R, 2 * D, dtype=BF16, device="cuda")[:, :, :D]
    paged.paged_attention(q, cache, table.cuda(), _i32([0, 1]), _i32([n]), 1, out=out)
    _check_attend(out, q, cache, table, [0, 1], [n], D ** -0.5)
    # one block alone decides: a tiny V beside huge ones that no weight reaches
    q = (q.float() * 300).to(BF16)
    out = paged.paged_attention(q, cache, table.cuda(), _i32([0, 1]), _i32([n]), 1)
    _check_attend(out, q, cache, table, [0, 1], [n], D ** -0.5)


def test_attention_long_and_offsets_past_32_bits():
    """A pool of more than 2^31 codes, a sequence in its last pages, split
    over many CTAs."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(9)
    G, R, D, page, n = 8, 2, 128, 128, 5000
    mp = 40
    P = 2 ** 31 // (G * page * D) + mp + 1
    table = (P - 1 - torch.randperm(mp, generator=g)).to(torch.int32)[None]
    small = _filled(I8, mp, G, page, D, g)
    cache = paged.PagedKVCache(*(torch.empty((P,) + t.shape[1:], dtype=t.dtype, device="cuda") for t in small))
    for t, s in zip(cache, small):
        t[P - mp:] = s
    q = torch.randn(1, G * R, D, generator=g).to(F16).cuda()
    out = paged.paged_attention(q, cache, table.cuda(), _i32([0, 1]), _i32([n]), 1)
    _check_attend(out, q, small, table - (P - mp), [0, 1], [n], D ** -0.5)
    k, v = paged.paged_read(cache, table.cuda(), _i32([n]), dtype=F16)
    ks, vs = paged.paged_read(small, table.cuda() - (P - mp), _i32([n]), dtype=F16)
    assert torch.equal(k, ks) and torch.equal(v, vs)
    # a token appended behind them
    x = torch.randn(1, 2 * G, D, generator=g).to(F16).cuda()
    for c, t in ((cache, table), (small, table - (P - mp))):
        paged.paged_append(c, x[:, :G], x[:, G:], t.cuda(), _i32([0, 1]), _i32([n + 1]), 1)
    assert torch.equal(cache.k[P - mp:], small.k) and torch.equal(cache.v_scale[P - mp:], small.v_scale)


@pytest.mark.parametrize("kv,dt,D,page,G", [(I8, BF16, 128, 64, 3), (E4, F16, 64, 16, 1), (E4, BF16, 64, 128, 2)])
def test_read(kv, dt, D, page, G):
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(10)
    lens, B, P = [0, 1, 130, 77], 4, 40
    table = _table(B, 9, P, g)
    table[3, 1] = -1
    cache = _filled(kv, P, G, page, D, g)
    idx = torch.randint(-3, 140, (B, 60), generator=g)
    idx[2, :4] = torch.tensor([5, 5, 2 ** 40, -2 ** 40])  # the same slot twice; far outside
    k, v = paged.paged_read(cache, table.cuda(), _i32(lens), idx=idx.cuda(), dtype=dt)
    kd, vd = paged.paged_read(cache, table.cuda(), _i32(lens), n_tokens=150, dtype=dt)
    assert k.shape == (B, 60, G, D) and kd.shape == (B, 150, G, D)
    host = _cpu(cache)
    for b in range(B):
        K, V, has = O.dense(host, table, b, lens[b])
        for got, gotd, x in ((k, kd, K), (v, vd, V)):
            x = x.float().to(dt).transpose(0, 1) if lens[b] else torch.zeros(0, G, D, dtype=dt)
            assert torch.equal(gotd[b, :lens[b]].cpu(), x[:150]) and (gotd[b, lens[b]:] == 0).all()
            for j in range(60):
                s = int(idx[b, j])
                want = x[s] if 0 <= s < lens[b] else torch.zeros(G, D, dtype=dt)
                assert torch.equal(got[b, j].cpu(), want)


def test_step_by_step_matches_oracle_and_graph_replay():
    """As a model uses them: prompts appended and attended, then single tokens
    with a captured append + attention replayed at growing lengths, another
    capture of a second cache sharing nothing but the stream."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(11)
    G, R, D, page, B = 2, 4, 128, 32, 3
    H, mp = G * R, 6
    cos, sin = _tables(mp * page, D)
    table = _table(B, mp, B * mp + 1, g)
    td = table.cuda()
    caches = [paged.new_paged_cache(B * mp + 1, G, D, page_size=page, kv_dtype=kv) for kv in (I8, E4)]

    def step(cache, x, cu, lens, mx):
        q = paged.paged_append(cache, x[:, H:H + G], x[:, H + G:], td, cu, lens, mx, q=x[:, :H], cos=cos, sin=sin)
        return q, paged.paged_attention(q, cache, td, cu, lens, mx)

    new, lens = [70, 1, 33], [70, 1, 33]
    cu = _cum(new)
    for cache in caches:
        x = torch.randn(cu[-1], H + 2 * G, D, generator=g).to(BF16)
        before = _cpu(cache)
        q, out = step(cache, x.cuda(), _i32(cu), _i32(lens), max(new))
        _check_append(cache, before, O.append(before, x[:, H:H + G], x[:, H + G:], table, cu, lens, q=x[:, :H],
                                              cos=cos.cpu(), sin=sin.cpu()), q)
        _check_attend(out, q, cache, table, cu, lens, D ** -0.5)
    # captured single-token steps
    cu1, ld = _i32(_cum([1] * B)), _i32(lens)
    xs = [torch.zeros(B, H + 2 * G, D, dtype=BF16, device="cuda") for _ in caches]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    keep = [[t.clone() for t in c] for c in caches]
    with torch.cuda.stream(side):
        for cache, x in zip(caches, xs):  # warm-up outside the capture
            ld.add_(1)
            step(cache, x, cu1, ld, 1)
            ld.sub_(1)
    side.synchronize()
    for c, old in zip(caches, keep):
        for t, o in zip(c, old):
            t.copy_(o)
    for cache, x in zip(caches, xs):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(cache, x, cu1, ld, 1))
        graphs.append(gr)
    for _ in range(5):
        ld.add_(1)
        lens = [n + 1 for n in lens]
        x1 = torch.randn(B, H + 2 * G, D, generator=g).to(BF16)
        for x in xs:
            x.copy_(x1)
        befores = [_cpu(c) for c in caches]
        for gr in graphs:  # one behind the other, nothing waiting between
            gr.replay()
        torch.cuda.synchronize()
        for cache, before, (q, out) in zip(caches, befores, outs):
            _check_append(cache, before, O.append(before, x1[:, H:H + G], x1[:, H + G:], table, _cum([1] * B), lens,
                                                  q=x1[:, :H], cos=cos.cpu(), sin=sin.cpu()), q)
            _check_attend(out, q, cache, table, _cum([1] * B), lens, D ** -0.5)


def test_two_streams_at_once_and_repeatable():
    """Calls in flight on two streams share nothing; the same call twice
    gives the same bits."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(12)
    G, R, D, page, B = 4, 4, 128, 64, 4
    cache = _filled(E4, 140, G, page, D, g)
    table = _table(B, 32, 140, g).cuda()
    lens, cu = _i32([2000, 1, 777, 1500]), _i32(_cum([1] * B))
    qs = [torch.randn(B, G * R, D, generator=g).to(F16).cuda() for _ in range(2)]
    alone = [paged.paged_attention(q, cache, table, cu, lens, 1) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(paged.paged_attention(qs[i], cache, table, cu, lens, 1))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in got[i])


def test_cascade_keeps_tokens_of_the_cache():
    """The cascade's gather on this cache: the most important tokens' keys and
    values read back and appended to fresh pages, attended over."""
    from spatten_b200 import paged, select
    g = torch.Generator().manual_seed(13)
    G, R, D, page, B, n, K = 2, 2, 64, 16, 2, 100, 37
    cache = _filled(I8, 20, G, page, D, g, spread=False)
    table = _table(B, 7, 20, g)
    imp = torch.rand(B, n, generator=g).cuda()
    kept = select.topk_indices(imp, K)
    k, v = paged.paged_read(cache, table.cuda(), _i32([n] * B), idx=kept)
    small = paged.new_paged_cache(B * 3, G, D, page_size=page, kv_dtype=E4)
    t2 = torch.arange(B * 3, dtype=torch.int32).view(B, 3)
    paged.paged_append(small, k.view(B * K, G, D), v.view(B * K, G, D), t2.cuda(), _i32([0, K, 2 * K]), _i32([K] * B), K)
    host = _cpu(small)
    for b in range(B):
        Kd, _, _ = O.dense(_cpu(cache), table, b, n)
        Ks, _, _ = O.dense(host, t2, b, K)
        want = Kd[:, kept[b].cpu()]
        # bf16, then e4m3 codes of blocks whose scale is under twice what their largest value needs
        assert ((Ks - want).abs() <= (2.0 ** -4 + 2.0 ** -8) * want.abs() + 2.0 ** -9 * want.abs().max() / 224).all()
    q = torch.randn(B, G * R, D, generator=g).to(BF16).cuda()
    out = paged.paged_attention(q, small, t2.cuda(), _i32([0, 1, 2]), _i32([K] * B), 1)
    _check_attend(out, q, small, t2, [0, 1, 2], [K] * B, D ** -0.5)


def test_refusals():
    from spatten_b200 import paged
    c = paged.new_paged_cache(4, 2, 64, page_size=16)
    t, cu, ln = _i32([[0, 1]]), _i32([0, 1]), _i32([1])
    x = torch.zeros(1, 2, 64, dtype=F16, device="cuda")
    for bad in (dict(k=x[:, :1]), dict(v=x.float()), dict(v=x.to(BF16)), dict(cos=torch.zeros(4, 32, device="cuda")),
                dict(page_table=t.long()), dict(page_table=_i32([[0], [1]])), dict(seq_lens=_i32([1, 1])),
                dict(q=x, q_norm_w=torch.ones(64, dtype=F16, device="cuda")), dict(k=x.cpu()),
                dict(positions=_i32([0])), dict(k=torch.zeros(1, 2, 128, dtype=F16, device="cuda")[..., ::2])):
        args = dict(k=x, v=x, page_table=t, cu_tokens=cu, seq_lens=ln) | bad
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            paged.paged_append(c, max_tokens=1, **args)
    for bad in (torch.zeros(1, 3, 64, dtype=F16, device="cuda"), x.float(), torch.zeros(1, 2, 128, dtype=F16, device="cuda")):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            paged.paged_attention(bad, c, t, cu, ln, 1)
    with pytest.raises(ValueError):
        paged.paged_read(c, t, ln, idx=_i32([[0]]))
    with pytest.raises(TypeError):
        paged.paged_read(c, t, ln, dtype=torch.float32)


def _device_error():
    import ctypes
    from spatten_b200 import _native as N
    code = ctypes.c_uint(1)
    N.check(N.lib.spatten_device_error(ctypes.byref(code), 0))
    return code.value


@pytest.mark.parametrize("kv,dt,D,page,G,R,news,lens,pad", [
    # every sequence as long as the largest: the tensor-memory kernel serves all of them
    (I8, BF16, 128, 64, 2, 4, [40, 40], [200, 41], 0),
    (E4, F16, 64, 32, 3, 3, [90, 90, 90], [90, 300, 91], 0),
    # mixed with shorter ones, one row tile and two, borders of both
    (I8, F16, 128, 32, 1, 4, [33, 32, 31, 64, 65], [64, 200, 31, 64, 513], 7),
    (E4, BF16, 128, 16, 2, 5, [1, 60, 0, 26, 2], [500, 77, 9, 26, 130], 3),
    (I8, BF16, 64, 128, 2, 16, [9, 1, 17], [300, 129, 17], 1),
    (E4, F16, 128, 64, 1, 128, [1, 2, 3], [64, 65, 130], 0),
    (I8, F16, 128, 64, 1, 100, [3, 1], [200, 64], 0),
])
def test_attention_pieces(kv, dt, D, page, G, R, news, lens, pad):
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(21)
    B, H = len(news), G * R
    mp = max(lens) // page + 1
    P = B * mp + 2
    table, cu = _table(B, mp, P, g), _cum(news)
    cache = _filled(kv, P, G, page, D, g)
    q = torch.randn(cu[-1] + pad, H, D, generator=g).to(dt).cuda()
    out = torch.full_like(q, 3.0)
    paged.paged_attention(q, cache, table.cuda(), _i32(cu), _i32(lens), max(news), out=out)
    _check_attend(out, q, cache, table, cu, lens, D ** -0.5)
    assert (out[cu[-1]:] == 3).all()
    again = paged.paged_attention(q, cache, table.cuda(), _i32(cu), _i32(lens), max(news))
    assert torch.equal(again[:cu[-1]], out[:cu[-1]])
    assert _device_error() == 0


@pytest.mark.parametrize("kv", [I8, E4])
def test_attention_pieces_masked_places(kv):
    """As test_attention_masked_places, with enough rows for the
    tensor-memory kernel; a row that is not finite stays alone; a negative
    scale of the scores."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(22)
    G, R, D, page = 2, 4, 128, 32
    news, lens = [50, 40, 0, 70], [0, 25, 40, 260]
    cu, B = _cum(news), 4
    table = _table(B, 9, 40, g)
    table[3, 1], table[3, 4], table[1, 0] = -1, 1000, -3
    cache = _filled(kv, 40, G, page, D, g)
    used = torch.zeros(40, dtype=torch.bool)
    for b in range(B):
        for s in range(lens[b]):
            if 0 <= table[b, s // page] < 40:
                used[table[b, s // page]] = True
        last = int(table[b, lens[b] // page])
        if 0 <= last < 40:
            for t in cache[:2]:
                t.view(I8)[last, :, lens[b] % page:] = 0x7F
    for t in cache[2:]:
        t[(~used).cuda()] = float("nan")
    q = torch.randn(cu[-1], G * R, D, generator=g).to(BF16).cuda()
    for sm in (D ** -0.5, -0.05):
        out = paged.paged_attention(q, cache, table.cuda(), _i32(cu), _i32(lens), max(news), sm_scale=sm)
        want, A, S = O.attend(q.cpu(), _cpu(cache), table, cu, lens, sm)
        S = S.abs().clamp(min=1.0) if sm < 0 else S
        tol = 2.0 ** -8 * want.abs() + A * (2.0 ** -11 + 2 * D * U * (abs(sm) * 127 * 4 * D) + 2.0 ** -16) + 1e-38
        assert ((out.cpu().double() - want).abs() <= tol).all()
        assert (out[:50] == 0).all() and (out[50:50 + 15] == 0).all()  # nothing held; the first 15 of 40 with 25 slots
    bad = q.clone()
    bad[100, 3, 5], bad[101, 6, 0] = float("nan"), float("inf")
    got = paged.paged_attention(bad, cache, table.cuda(), _i32(cu), _i32(lens), max(news), sm_scale=-0.05)
    assert torch.isnan(got[100, 3]).all() and torch.isnan(got[101, 6]).all()
    same = torch.ones(out.shape[:2], dtype=torch.bool)
    same[100, 3] = same[101, 6] = False
    assert torch.equal(got[same.cuda()], out[same.cuda()])
    assert _device_error() == 0


def test_attention_pieces_extremes():
    """test_attention_extremes with 80 queries per KV head."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(23)
    G, R, D, page, n, T = 1, 4, 128, 16, 200, 20
    table = _table(1, 13, 15, g)
    cache = _filled(I8, 15, G, page, D, g, spread=False)
    cache.v_scale[:, 0] = 2.0 ** torch.linspace(-100, 100, 15)[torch.randperm(15, generator=g)].round().cuda()
    cache.v_scale[int(table[0, 2])] = 0.0
    cache.k_scale[int(table[0, 4])] = 0.0
    q = torch.randn(T, R, D, generator=g).to(BF16).cuda()
    for x in (q, (q.float() * 300).to(BF16)):
        out = paged.paged_attention(x, cache, table.cuda(), _i32([0, T]), _i32([n]), T)
        _check_attend(out, x, cache, table, [0, T], [n], D ** -0.5)


def test_attention_many_sequences():
    """More sequences than the threads that number them, for both kernels, and
    more than one launch can take."""
    from spatten_b200 import _native as N
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(24)
    G, D, page, P = 1, 64, 16, 50
    cache = _filled(I8, P, G, page, D, g)
    for B, R, hi in ((700, 1, 2), (700, 3, 30), (1100, 16, 5)):
        news = torch.randint(0, hi, (B,), generator=g).tolist()
        news[B // 2] = hi
        lens = [n + int(x) for n, x in zip(news, torch.randint(0, 20, (B,), generator=g))]
        table = torch.randint(0, P, (B, 4), generator=g).to(torch.int32)  # pages shared by the sequences
        cu = _cum(news)
        q = torch.randn(cu[-1], R, D, generator=g).to(F16).cuda()
        out = paged.paged_attention(q, cache, table.cuda(), _i32(cu), _i32(lens), hi)
        _check_attend(out, q, cache, table, cu, lens, D ** -0.5)
    B = 8193
    with pytest.raises(N.SpattenError, match="at most 8192"):
        paged.paged_attention(q[:1], cache, torch.zeros(B, 1, dtype=torch.int32, device="cuda"), _i32([0] * B + [1]),
                              _i32([1] * B), 1)


def test_attention_captured_over_changing_pieces():
    """One captured call, replayed while the sequences' new tokens, lengths and
    pages change: sequences move between the two kernels."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(25)
    G, R, D, page, B, T, mx = 2, 4, 128, 32, 3, 150, 100
    cache = _filled(E4, 60, G, page, D, g)
    q = torch.randn(T, G * R, D, generator=g).to(BF16).cuda()
    td, cu, ln = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((B, 12), B + 1, B))
    paged.paged_attention(q, cache, td, cu, ln, mx)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = paged.paged_attention(q, cache, td, cu, ln, mx)
    for news, lens in (([1, 100, 20], [300, 100, 50]), ([70, 1, 1], [70, 384, 2]), ([16, 17, 0], [16, 40, 9])):
        table = _table(B, 12, 60, g)
        td.copy_(table)
        cu.copy_(_i32(_cum(news)))
        ln.copy_(_i32(lens))
        gr.replay()
        torch.cuda.synchronize()
        _check_attend(out, q, cache, table, _cum(news), lens, D ** -0.5)


@pytest.mark.parametrize("kv,D,R,n,last", [(I8, 128, 2, 150, 150), (E4, 64, 2, 150, 129), (I8, 128, 3, 171, 40)])
def test_attention_pieces_many_lines(kv, D, R, n, last):
    """More lines of query rows than CTAs, every other with one row tile of two
    in use, so that a CTA goes from one kind to the other."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(26)
    G, page, B = 8, 64, 12
    news = [n] * (B - 1) + [last]
    lens = [x + 64 * b + 30 for b, x in enumerate(news)]
    mp = max(lens) // page + 1
    table, cu = _table(B, mp, B * mp, g), _cum(news)
    cache = _filled(kv, B * mp, G, page, D, g)
    q = torch.randn(cu[-1], G * R, D, generator=g).to(F16).cuda()
    out = paged.paged_attention(q, cache, table.cuda(), _i32(cu), _i32(lens), max(news))
    _check_attend(out, q, cache, table, cu, lens, D ** -0.5)
    for _ in range(5):
        assert torch.equal(paged.paged_attention(q, cache, table.cuda(), _i32(cu), _i32(lens), max(news)), out)
    assert _device_error() == 0


@pytest.mark.parametrize("R,n", [(2, 5), (8, 40)])
def test_index_tensors_out_of_range(R, n):
    """cu_tokens that leave the rows, descend or claim every row many times,
    lengths below zero and far beyond the page table: sequences that are in
    order come out right, nothing is touched outside."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(31)
    G, D, page, T = 2, 64, 16, 3 * n
    big = 2 ** 31 - 1
    cu = [0, n, n, -7, 2 * n, 2 * n - 3, big]
    lens = [n + 50, 9, -big, 3, big, n]
    table = _table(6, 8, 60, g)
    table[5] = -1
    cache = _filled(I8, 60, G, page, D, g)
    q = torch.randn(T, G * R, D, generator=g).to(F16).cuda()
    out = paged.paged_attention(q, cache, table.cuda(), _i32(cu), _i32(lens), n)
    _check_attend(out[:n], q[:n], cache, table[:1], cu[:2], lens[:1], D ** -0.5)
    before = _cpu(cache)
    x = torch.randn(T, 2 * G, D, generator=g).to(F16).cuda()
    own = torch.full_like(table, -1)
    own[0] = table[0]
    paged.paged_append(cache, x[:, :G], x[:, G:], own.cuda(), _i32(cu), _i32(lens), n)
    want = O.append(before, x[:n, :G].cpu(), x[:n, G:].cpu(), own[:1], [0, n], lens[:1])
    _check_append(cache, before, want)
    k, _ = paged.paged_read(cache, table.cuda(), _i32(lens), n_tokens=140)
    assert (k[2] == 0).all() and (k[4, 128:] == 0).all()
    # every sequence claims every row: more work than the numbering holds in earnest, none of it out of range
    B = 600
    many = _i32([0 if b % 2 == 0 else T for b in range(B + 1)])
    out = paged.paged_attention(q, cache, table[:1].expand(B, -1).contiguous().cuda(), many, _i32([n + 50] * B), T)
    assert out.shape == q.shape and _device_error() == 0


def test_copies_of_a_cache():
    import copy
    from spatten_b200 import paged
    c = paged.new_paged_cache(3, 1, 64, page_size=16)
    t, ln = _i32([[0]]), _i32([4])
    paged.paged_read(c, t, ln)  # its C form exists
    d = copy.deepcopy(c)
    x = torch.ones(4, 1, 64, dtype=F16, device="cuda")
    paged.paged_append(d, x, x, t, _i32([0, 4]), ln, 4)
    assert (c.k == 0).all() and (d.k[0, 0, :4] == 127).all()
    assert copy.copy(d).k.data_ptr() == d.k.data_ptr()
