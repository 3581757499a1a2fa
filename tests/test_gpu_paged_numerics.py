"""Where the paged attention's kernels could keep fewer bits than their formula:
query rows with outlier channels, weights far below the row's largest. Bounds
are those of tests/test_gpu_paged.py, with the score term as it is there: the
rounding of a sum of exact products."""
import pytest
import torch

from oracle import paged as O
from tests.test_gpu_paged import BF16, E4, F16, I8, U, _check_attend, _cpu, _filled, _i32, _table

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


@pytest.mark.parametrize("kv", [I8, E4])
@pytest.mark.parametrize("dt,outlier", [(BF16, 40.0), (F16, 40.0), (BF16, 90.0), (BF16, 900.0), (F16, 900.0), (F16, 60000.0)])
@pytest.mark.parametrize("T", [1, 4, 40])
def test_outlier_channels(kv, dt, outlier, T):
    """A channel in which the keys hold little may hold a query's largest
    element: the others keep their bits (T = 40: the kernel for pieces)."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(41)
    G, R, D, page, n = 2, 2, 128, 64, 300
    table = _table(1, 5, 7, g)
    cache = _filled(kv, 7, G, page, D, g, spread=False)
    cache.k.view(I8)[..., 17] = 0
    q = 3 * torch.randn(T, G * R, D, generator=g)
    q[..., 17] = outlier
    q = q.to(dt).cuda()
    out = paged.paged_attention(q, cache, table.cuda(), _i32([0, T]), _i32([n]), T)
    _check_attend(out, q, cache, table, [0, T], [n], D ** -0.5)


@pytest.mark.parametrize("kv", [I8, E4])
@pytest.mark.parametrize("D,R,T", [(64, 8, 1), (128, 1, 5), (128, 4, 3), (64, 2, 50)])
def test_rows_of_all_kinds_side_by_side(kv, D, R, T):
    """Rows of zeros, of one element, of bf16's smallest and largest values, and
    with every magnitude from 2^-40 to 1, beside plain ones."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(42)
    G, page, n = 2, 32, 130
    table = _table(1, 5, 7, g)
    cache = _filled(kv, 7, G, page, D, g, spread=False)
    q = torch.randn(T, G * R, D, generator=g)
    flat = q.view(-1, D)
    flat[0] = 0
    flat[1 % len(flat)] *= 2.0 ** -120
    flat[2 % len(flat)] = 0
    flat[2 % len(flat), 5] = -3.0
    flat[3 % len(flat)] *= 2.0 ** (-40 * torch.rand(D, generator=g))
    flat[4 % len(flat)] *= 1e-39
    q = q.to(BF16).cuda()
    out = paged.paged_attention(q, cache, table.cuda(), _i32([0, T]), _i32([n]), T)
    _check_attend(out, q, cache, table, [0, T], [n], D ** -0.5)
    alone = out.clone()
    q.view(-1, D)[0] = float("nan")  # a row that is not finite stays alone
    out = paged.paged_attention(q, cache, table.cuda(), _i32([0, T]), _i32([n]), T)
    assert torch.isnan(out.view(-1, D)[0]).all()
    other = torch.ones(T * G * R, dtype=torch.bool)
    other[0] = False
    assert torch.isfinite(out.view(-1, D)[other.cuda()]).all()
    part = out.view(-1, D).clone()
    part[0] = alone.view(-1, D)[0]
    q.view(-1, D)[0] = 0
    _check_attend(part.view_as(out), q, cache, table, [0, T], [n], D ** -0.5)


@pytest.mark.parametrize("kv", [I8, E4])
@pytest.mark.parametrize("T", [1, 4, 30])
@pytest.mark.parametrize("below", [18.0, 25.5, 29.0])
def test_many_weak_keys_beside_a_strong_one(kv, T, below):
    """A key with nearly all the weight whose values are zeros, and keys of
    2^-below of its weight that make the whole output. A weight is an fp16 of
    which the row's largest is 2^7 or more, so one below 2^-21 of it is off by at
    most half of fp16's smallest step, 2^-25 / 2^7 = 2^-32 of the largest."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(43)
    R, D, page, n, strong = 4, 128, 16, 600, 37
    top = 127 if kv == I8 else 448
    table = _table(1, 38, 40, g)
    cache = paged.new_paged_cache(40, 1, D, page_size=page, kv_dtype=kv)

    def put(t, x):
        t.view(I8).copy_(x.round().to(I8) if kv == I8 else x.to(E4).view(I8))
    q = torch.randn(D, generator=g)
    k = torch.randn(40, 1, page, D, generator=g) * top / 5
    v = torch.rand(40, 1, page, D, generator=g) * (top - 1) + 1
    pid, row = int(table[0, strong // page]), strong % page
    k[pid] = 0
    k[pid, 0, row] = q / q.abs().max() * top
    v[pid, 0, row] = 0
    put(cache.k, k.clamp(-top, top))
    put(cache.v, v)
    cache.v_scale.fill_(2.0 ** (below - 14))
    cache.k_scale.fill_(2.0 ** -20 / top)  # the weak keys' scores: near 0
    cache.k_scale[pid] = 1.0 / top
    q = q.to(F16)
    score = float((q.double() * O.code_values(cache.k[pid, 0, row].cpu()) / top).sum())
    sm = below * 0.6931471805599453 / score
    q = q.expand(T, R, D).contiguous().cuda()
    out = paged.paged_attention(q, cache, table.cuda(), _i32([0, T]), _i32([n]), T, sm_scale=sm)
    want, A, S = O.attend(q.cpu(), _cpu(cache), table, [0, T], [n], sm)
    tol = 2.0 ** -11 * want.abs() + A * (2.0 ** -11 + 2 * D * U * S + 2.0 ** -16) + \
        n * 2.0 ** -32 * top * 2.0 ** (below - 14) + torch.finfo(F16).smallest_normal
    assert ((out.cpu().double() - want).abs() <= tol).all()
    assert (tol < 0.3 * want.abs()).all()  # they are seen
