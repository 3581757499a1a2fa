"""The tensor-memory kernel of the paged attention (pieces of prompts): masked
places to the bounds of tests/test_gpu_paged.py, rows of a fused projection, calls
in flight on two streams, more work than the numbering of units holds."""
import pytest
import torch

from oracle import paged as O
from tests.test_gpu_paged import BF16, E4, F16, I8, U, _cpu, _cum, _device_error, _filled, _i32, _table

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _close(out, want, A, S, D, n):
    """_check_attend's bound (S: of a negative scale too)."""
    tol = torch.finfo(out.dtype).eps / 2 * want.abs() + A * (2.0 ** -11 + 2 * D * U * S.abs() + 2.0 ** -16) + \
        n * U * A.amax(-1, keepdim=True) + torch.finfo(out.dtype).smallest_normal
    return ((out.cpu().double() - want).abs() <= tol)


def _masked(kv, lens, table, P, G, page, D, g):
    """A pool with garbage wherever no key is: codes behind a sequence's last
    slot, scales of pages that no sequence uses."""
    cache = _filled(kv, P, G, page, D, g)
    used = torch.zeros(P, dtype=torch.bool)
    for b, n in enumerate(lens):
        for s in range(n):
            if 0 <= table[b, s // page] < P:
                used[table[b, s // page]] = True
        last = int(table[b, n // page])
        if n % page and 0 <= last < P:
            for t in cache[:2]:
                t.view(I8)[last, :, n % page:] = 0x7F
    for t in cache[2:]:
        t[(~used).cuda()] = float("nan")
    return cache


@pytest.mark.parametrize("kv", [I8, E4])
@pytest.mark.parametrize("sm", [128 ** -0.5, -0.05])
@pytest.mark.parametrize("R,news,lens", [(4, [50, 40, 0, 70], [0, 25, 40, 260]), (1, [3, 0, 66, 2], [3, 7, 130, 250]),
                                         (4, [1, 3, 2, 2], [9, 40, 2, 257])])
def test_masked_places(kv, sm, R, news, lens):
    """Pages without memory, empty rows, garbage behind the last slots: a key
    too many or too few would change an output by a multiple of the bound. The
    last two have few rows for a sequence, the last none for this kernel."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(51)
    G, D, page = 2, 128, 32
    cu, B = _cum(news), 4
    table = _table(B, 9, 40, g)
    table[3, 1], table[3, 4], table[1, 0] = -1, 1000, -3
    cache = _masked(kv, lens, table, 40, G, page, D, g)
    q = torch.randn(cu[-1], G * R, D, generator=g).to(BF16).cuda()
    out = paged.paged_attention(q, cache, table.cuda(), _i32(cu), _i32(lens), max(news), sm_scale=sm)
    want, A, S = O.attend(q.cpu(), _cpu(cache), table, cu, lens, sm)
    if sm < 0:  # the oracle's S is the largest of a negative multiple: the smallest magnitude
        _, _, S = O.attend(q.cpu(), _cpu(cache), table, cu, lens, -sm)
    ok = _close(out, want, A, S, D, max(lens))
    assert ok.all(), (~ok).nonzero()[:4].tolist()
    # the bound does see a foreign key: the value of one more slot at an average weight
    seen = want.abs().amax((1, 2)) > 0
    assert not _close(out[seen.cuda()] * (1 - 1 / max(lens)), want[seen], A[seen], S[seen], D, max(lens)).all()
    assert _device_error() == 0


@pytest.mark.parametrize("kv,dt", [(I8, BF16), (E4, F16)])
def test_rows_of_a_fused_projection(kv, dt):
    """q as a slice of [T, (H + 2 G) D] rows, head-major q, an output inside a
    wider row: the results of contiguous ones, and nothing beside them written."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(52)
    G, R, D, page = 2, 4, 128, 64
    H, news, lens = G * R, [70, 1, 33], [200, 64, 33]
    cu, T = _cum(news), 104
    table = _table(3, 4, 12, g)
    cache = _filled(kv, 12, G, page, D, g)
    x = torch.randn(T, H + 2 * G, D, generator=g).to(dt).cuda()
    args = (cache, table.cuda(), _i32(cu), _i32(lens), max(news))
    want = paged.paged_attention(x[:, :H].contiguous(), *args)
    w64, A, S = O.attend(x[:, :H].cpu(), _cpu(cache), table, cu, lens, D ** -0.5)
    assert _close(want, w64, A, S, D, max(lens)).all()
    assert torch.equal(paged.paged_attention(x[:, :H], *args), want)
    major = x[:, :H].transpose(0, 1).contiguous().transpose(0, 1)  # [H, T, D] in memory
    wide = torch.full((T, 2 * H, D + 8), 7.0, dtype=dt, device="cuda")
    out = wide[:, 1::2, :D]
    assert paged.paged_attention(major, *args, out=out) is out and torch.equal(out, want)
    wide[:, 1::2, :D] = 7.0
    assert (wide == 7).all()
    rows = torch.full((H, T, D), 7.0, dtype=dt, device="cuda").transpose(0, 1)
    paged.paged_attention(x[:, :H], *args, out=rows)
    assert torch.equal(rows, want) and _device_error() == 0


def test_two_streams_at_once():
    """Pieces in flight on two streams share nothing."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(53)
    G, R, D, page, B = 4, 4, 128, 64, 2
    cache = _filled(I8, 70, G, page, D, g)
    table = _table(B, 32, 70, g).cuda()
    news, lens = [[100, 64], [5, 200]], [[2000, 64], [1500, 777]]
    qs = [torch.randn(sum(n), G * R, D, generator=g).to(F16).cuda() for n in news]
    ix = [(_i32(_cum(n)), _i32(ln), max(n)) for n, ln in zip(news, lens)]
    alone = [paged.paged_attention(q, cache, table, *i) for q, i in zip(qs, ix)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(paged.paged_attention(qs[i], cache, table, *ix[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in got[i])
    assert _device_error() == 0


@pytest.mark.parametrize("B,T,slots", [(1024, 16384, 8192), (8192, 4096, 8192)])
def test_more_work_than_the_numbering_holds(B, T, slots):
    """Sequences that all claim the same rows, by more units of work than 32
    bits number (first the tensor-memory kernel's, then the other's): nothing is
    done, the output stays as it was."""
    from spatten_b200 import paged
    G, R, D, page = 8, 8, 64, 128
    # units of one sequence, at the least: its row tiles times the tiles (keys) they see
    rows = T * R // (256 if B <= 1024 else 16)
    assert B * G * rows * (slots // 2 if B <= 1024 else slots // 16) > 2 ** 32
    cache = paged.new_paged_cache(4, G, D, page_size=page)
    table = torch.zeros(B, slots // page, dtype=torch.int32, device="cuda")
    cu = _i32([0 if b % 2 == 0 else T for b in range(B + 1)])  # every other one claims all rows
    q = torch.zeros(T, G * R, D, dtype=F16, device="cuda")
    out = torch.full_like(q, 3.0)
    paged.paged_attention(q, cache, table, cu, _i32([slots + T] * B), T, out=out)
    assert (out == 3).all() and _device_error() == 0
    # the same claims of one sequence are work in order
    one = paged.paged_attention(q, cache, table[:1], cu[:2], _i32([slots]), T, out=out)
    assert (one == 0).all() and _device_error() == 0
