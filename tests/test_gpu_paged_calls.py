"""Calls of the paged cache's Python entry points that batches make at their
edges: no sequences, columns of other tensors, one page table for all."""
import pytest
import torch

from oracle import paged as O
from tests.test_gpu_paged import BF16, F16, I8, _check_attend, _cpu, _cum, _filled, _i32, _table

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


@pytest.mark.parametrize("cols", [3, 0])
def test_no_sequences(cols):
    from spatten_b200 import paged
    c = paged.new_paged_cache(4, 2, 64, page_size=16)
    t = torch.zeros(0, cols, dtype=torch.int32, device="cuda")
    x = torch.zeros(0, 2, 64, dtype=F16, device="cuda")
    assert paged.paged_append(c, x, x, t, _i32([0]), _i32([]), 0, q=x).shape == (0, 2, 64)
    assert paged.paged_attention(x, c, t, _i32([0]), _i32([]), 0).shape == (0, 2, 64)
    k, v = paged.paged_read(c, t, _i32([]), n_tokens=5)
    assert k.shape == v.shape == (0, 5, 2, 64)
    # rows of a padded batch, none of them a sequence's
    out = torch.full((3, 2, 64), 5.0, dtype=F16, device="cuda")
    paged.paged_attention(out.clone(), c, t, _i32([0]), _i32([]), 1, out=out)
    assert (out == 5).all()


def test_columns_of_other_tensors():
    """Index tensors with one column: the stride of a dimension of one entry
    says nothing."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(61)
    G, D, page, lens = 2, 64, 16, [5, 16, 1]
    cache = _filled(I8, 8, G, page, D, g)
    table = _table(3, 1, 8, g)
    wide = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    wide[1] = table[:, 0].cuda()
    column = wide[1:].t()  # [3, 1], strides (1, 3)
    assert column.stride() == (1, 3)
    q = torch.randn(3, G, D, generator=g).to(BF16).cuda()
    cu = _cum([1] * 3)
    out = paged.paged_attention(q, cache, column, _i32(cu), _i32(lens), 1)
    _check_attend(out, q, cache, table, cu, lens, D ** -0.5)
    idx = torch.tensor([[9, 3, 9], [4, 15, 0]], device="cuda")[1:].t()
    for got, want in zip(paged.paged_read(cache, column, _i32(lens), idx=idx),
                         paged.paged_read(cache, table.cuda(), _i32(lens), idx=idx.contiguous())):
        assert torch.equal(got, want)
    before = _cpu(cache)
    x = torch.randn(3, 2 * G, D, generator=g).to(BF16).cuda()
    paged.paged_append(cache, x[:, :G], x[:, G:], column, _i32(cu), _i32(lens), 1)
    want = O.append(before, x[:, :G].cpu(), x[:, G:].cpu(), table, cu, lens)
    for got, c in zip(_cpu(cache)[:2], want[1]):
        assert ((O.code_values(got) - c).abs() <= 1).all()


def test_one_table_for_every_sequence():
    """Samples of one prompt that only read it: an expanded page table."""
    from spatten_b200 import paged
    g = torch.Generator().manual_seed(62)
    G, R, D, page, lens = 2, 4, 128, 32, [100, 33, 100]
    cache = _filled(I8, 6, G, page, D, g)
    table = _table(1, 4, 6, g).cuda()
    for new in ([1, 1, 1], [30, 20, 25]):
        cu = _cum(new)
        q = torch.randn(cu[-1], G * R, D, generator=g).to(BF16).cuda()
        out = paged.paged_attention(q, cache, table.expand(3, -1), _i32(cu), _i32(lens), max(new))
        _check_attend(out, q, cache, table.cpu().expand(3, -1), cu, lens, D ** -0.5)
    for a, b in zip(paged.paged_read(cache, table.expand(3, -1), _i32(lens)),
                    paged.paged_read(cache, table.repeat(3, 1), _i32(lens))):
        assert torch.equal(a, b)
    x = torch.zeros(3, G, D, dtype=BF16, device="cuda")
    with pytest.raises(RuntimeError, match="stride"):
        paged.paged_append(cache, x, x, table.expand(3, -1), _i32([0, 1, 2, 3]), _i32(lens), 1)
