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
