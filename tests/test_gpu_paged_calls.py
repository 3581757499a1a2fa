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
