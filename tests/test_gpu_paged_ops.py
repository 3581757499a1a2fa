"""A loop that drafts trees into a cache of bounded length, by the registered
operators alone (torch.ops.spatten): weights and positions go with their tokens."""
import pytest
import torch

from oracle import paged_tokens as OT
from tests.test_gpu_paged import BF16, I8, _cpu, _cum, _filled, _i32, _table
from tests.test_gpu_paged_tokens import _check, _weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def test_weighed_tree_then_keep_then_evict():
    from spatten_b200 import paged
    import spatten_b200.torch_ops  # noqa: F401
    ops, g = torch.ops.spatten, torch.Generator().manual_seed(71)
    G, R, D, page = 2, 2, 64, 16
    a = _filled(I8, 8, G, page, D, torch.Generator().manual_seed(72))
    b = paged.PagedKVCache(*(t.clone() for t in a))
    table, cu, lens, parents = _table(2, 4, 8, g), _cum([5, 4]), [45, 54], [-1, 0, 0, 1, 2, -1, 0, 0, 1]
    tree, pos = ops.paged_tree(_i32(parents), _i32(cu), _i32(lens), 5)
    q = torch.randn(9, G * R, D, generator=g).to(BF16).cuda()
    wa = _weights(a, g)
    wb = paged.PagedWeights(*(t.clone() for t in wa))
    before = paged.PagedWeights(*(t.clone() for t in wa))
    out = ops.paged_weighing_attention(q, *a, *wa, table.cuda(), _i32(cu), _i32(lens), pos, 5, D ** -0.5, tree)
    _check(out, q, a, table, cu, lens, D ** -0.5, OT.tree(parents, cu, lens, 5)[0], before, wa, pos.tolist())
    assert torch.equal(out, paged.paged_attention(q, b, table.cuda(), _i32(cu), _i32(lens), 5, tree=tree, weights=wb,
                                                  positions=pos))
    accepted = [[0, 2, 4], [0, 2, -1]]
    codes, was = _cpu(a), [t.cpu() for t in wa]
    kept = ops.paged_keep_weighed(*a, *wa, table.cuda(), _i32(cu), _i32(lens), _i32(accepted))
    moves, new = OT.keep(codes, table, cu, lens, accepted)
    assert kept.tolist() == new and any(m[0] for m in moves)
    for got, t in zip(wa, was):
        assert torch.equal(got.cpu(), OT.move_beside(t, table, moves)) and not torch.equal(got.cpu(), t)
    assert torch.equal(kept, paged.paged_keep(b, table.cuda(), _i32(cu), _i32(lens), _i32(accepted), weights=wb))
    assert torch.equal(ops.paged_evict(*a, *wa, table.cuda(), kept, 20, 3, False),
                       paged.paged_evict(b, wb, table.cuda(), kept, 20, recent=3))
    for x, y in zip((*a, *wa), (*b, *wb)):
        assert torch.equal(x, y)
