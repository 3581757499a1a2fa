"""Workspaces of the paged cache's calls go by the pool where page tables are wider (CPU)."""
import pytest

from spatten_b200 import _native as N
from tests.test_paged_tokens_host import _evict


@pytest.mark.parametrize("recent", [0, 5])
@pytest.mark.parametrize("B,per_head,page,max_pages,P", [
    (256, 1, 64, 2048, 20480),       # 131072 slots reserved for each of 256 sequences: 2.5 GiB of codes
    (256, 1, 64, 1 << 14, 20480),    # ... 2^20
    (4096, 0, 16, 4096, 50000),
    (1, 1, 128, 8192, 100),
])
def test_eviction(B, per_head, page, max_pages, P, recent):
    """Per slot and line of the pool a key, a position and two places in lists; beside them a
    number for each block that `keep` has in a line."""
    G, keep = 8, 1024
    cache = dict(G=G, page_size=page, max_pages=max_pages, table_stride=max_pages, num_pages=P).items()
    n = N.lib.spatten_paged_evict_workspace_size(_evict(cache=cache, B=B, per_head=per_head, keep=keep, recent=recent))
    lines = G if per_head else 1
    slots, blocks = P * page, -(-min(keep, P * page) // page)
    assert 0 < n <= lines * slots * (16 if recent else 12) + B * lines * (4 * (blocks + 1) + 16) + B * G * 8 + 8 * 256
    assert n < 0.15 * 2 * P * G * page * 128  # of the codes


def test_eviction_by_sequence_where_that_is_less():
    few = dict(G=8, page_size=64, max_pages=20, table_stride=20, num_pages=100000).items()
    n = N.lib.spatten_paged_evict_workspace_size(_evict(cache=few, B=4, per_head=1, keep=640, recent=1))
    assert n <= 4 * 8 * 1280 * 16 + 4 * 8 * (4 * 11 + 16) + 4 * 8 * 8 + 8 * 256
