"""Argument checks of the paged KV cache's C entry points (CPU): what they
refuse, and what they take although it looks odd."""
import pytest

from spatten_b200 import _native as N
from tests.test_paged_host import _append, _attend, _read, _run


@pytest.mark.parametrize("T,H,st,sh,ok", [
    (3, 8, 128, 128, False),             # head 1 of token 0 is head 0 of token 1
    (3, 8, 256, 128, False),             # ... and head 2 of token 0
    (3, 8, 128, 256, False),
    (3, 8, 8 * 128 - 8, 128, False),     # one row into the next by 8 elements
    (3, 8, 8 * 128, 128, True),          # token-major
    (3, 8, 128, 3 * 128, True),          # head-major
    (3, 8, 128, 3 * 128 - 8, False),
    (1, 8, 0, 128, True), (1, 8, 0, 120, False), (3, 1, 128, 0, True), (3, 1, 120, 0, False),
    (3, 8, 2 ** 62, 2 ** 61, False),     # products past 64 bits
    (3, 8, 2 ** 62, 2 ** 59 - 8, True),
])
def test_rows_of_an_output_do_not_interleave(T, H, st, sh, ok):
    """Launches are not reached: a call whose output passes is refused for its
    tables, or for its workspace."""
    a = _append(H=H, T=T, B=1, max_tokens=T, qo_st=st, qo_sh=sh, cs_rows=0)
    assert N.lib.spatten_paged_append(a, None) == N.ERR_INVALID
    err = N.lib.spatten_last_error().decode()
    assert ("rows of q_out overlap" in err) == (not ok) and ("cos/sin rows" in err) == ok, err
    a = _attend(cache={"G": 1}.items(), H=H, T=T, B=1, max_tokens=T, o_st=st, o_sh=sh)
    assert N.lib.spatten_paged_attend(a, None, 0, None) == N.ERR_INVALID
    err = N.lib.spatten_last_error().decode()
    assert ("rows of out overlap" in err) == (not ok) and ("workspace of" in err) == ok, err


@pytest.mark.parametrize("max_pages", [4, 0])
def test_batches_without_sequences(max_pages):
    """Tensors of an empty batch have no memory: their pointers are null."""
    none = dict(page_table=0, max_pages=max_pages, table_stride=max_pages).items()
    empty = dict(B=0, T=0, max_tokens=0, cu_tokens=1 << 20, seq_lens=0)
    assert N.lib.spatten_paged_append(_append(cache=none, q=0, k=0, v=0, q_out=0, **empty), None) == N.OK
    a = _attend(cache=none, q=0, out=0, **empty)
    assert N.lib.spatten_paged_attend_workspace_size(a) == 0
    assert N.lib.spatten_paged_attend(a, None, 0, None) == N.OK
    assert N.lib.spatten_paged_read(_read(cache=none, B=0, seq_lens=0, idx=0, k_out=0, v_out=0), None) == N.OK
    assert N.lib.spatten_paged_read(_read(cache=none), None) == N.ERR_INVALID  # three sequences need one


def test_one_table_for_every_sequence():
    """A row stride of 0: sequences that share their pages may read them, not
    append to them."""
    shared = dict(table_stride=0).items()
    a = _attend(cache=shared)
    assert N.lib.spatten_paged_attend(a, None, 0, None) == N.ERR_INVALID
    assert "workspace of" in N.lib.spatten_last_error().decode()  # that is all it misses
    assert N.lib.spatten_paged_read(_read(cache=shared, k_out=0, v_out=0), None) == N.ERR_INVALID
    assert "neither k_out" in N.lib.spatten_last_error().decode()
    assert N.lib.spatten_paged_append(_append(cache=shared), None) == N.ERR_INVALID
    assert "stride" in N.lib.spatten_last_error().decode()
