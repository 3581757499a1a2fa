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
