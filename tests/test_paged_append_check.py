"""spatten_paged_append_check: the append's refusals without the append (CPU)."""
import pytest

from spatten_b200 import _native as N
from tests.test_paged_host import BAD_CACHE, _append


@pytest.mark.parametrize("cache,kw", [({f: v}, {}) for f, v, _ in BAD_CACHE if f != "max_pages"] + [({}, kw) for kw in (
    dict(dtype=N.DTYPE_F32), dict(k=0), dict(v=(1 << 20) + 8), dict(q_st=1020), dict(q_out=0), dict(q_norm_w=1 << 20),
    dict(sin=0), dict(cs_rows=0), dict(T=-1), dict(B=70000), dict(cu_tokens=0),
    dict(k_norm_w=1 << 20, q_norm_w=1 << 20, eps=-1.0))])
def test_the_appends_own_answer(cache, kw):
    code = N.lib.spatten_paged_append(_append(cache=cache.items(), **kw), None)
    err = N.lib.spatten_last_error()
    assert code in (N.ERR_INVALID, N.ERR_UNSUPPORTED)
    assert N.lib.spatten_paged_append_check(_append(cache=cache.items(), **kw)) == code
    assert N.lib.spatten_last_error() == err


def test_good_arguments_pass():
    assert N.lib.spatten_paged_append_check(_append()) == N.OK
    assert N.lib.spatten_paged_append_check(_append(T=0)) == N.OK
    assert N.lib.spatten_paged_append_check(None) == N.ERR_INVALID
