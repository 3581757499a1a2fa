"""The paged KV cache's refusals: bad arguments end before any launch (CPU)."""
import pytest
import torch

from spatten_b200 import _native as N


def _cache(c, **kw):
    c.kv_type, c.num_pages, c.page_size, c.G, c.D = N.KV_INT8, 10, 64, 2, 128
    c.k = c.v = c.k_scale = c.v_scale = c.page_table = 1 << 20
    c.table_stride, c.max_pages = 4, 4
    for k, v in kw.items():
        setattr(c, k, v)


def _append(cache=(), **kw):
    a = N.PagedAppendArgs()
    _cache(a.cache, **dict(cache))
    a.dtype, a.B, a.H, a.T, a.max_tokens = N.DTYPE_BF16, 3, 8, 3, 1
    a.cu_tokens = a.seq_lens = a.q = a.k = a.v = a.q_out = a.cos = a.sin = 1 << 20
    a.q_st, a.q_sh, a.k_st, a.k_sh, a.v_st, a.v_sh, a.qo_st, a.qo_sh = 1024, 128, 256, 128, 256, 128, 1024, 128
    a.cs_dtype, a.cs_rows, a.cs_stride = N.DTYPE_F32, 100, 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _attend(cache=(), **kw):
    a = N.PagedAttendArgs()
    _cache(a.cache, **dict(cache))
    a.dtype, a.B, a.H, a.T, a.max_tokens, a.sm_scale = N.DTYPE_BF16, 3, 8, 3, 1, 0.1
    a.cu_tokens = a.seq_lens = a.q = a.out = 1 << 20
    a.q_st, a.q_sh, a.o_st, a.o_sh = 1024, 128, 1024, 128
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _read(cache=(), **kw):
    a = N.PagedReadArgs()
    _cache(a.cache, **dict(cache))
    a.dtype, a.B, a.N = N.DTYPE_BF16, 3, 5
    a.seq_lens = a.idx = a.k_out = a.v_out = 1 << 20
    a.idx_stride = 5
    for k, v in kw.items():
        setattr(a, k, v)
    return a


BAD_CACHE = [
    ("kv_type", 2, N.ERR_INVALID), ("num_pages", 0, N.ERR_INVALID), ("page_size", 48, N.ERR_UNSUPPORTED),
    ("page_size", 256, N.ERR_UNSUPPORTED), ("G", 0, N.ERR_INVALID), ("G", 5000, N.ERR_UNSUPPORTED),
    ("D", 96, N.ERR_UNSUPPORTED), ("k", 0, N.ERR_INVALID), ("v", (1 << 20) + 8, N.ERR_INVALID),
    ("k_scale", 0, N.ERR_INVALID), ("v_scale", (1 << 20) + 2, N.ERR_INVALID), ("page_table", 0, N.ERR_INVALID),
    ("table_stride", 3, N.ERR_INVALID), ("max_pages", 0, N.ERR_INVALID), ("max_pages", 1 << 26, N.ERR_UNSUPPORTED),
]


def _run(kind, a):
    if kind == "append":
        return N.lib.spatten_paged_append(a, None)
    if kind == "attend":
        return N.lib.spatten_paged_attend(a, None, 0, None)
    return N.lib.spatten_paged_read(a, None)


@pytest.mark.parametrize("kind", ["append", "attend", "read"])
@pytest.mark.parametrize("field,value,code", BAD_CACHE)
def test_bad_cache(kind, field, value, code):
    kw = {field: value}
    if field == "max_pages" and value > 4:
        kw["table_stride"] = value
    a = {"append": _append, "attend": _attend, "read": _read}[kind](cache=kw.items())
    assert _run(kind, a) == code
    assert N.lib.spatten_last_error().decode().startswith("paged_")


@pytest.mark.parametrize("field,value,code", [
    ("dtype", N.DTYPE_F32, N.ERR_UNSUPPORTED), ("B", -1, N.ERR_INVALID), ("B", 70000, N.ERR_UNSUPPORTED),
    ("T", -1, N.ERR_INVALID), ("max_tokens", -1, N.ERR_INVALID), ("cu_tokens", 0, N.ERR_INVALID),
    ("seq_lens", (1 << 20) + 2, N.ERR_INVALID), ("k", 0, N.ERR_INVALID), ("k", (1 << 20) + 8, N.ERR_INVALID),
    ("v_st", 260, N.ERR_INVALID), ("k_sh", -128, N.ERR_INVALID), ("q_out", 0, N.ERR_INVALID),
    ("q", 0, N.ERR_INVALID), ("H", 0, N.ERR_INVALID), ("q_norm_w", 1 << 20, N.ERR_INVALID),
    ("k_norm_w", 1 << 20, N.ERR_INVALID), ("cos", 0, N.ERR_INVALID), ("cs_dtype", N.DTYPE_F16, N.ERR_UNSUPPORTED),
    ("qo_st", 0, N.ERR_INVALID), ("qo_sh", 64, N.ERR_INVALID),
    ("cs_rows", 0, N.ERR_INVALID), ("cs_stride", 60, N.ERR_INVALID), ("positions", (1 << 20) + 1, N.ERR_INVALID),
])
def test_bad_append(field, value, code):
    assert N.lib.spatten_paged_append(_append(**{field: value}), None) == code


def test_bad_append_norm():
    a = _append(q_norm_w=1 << 20, k_norm_w=1 << 20, eps=-1.0)
    assert N.lib.spatten_paged_append(a, None) == N.ERR_INVALID
    a = _append(q_norm_w=1 << 20, k_norm_w=(1 << 20) + 8, eps=1e-6)
    assert N.lib.spatten_paged_append(a, None) == N.ERR_INVALID
    assert N.lib.spatten_paged_append(None, None) == N.ERR_INVALID


@pytest.mark.parametrize("field,value,code", [
    ("dtype", N.DTYPE_F32, N.ERR_UNSUPPORTED), ("H", 0, N.ERR_INVALID), ("H", 7, N.ERR_INVALID),
    ("H", 2 * 129, N.ERR_UNSUPPORTED), ("q", 0, N.ERR_INVALID), ("out", (1 << 20) + 8, N.ERR_INVALID),
    ("q_st", 1020, N.ERR_INVALID), ("o_sh", 4, N.ERR_INVALID), ("sm_scale", float("nan"), N.ERR_INVALID),
    ("cu_tokens", 0, N.ERR_INVALID), ("B", 70000, N.ERR_UNSUPPORTED), ("T", -2, N.ERR_INVALID),
    ("B", 8193, N.ERR_UNSUPPORTED), ("o_st", 0, N.ERR_INVALID), ("o_sh", 64, N.ERR_INVALID),
])
def test_bad_attend(field, value, code):
    assert N.lib.spatten_paged_attend(_attend(**{field: value}), None, 0, None) == code


@pytest.mark.parametrize("field,value,code", [
    ("dtype", N.DTYPE_F32, N.ERR_UNSUPPORTED), ("N", -1, N.ERR_INVALID), ("seq_lens", 0, N.ERR_INVALID),
    ("idx", (1 << 20) + 4, N.ERR_INVALID), ("idx_stride", -1, N.ERR_INVALID), ("k_out", (1 << 20) + 8, N.ERR_INVALID),
])
def test_bad_read(field, value, code):
    assert N.lib.spatten_paged_read(_read(**{field: value}), None) == code


def test_no_work_is_ok():
    """Empty batches and calls without new tokens touch nothing."""
    assert N.lib.spatten_paged_append(_append(B=0), None) == N.OK
    assert N.lib.spatten_paged_append(_append(T=0, k=0, v=0, q=0, q_out=0), None) == N.OK
    assert N.lib.spatten_paged_append(_append(max_tokens=0), None) == N.OK
    assert N.lib.spatten_paged_attend(_attend(T=0, q=0, out=0), None, 0, None) == N.OK
    assert N.lib.spatten_paged_attend(_attend(B=0), None, 0, None) == N.OK
    assert N.lib.spatten_paged_read(_read(B=0), None) == N.OK
    assert N.lib.spatten_paged_read(_read(N=0), None) == N.OK


def test_neither_output_of_read():
    assert N.lib.spatten_paged_read(_read(k_out=0, v_out=0), None) == N.ERR_INVALID


def test_python_refuses_cpu_tensors():
    from spatten_b200 import paged
    c = paged.new_paged_cache(4, 2, 64, page_size=16, device="cpu")
    i32 = dict(dtype=torch.int32)
    with pytest.raises(ValueError, match="no CPU path"):
        paged.paged_read(c, torch.zeros(1, 2, **i32), torch.zeros(1, **i32))
    with pytest.raises(TypeError):
        paged.new_paged_cache(4, 2, 64, kv_dtype=torch.float16, device="cpu")
