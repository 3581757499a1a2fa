"""A paged KV cache held in 8 bits, on the C-ABI kernels (``spatten_paged_*`` in
include/spatten_b200.h): the cache that a model appends to and attends over
while it generates.

K and V are codes (int8 or e4m3) in pages of ``page_size`` tokens with one
fp32 scale per page and KV head; a value is code * scale. Sequence b's slot s
is row ``s % page_size`` of page ``page_table[b, s // page_size]`` (int32; an
entry outside the pool has no memory: nothing is stored there, and its slots
are no keys; an expanded table, one row for all sequences, can be read). The new tokens of a batch are packed: sequence b brings rows
``cu_tokens[b] .. cu_tokens[b+1]-1`` and holds ``seq_lens[b]`` tokens in all,
these included, which are its last ones. ``max_tokens`` bounds the tokens of
one sequence; the index tensors stay on the device, so a captured call can be
replayed with other lengths, pages and contents.

* ``new_paged_cache(num_pages, kv_heads, head_dim, ...)`` -> ``PagedKVCache``
* ``paged_append`` -- K (RMS-normed and rotated on request) and V into the
  cache, the query rows normed and rotated beside them;
* ``paged_attention`` -- causal attention of the new tokens over the cache:
  one token per sequence, a few drafted ones, or a piece of a prompt;
* ``paged_read`` -- cached tokens back in 16 bits: the ones that a cascade
  keeps (``topk_indices``), or whole sequences.

Rows behind ``cu_tokens[-1]`` (a padded batch) are neither read nor written.
"""
import math
from collections import namedtuple

import torch

from . import _native as N

_DT = {torch.float16: N.DTYPE_F16, torch.bfloat16: N.DTYPE_BF16}
_KV = {torch.int8: N.KV_INT8, torch.float8_e4m3fn: N.KV_E4M3}


class PagedKVCache(namedtuple("PagedKVCache", "k v k_scale v_scale")):
    """The pool: k, v codes [P, G, page, D], k_scale, v_scale fp32 [P, G], all
    contiguous. Its checks and the C form of it are made once, at its first
    use (the tensors of a tuple do not change)."""

    def __reduce__(self):  # copies and pickles make their own C form
        return PagedKVCache, tuple(self)

    @property
    def native(self):
        """(device index, shape of the pool, C form without a page table)."""
        try:
            return self._native
        except AttributeError:
            pass
        k, v, ks, vs = self
        dev, dt, shape = k.get_device(), k.dtype, k.shape
        if dev < 0:
            raise ValueError("paged cache: CUDA tensors expected (no CPU path)")
        if dt not in _KV or v.dtype != dt:
            raise TypeError(f"paged cache: codes {dt} and {v.dtype} (need int8 or float8_e4m3fn)")
        if len(shape) != 4 or v.shape != shape or ks.shape != shape[:2] or vs.shape != shape[:2] or \
                ks.dtype != torch.float32 or vs.dtype != torch.float32:
            raise ValueError("paged cache: need k, v [P, G, page, D] and fp32 scales [P, G]")
        if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
            raise ValueError("paged cache: contiguous tensors expected")
        if not v.get_device() == ks.get_device() == vs.get_device() == dev:
            raise ValueError("paged cache: tensors on several devices")
        P, G, page, D = shape
        self._native = dev, (P, G, page, D), N.PagedCache(_KV[dt], P, page, G, D, k.data_ptr(), v.data_ptr(),
                                                          ks.data_ptr(), vs.data_ptr())
        return self._native


def new_paged_cache(num_pages, kv_heads, head_dim, page_size=64, kv_dtype=torch.int8, device="cuda"):
    """An empty pool of ``num_pages`` pages. A page's contents and scale start
    with the first token that is appended to its first slot."""
    if kv_dtype not in _KV:
        raise TypeError(f"kv_dtype {kv_dtype} (need int8 or float8_e4m3fn)")
    shape = (num_pages, kv_heads, page_size, head_dim)
    k, v = (torch.zeros(shape, dtype=torch.int8, device=device).view(kv_dtype) for _ in range(2))
    ks, vs = (torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in range(2))
    return PagedKVCache(k, v, ks, vs)


def _index(t, name, dev, dim, dtype=torch.int32):
    """Pointer of an index tensor; its checks."""
    if t.get_device() != dev:
        raise ValueError(f"{name}: on {t.device}, the cache is on cuda:{dev}")
    if t.dtype != dtype or t.dim() != dim:
        raise ValueError(f"{name}: {t.dtype} of {t.dim()} dimensions (need {dtype} of {dim})")
    if t.stride()[-1] != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name}: last dimension must be contiguous")
    return t.data_ptr()


def _fill(a, cache, page_table, seq_lens):
    """The cache and the sequences into ``a``; returns (device index, the
    pool's shape)."""
    dev, shape, a.cache = cache.native
    B = seq_lens.shape[0]
    rows, cols = page_table.shape
    if rows != B:
        raise ValueError(f"page_table: {rows} rows for {B} sequences")
    c = a.cache
    c.page_table, c.max_pages = _index(page_table, "page_table", dev, 2), cols
    c.table_stride = page_table.stride()[0] if B > 1 else cols
    a.B, a.seq_lens = B, _index(seq_lens, "seq_lens", dev, 1)
    return dev, shape


def _fill_tokens(a, dev, cu_tokens, T, max_tokens):
    a.cu_tokens = _index(cu_tokens, "cu_tokens", dev, 1)
    if cu_tokens.shape[0] != a.B + 1:
        raise ValueError(f"cu_tokens: {cu_tokens.shape[0]} entries for {a.B} sequences")
    a.T, a.max_tokens = T, int(max_tokens)


def _rows(x, name, dev, dt, shape):
    """Pointer and (token, head) strides of a [T, heads, D] tensor."""
    if x.get_device() != dev:
        raise ValueError(f"{name}: on {x.device}, the cache is on cuda:{dev}")
    if x.dtype != dt:
        raise TypeError(f"{name}: dtype {x.dtype} (need {dt})")
    if x.shape != shape:
        raise ValueError(f"{name}: shape {tuple(x.shape)} (need {shape})")
    st, sh, sd = x.stride()
    if sd != 1 and shape[0]:
        raise ValueError(f"{name}: last dimension must be contiguous")
    return x.data_ptr(), st if shape[0] > 1 else 0, sh if shape[1] > 1 else 0


def _call(fn, dev, *args):
    """``fn`` on the current stream of device ``dev`` (the library works on
    the current device)."""
    if dev == torch._C._cuda_getDevice():
        return N.check(fn(*args, torch._C._cuda_getCurrentRawStream(dev)))
    with torch.cuda.device(dev):
        return N.check(fn(*args, torch._C._cuda_getCurrentRawStream(dev)))


def paged_append(cache, k, v, page_table, cu_tokens, seq_lens, max_tokens, q=None, cos=None, sin=None,
                 positions=None, q_norm_w=None, k_norm_w=None, eps=1e-6, q_out=None):
    """Append k, v [T, G, D] (fp16 / bf16, any token and head strides that are
    multiples of 8) to the cache; returns q [T, H, D] normed and rotated the
    same way (``q_out``, which may be ``q``; None without ``q``).

    ``q_norm_w`` / ``k_norm_w`` [D]: RMS norm weights (QK-norm). ``cos`` /
    ``sin`` [rows, >= D/2], fp32 or the rows' dtype: rotation of the halves of
    a row by row ``positions[t]`` (int32 [T]; default: the token's slot) of
    the tables, clamped to them. The arithmetic is fp32, rounded once. A page's
    scale only grows; where it does, its earlier codes are rounded again.
    Two sequences must not append into the same page in one call."""
    a = N.PagedAppendArgs()
    dev, (_, G, _, D) = _fill(a, cache, page_table, seq_lens)
    dt, T = k.dtype, k.shape[0]
    if dt not in _DT:
        raise TypeError(f"k: dtype {dt} (need float16 or bfloat16)")
    a.dtype = _DT[dt]
    _fill_tokens(a, dev, cu_tokens, T, max_tokens)
    a.k, a.k_st, a.k_sh = _rows(k, "k", dev, dt, (T, G, D))
    a.v, a.v_st, a.v_sh = _rows(v, "v", dev, dt, (T, G, D))
    if q is not None:
        shape = (T, q.shape[1], D)
        a.H = shape[1]
        a.q, a.q_st, a.q_sh = _rows(q, "q", dev, dt, shape)
        if q_out is None:
            q_out = q.new_empty(shape)
        a.q_out, a.qo_st, a.qo_sh = _rows(q_out, "q_out", dev, dt, shape)
    elif q_out is not None or q_norm_w is not None:
        raise ValueError("q_out / q_norm_w without q")
    for w, name in ((q_norm_w, "q_norm_w"), (k_norm_w, "k_norm_w")):
        if w is not None and (w.dtype != dt or w.get_device() != dev or w.shape != (D,) or not w.is_contiguous()):
            raise ValueError(f"{name}: need a contiguous {dt} [{D}] on cuda:{dev}")
    if k_norm_w is not None:
        a.k_norm_w, a.eps = k_norm_w.data_ptr(), float(eps)
    if q_norm_w is not None:
        a.q_norm_w = q_norm_w.data_ptr()
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    if cos is not None:
        shape, st = cos.shape, cos.stride()
        if sin.shape != shape or sin.stride() != st or sin.dtype != cos.dtype or len(shape) != 2 or \
                shape[1] < D // 2 or st[1] != 1 or cos.get_device() != dev or sin.get_device() != dev:
            raise ValueError(f"cos / sin: need two alike [rows, >= {D // 2}] tables on cuda:{dev}")
        if cos.dtype not in (torch.float32, dt):
            raise TypeError(f"cos / sin: dtype {cos.dtype} (need float32 or {dt})")
        a.cos, a.sin = cos.data_ptr(), sin.data_ptr()
        a.cs_dtype = N.DTYPE_F32 if cos.dtype == torch.float32 else _DT[dt]
        a.cs_rows, a.cs_stride = shape[0], st[0] if shape[0] > 1 else shape[1] // 8 * 8
        if positions is not None:
            a.positions = _index(positions, "positions", dev, 1)
            if positions.shape[0] != T:
                raise ValueError(f"positions: {positions.shape[0]} for {T} rows")
    elif positions is not None:
        raise ValueError("positions without cos / sin")
    _call(N.lib.spatten_paged_append, dev, a)
    return q_out


def paged_attention(q, cache, page_table, cu_tokens, seq_lens, max_tokens, sm_scale=None, out=None):
    """Causal attention of the new tokens' queries q [T, H, D] over the cache
    -> [T, H, D]: query i of sequence b sees slots ``n < seq_lens[b] - n_b + i
    + 1`` (its own among them, appended before); 0 where it sees none. GQA as
    in HF's ``repeat_kv``. ``out`` rows behind the last sequence keep what they
    held."""
    a = N.PagedAttendArgs()
    dev, (_, _, _, D) = _fill(a, cache, page_table, seq_lens)
    shape, dt = (q.shape[0], q.shape[1], D), q.dtype
    if dt not in _DT:
        raise TypeError(f"q: dtype {dt} (need float16 or bfloat16)")
    a.dtype, a.H = _DT[dt], shape[1]
    _fill_tokens(a, dev, cu_tokens, shape[0], max_tokens)
    a.q, a.q_st, a.q_sh = _rows(q, "q", dev, dt, shape)
    if out is None:
        out = q.new_empty(shape)
    a.out, a.o_st, a.o_sh = _rows(out, "out", dev, dt, shape)
    a.sm_scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    n = N.lib.spatten_paged_attend_workspace_size(a)
    ws = q.new_empty((n,), dtype=torch.uint8) if n else None
    _call(N.lib.spatten_paged_attend, dev, a, ws.data_ptr() if n else None, n)
    return out


def paged_read(cache, page_table, seq_lens, idx=None, n_tokens=None, dtype=torch.bfloat16):
    """Cached tokens back as (k, v) [B, n, G, D] of ``dtype``: slots idx [B, n]
    (int64; e.g. the kept tokens of ``topk_indices``) or, without it, the
    first ``n_tokens`` slots (default: what the page table spans). Zeros where
    a slot is outside the sequence."""
    a = N.PagedReadArgs()
    dev, (_, G, page, D) = _fill(a, cache, page_table, seq_lens)
    if dtype not in _DT:
        raise TypeError(f"dtype {dtype} (need float16 or bfloat16)")
    B = a.B
    a.dtype = _DT[dtype]
    if idx is not None:
        a.idx = _index(idx, "idx", dev, 2, torch.int64)
        rows, n = idx.shape
        if rows != B:
            raise ValueError(f"idx: {rows} rows for {B} sequences")
        a.N, a.idx_stride = n, idx.stride()[0]
    else:
        n = a.N = page_table.shape[1] * page if n_tokens is None else int(n_tokens)
    k, v = (cache.k.new_empty((B, max(n, 0), G, D), dtype=dtype) for _ in range(2))
    a.k_out, a.v_out = k.data_ptr(), v.data_ptr()
    _call(N.lib.spatten_paged_read, dev, a)
    return k, v


__all__ = ["PagedKVCache", "new_paged_cache", "paged_append", "paged_attention", "paged_read"]
