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

Trees of drafted tokens, checked in one pass:

* ``paged_tree`` -- from the drafted tokens' parents the bits of the new tokens
  that each of them sees (for ``paged_attention``) and their positions (for
  ``paged_append``), once per step for all layers;
* ``paged_keep`` -- of the new tokens the accepted ones stay.

A cache of bounded length, the cascade's token pruning while a model generates:

* ``new_paged_weights(cache)`` -> ``PagedWeights``, in which ``paged_attention``
  accumulates the attention weight of every cached token;
* ``paged_evict`` -- the recent tokens and those of the largest weight stay.

Rows behind ``cu_tokens[-1]`` (a padded batch) are neither read nor written.
"""
import math
from collections import namedtuple

import torch

from . import _native as N

_DT = {torch.float16: N.DTYPE_F16, torch.bfloat16: N.DTYPE_BF16}
_KV = {torch.int8: N.KV_INT8, torch.float8_e4m3fn: N.KV_E4M3}
_INT_MAX = 2 ** 31 - 1


class PagedKVCache(namedtuple("PagedKVCache", "k v k_scale v_scale")):
    """The pool: k, v codes [P, G, page, D], k_scale, v_scale fp32 [P, G], all
    contiguous. Its checks and the C form of it are made once, at its first
    use (the tensors of a tuple do not change)."""

    def __reduce__(self):  # copies and pickles make their own C form
        return PagedKVCache, tuple(self)

    @property
    def native(self):
        """(device index, shape of the pool, C form without a page table)."""
        got = self.__dict__.get("_native")
        if got is not None:
            return got
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


class PagedWeights(namedtuple("PagedWeights", "weight position")):
    """Beside a pool: the attention weight that each cached token has gathered,
    fp32 [P, G, page], and its position, int32 [P, G, page]; contiguous."""


def new_paged_weights(cache):
    """No weight and position 0 everywhere; a slot's start with the first
    ``paged_attention`` call that has its token among the new ones."""
    shape, dev = cache.k.shape[:3], cache.k.device
    return PagedWeights(torch.zeros(shape, dtype=torch.float32, device=dev),
                        torch.zeros(shape, dtype=torch.int32, device=dev))


def _weights(a, weights, dev, shape):
    """The weights beside a pool of ``shape`` into ``a``; their checks."""
    w, p = weights
    if w.get_device() != dev or p.get_device() != dev:
        raise ValueError(f"weights.weight / position: on {w.device} and {p.device}, the cache is on cuda:{dev}")
    if w.dtype is not torch.float32 or w.shape != shape or not w.is_contiguous():
        raise ValueError(f"weights.weight: need a contiguous float32 {tuple(shape)}, got {w.dtype} {tuple(w.shape)}")
    if p.dtype is not torch.int32 or p.shape != shape or not p.is_contiguous():
        raise ValueError(f"weights.position: need a contiguous int32 {tuple(shape)}, got {p.dtype} {tuple(p.shape)}")
    a.weight, a.position = w.data_ptr(), p.data_ptr()


def _index(t, name, dev, dim, dtype=torch.int32):
    """Pointer of an index tensor; its checks."""
    if t.get_device() != dev:
        raise ValueError(f"{name}: on {t.device}, the cache is on cuda:{dev}")
    st = t.stride()
    if t.dtype is not dtype or len(st) != dim:
        raise ValueError(f"{name}: {t.dtype} of {t.dim()} dimensions (need {dtype} of {dim})")
    if st[-1] != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name}: last dimension must be contiguous")
    return t.data_ptr()


def _like(q, shape):
    """Uninitialised [T, heads, D] of q's type (its own shape, where it is contiguous, costs least)."""
    return torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)


def _scratch(n, t):
    """n bytes of workspace (a multiple of 256) beside an int32 tensor, and their address."""
    if not n:
        return None, None
    ws = t.new_empty((n // 4,))
    return ws, ws.data_ptr()


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
    dev, a, q_out = _append_args(cache, k, v, page_table, cu_tokens, seq_lens, max_tokens, q, cos, sin, positions,
                                 q_norm_w, k_norm_w, eps, q_out)
    _call(N.lib.spatten_paged_append, dev, a)
    return q_out


def _check_append(*args, **kw):
    """Raises what ``paged_append`` would with these arguments; does nothing else."""
    N.check(N.lib.spatten_paged_append_check(_append_args(*args, **kw)[1]))


def _append_args(cache, k, v, page_table, cu_tokens, seq_lens, max_tokens, q=None, cos=None, sin=None,
                 positions=None, q_norm_w=None, k_norm_w=None, eps=1e-6, q_out=None):
    """(device index, the call's arguments, q_out); their checks."""
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
    return dev, a, q_out


def paged_tree(parents, cu_tokens, seq_lens, max_tokens):
    """Bits and positions of trees of drafted tokens: ``parents`` int32 [T]
    holds, per new token, its parent's place among its sequence's new tokens
    (which comes before its own), or -1 for a child of the cached tokens.
    Returns (tree int32 [T, ceil(min(max_tokens, T) / 32)], positions int32 [T]): bit j
    of a row's words is set if it sees new token j (itself and its ancestors);
    its position is that of the sequence's first new token, ``seq_lens`` less
    the new tokens, plus its depth (after an eviction, which leaves the cache
    shorter than the text: pass the text's lengths). At most 1024 tokens per
    sequence."""
    dev = parents.get_device()
    if dev < 0:
        raise ValueError("paged_tree: CUDA tensors expected (no CPU path)")
    a = N.PagedTreeArgs()
    a.B, a.seq_lens = seq_lens.shape[0], _index(seq_lens, "seq_lens", dev, 1)
    a.parents = _index(parents, "parents", dev, 1)
    _fill_tokens(a, dev, cu_tokens, parents.shape[0], max_tokens)
    a.tree_words = a.tree_stride = max(-(-min(a.max_tokens, a.T) // 32), 1)
    tree, positions = parents.new_empty((a.T, a.tree_words)), parents.new_empty((a.T,))
    a.tree, a.positions = tree.data_ptr(), positions.data_ptr()
    _call(N.lib.spatten_paged_tree, dev, a)
    return tree, positions


def paged_attention(q, cache, page_table, cu_tokens, seq_lens, max_tokens, sm_scale=None, out=None, tree=None,
                    weights=None, positions=None):
    """Causal attention of the new tokens' queries q [T, H, D] over the cache
    -> [T, H, D]: query i of sequence b sees slots ``n < seq_lens[b] - n_b + i
    + 1`` (its own among them, appended before); 0 where it sees none. GQA as
    in HF's ``repeat_kv``. ``out`` rows behind the last sequence keep what they
    held.

    ``tree`` (int32 [T, >= max_tokens / 32], e.g. of ``paged_tree``): a query
    sees every slot before its sequence's new tokens, and of these the ones
    whose bits its row has. ``weights``: the softmax weight that the queries
    give each cached token, summed over the query heads of its KV head, is
    added to ``weights.weight`` (all rows count, also drafts that are rejected
    later); the new tokens' own start at 0, and their
    ``weights.position`` becomes ``positions`` (int32 [T]; default: the slot).
    Sequences must not share pages, nor claim the same rows, then."""
    return _attend(q, cache, page_table, cu_tokens, seq_lens, max_tokens, sm_scale, out, tree, weights, positions)


def _attend(q, cache, page_table, cu_tokens, seq_lens, max_tokens, sm_scale=None, out=None, tree=None, weights=None,
            positions=None):
    ext = N.PagedAttendExtArgs() if tree is not None or weights is not None else None
    a = N.PagedAttendArgs() if ext is None else ext.attend
    dev, (P, G, page, D) = _fill(a, cache, page_table, seq_lens)
    shape, dt = (q.shape[0], q.shape[1], D), q.dtype
    if dt not in _DT:
        raise TypeError(f"q: dtype {dt} (need float16 or bfloat16)")
    a.dtype, a.H = _DT[dt], shape[1]
    _fill_tokens(a, dev, cu_tokens, shape[0], max_tokens)
    a.q, a.q_st, a.q_sh = _rows(q, "q", dev, dt, shape)
    if out is None:
        out = _like(q, shape)
    a.out, a.o_st, a.o_sh = _rows(out, "out", dev, dt, shape)
    a.sm_scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    if tree is not None:
        ext.tree = _index(tree, "tree", dev, 2)
        if tree.shape[0] != shape[0]:
            raise ValueError(f"tree: {tree.shape[0]} rows for {shape[0]}")
        if 32 * tree.shape[1] < min(a.max_tokens, a.T):
            raise ValueError(f"tree: {tree.shape[1]} words of 32 tokens for {a.max_tokens}")
        ext.tree_words, ext.tree_stride = tree.shape[1], tree.stride()[0]
    if weights is not None:
        _weights(ext, weights, dev, (P, G, page))
    if positions is not None:
        if weights is None:
            raise ValueError("positions without weights")
        ext.positions = _index(positions, "positions", dev, 1)
        if positions.shape[0] != shape[0]:
            raise ValueError(f"positions: {positions.shape[0]} for {shape[0]} rows")
    if ext is None:
        size, call = N.lib.spatten_paged_attend_workspace_size, N.lib.spatten_paged_attend
    else:
        a, size, call = ext, N.lib.spatten_paged_attend_ext_workspace_size, N.lib.spatten_paged_attend_ext
    n = size(a)
    ws, at = _scratch(n, seq_lens)
    _call(call, dev, a, at, n)
    return out


def paged_evict(cache, weights, page_table, seq_lens, keep, recent=0, per_head=False):
    """Sequences of more than ``keep`` tokens keep that many: those of the
    ``recent`` newest positions, then those of the largest accumulated weight
    (``weights``, see ``paged_attention``), ties to the lower slot. One choice
    for all KV heads, by the sum of their weights (rounded to fp32), or with
    ``per_head`` each head's own (its slots then hold other tokens than the
    other heads'). Returns the sequences' new lengths, int32 [B].

    Kept tokens in the first ``keep`` slots stay; the others move, with their
    weights and positions, into the slots that became free, both in ascending
    order: from then on slots are not in order of position, so later
    ``paged_append`` and ``paged_attention`` calls need ``positions``. A moved
    token is rounded to the scale of its new page, which grows as in
    ``paged_append``. Sequences with slots that have no memory, or more slots
    than the pool, are left as they are; sequences must not share the pages that
    tokens move into."""
    a = N.PagedEvictArgs()
    dev, (P, G, page, _) = _fill(a, cache, page_table, seq_lens)
    _weights(a, weights, dev, (P, G, page))
    a.keep, a.recent, a.per_head = min(int(keep), _INT_MAX), min(int(recent), _INT_MAX), bool(per_head)
    new_lens = torch.empty_like(seq_lens, memory_format=torch.contiguous_format)
    a.new_lens = new_lens.data_ptr()
    n = N.lib.spatten_paged_evict_workspace_size(a)
    ws, at = _scratch(n, seq_lens)
    _call(N.lib.spatten_paged_evict, dev, a, at, n)
    return new_lens


def paged_keep(cache, page_table, cu_tokens, seq_lens, accepted, weights=None):
    """Of the new tokens the accepted ones stay: ``accepted`` int32 [B, A] lists
    their places among their sequence's new tokens in ascending order, -1 behind
    a short list (it ends at the first entry that is not above the one before
    it, or no new token). They move to the front of the new tokens' slots in
    that order, with their ``weights`` where given, rounded to the scales of
    the pages they come to. Returns the sequences' new lengths, int32 [B].
    Sequences must not share the pages of the new tokens."""
    a = N.PagedKeepArgs()
    dev, (P, G, page, _) = _fill(a, cache, page_table, seq_lens)
    a.cu_tokens = _index(cu_tokens, "cu_tokens", dev, 1)
    if cu_tokens.shape[0] != a.B + 1:
        raise ValueError(f"cu_tokens: {cu_tokens.shape[0]} entries for {a.B} sequences")
    a.accepted = _index(accepted, "accepted", dev, 2)
    rows, a.n_accepted = accepted.shape
    if rows != a.B:
        raise ValueError(f"accepted: {rows} rows for {a.B} sequences")
    a.accepted_stride = accepted.stride()[0]
    if weights is not None:
        _weights(a, weights, dev, (P, G, page))
    new_lens = torch.empty_like(seq_lens, memory_format=torch.contiguous_format)
    a.new_lens = new_lens.data_ptr()
    _call(N.lib.spatten_paged_keep, dev, a)
    return new_lens


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


__all__ = ["PagedKVCache", "PagedWeights", "new_paged_cache", "new_paged_weights", "paged_append", "paged_attention",
           "paged_evict", "paged_keep", "paged_read", "paged_tree"]
