"""The path's operators registered with the PyTorch dispatcher (``torch.ops.spatten``).

Thin ``torch.library`` custom ops over the same C-ABI calls as the Python API
(no second implementation): code that addresses ops by name -- graph
capture, ``torch.ops.spatten.<op>`` in TorchScript-free pipelines, operator
registries -- finds them under the ``spatten`` namespace:

* ``spatten::quant_q_int8(Tensor x) -> (Tensor q8, Tensor scale)``
* ``spatten::quant_k_planes(Tensor k) -> (Tensor msb, Tensor lsb, Tensor scale)``
* ``spatten::progressive_attention(Tensor q, Tensor k, Tensor v, float refetch_threshold,
  float v_prune_threshold, float sm_scale, bool causal)
  -> (Tensor out, Tensor token_importance, Tensor head_abs_sum, Tensor refetch)``
* ``spatten::topk_select(Tensor x, int k) -> Tensor`` (sorted indices of the k largest per row)
* ``spatten::gather_rows(Tensor src, Tensor idx) -> Tensor``
* ``spatten::paged_append(Tensor(a!) k_pool, Tensor(b!) v_pool, Tensor(c!) k_scale, Tensor(d!) v_scale,
  Tensor k, Tensor v, Tensor page_table, Tensor cu_tokens, Tensor seq_lens, int max_tokens) -> ()``
  (no queries, norm or rotation: those are arguments of ``paged.paged_append``)
* ``spatten::paged_attention(Tensor q, Tensor k_pool, Tensor v_pool, Tensor k_scale, Tensor v_scale,
  Tensor page_table, Tensor cu_tokens, Tensor seq_lens, int max_tokens, float sm_scale) -> Tensor``
* ``spatten::paged_read(Tensor k_pool, Tensor v_pool, Tensor k_scale, Tensor v_scale, Tensor page_table,
  Tensor seq_lens, Tensor idx) -> (Tensor k, Tensor v)`` (bf16)
* ``spatten::paged_tree(Tensor parents, Tensor cu_tokens, Tensor seq_lens, int max_tokens)
  -> (Tensor tree, Tensor positions)``
* ``spatten::paged_tree_attention(Tensor q, Tensor k_pool, Tensor v_pool, Tensor k_scale, Tensor v_scale,
  Tensor page_table, Tensor cu_tokens, Tensor seq_lens, Tensor tree, int max_tokens, float sm_scale) -> Tensor``
* ``spatten::paged_weighing_attention(Tensor q, Tensor k_pool, Tensor v_pool, Tensor k_scale, Tensor v_scale,
  Tensor(a!) weight, Tensor(b!) position, Tensor page_table, Tensor cu_tokens, Tensor seq_lens, Tensor positions,
  int max_tokens, float sm_scale, Tensor? tree=None) -> Tensor`` (attention that accumulates its weights; causal, or
  under a tree's bits)
* ``spatten::paged_evict(Tensor(a!) k_pool, Tensor(b!) v_pool, Tensor(c!) k_scale, Tensor(d!) v_scale,
  Tensor(e!) weight, Tensor(f!) position, Tensor page_table, Tensor seq_lens, int keep, int recent, bool per_head)
  -> Tensor`` (new lengths)
* ``spatten::paged_keep(Tensor(a!) k_pool, Tensor(b!) v_pool, Tensor(c!) k_scale, Tensor(d!) v_scale,
  Tensor page_table, Tensor cu_tokens, Tensor seq_lens, Tensor accepted) -> Tensor`` (new lengths; for a cache
  without accumulated weights)
* ``spatten::paged_keep_weighed(Tensor(a!) k_pool, Tensor(b!) v_pool, Tensor(c!) k_scale, Tensor(d!) v_scale,
  Tensor(e!) weight, Tensor(f!) position, Tensor page_table, Tensor cu_tokens, Tensor seq_lens, Tensor accepted)
  -> Tensor`` (the same with the tokens' weights and positions moving along)

CUDA tensors only, like the rest of the package. Importing this module
registers the ops once.
"""
from typing import Optional

import torch

from . import paged as _pd
from . import progressive as _pg
from . import select as _sel


@torch.library.custom_op("spatten::quant_q_int8", mutates_args=())
def quant_q_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    q8, s = _pg.quant_q_int8(x)
    return q8, s


@torch.library.custom_op("spatten::quant_k_planes", mutates_args=())
def quant_k_planes(k: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    kp = _pg.quant_k_planes(k)
    return kp.msb, kp.lsb, kp.scale


@torch.library.custom_op("spatten::progressive_attention", mutates_args=())
def progressive_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, refetch_threshold: float,
                          v_prune_threshold: float, sm_scale: float, causal: bool
                          ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    r = _pg.progressive_attention(q, k, v, refetch_threshold=refetch_threshold,
                                  v_prune_threshold=v_prune_threshold, sm_scale=sm_scale,
                                  causal=causal, return_importance=True)
    return r.out, r.token_importance, r.head_abs_sum, r.refetch


@torch.library.custom_op("spatten::topk_select", mutates_args=())
def topk_select(x: torch.Tensor, k: int) -> torch.Tensor:
    return _sel.topk_indices(x, k)


@torch.library.custom_op("spatten::gather_rows", mutates_args=())
def gather_rows(src: torch.Tensor, idx: torch.Tensor) -> torch.Tensor:
    return _sel.gather_rows(src, idx)


@torch.library.custom_op("spatten::paged_append", mutates_args=("k_pool", "v_pool", "k_scale", "v_scale"))
def paged_append(k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                 k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, cu_tokens: torch.Tensor,
                 seq_lens: torch.Tensor, max_tokens: int) -> None:
    _pd.paged_append(_pd.PagedKVCache(k_pool, v_pool, k_scale, v_scale), k, v, page_table, cu_tokens, seq_lens,
                     max_tokens)


@torch.library.custom_op("spatten::paged_attention", mutates_args=())
def paged_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor,
                    v_scale: torch.Tensor, page_table: torch.Tensor, cu_tokens: torch.Tensor,
                    seq_lens: torch.Tensor, max_tokens: int, sm_scale: float) -> torch.Tensor:
    return _pd.paged_attention(q, _pd.PagedKVCache(k_pool, v_pool, k_scale, v_scale), page_table, cu_tokens,
                               seq_lens, max_tokens, sm_scale=sm_scale)


@torch.library.custom_op("spatten::paged_read", mutates_args=())
def paged_read(k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
               page_table: torch.Tensor, seq_lens: torch.Tensor, idx: torch.Tensor
               ) -> tuple[torch.Tensor, torch.Tensor]:
    return _pd.paged_read(_pd.PagedKVCache(k_pool, v_pool, k_scale, v_scale), page_table, seq_lens, idx=idx)


@torch.library.custom_op("spatten::paged_tree", mutates_args=())
def paged_tree(parents: torch.Tensor, cu_tokens: torch.Tensor, seq_lens: torch.Tensor, max_tokens: int
               ) -> tuple[torch.Tensor, torch.Tensor]:
    return _pd.paged_tree(parents, cu_tokens, seq_lens, max_tokens)


@torch.library.custom_op("spatten::paged_tree_attention", mutates_args=())
def paged_tree_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor,
                         v_scale: torch.Tensor, page_table: torch.Tensor, cu_tokens: torch.Tensor,
                         seq_lens: torch.Tensor, tree: torch.Tensor, max_tokens: int, sm_scale: float) -> torch.Tensor:
    return _pd.paged_attention(q, _pd.PagedKVCache(k_pool, v_pool, k_scale, v_scale), page_table, cu_tokens,
                               seq_lens, max_tokens, sm_scale=sm_scale, tree=tree)


@torch.library.custom_op("spatten::paged_weighing_attention", mutates_args=("weight", "position"))
def paged_weighing_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor,
                             v_scale: torch.Tensor, weight: torch.Tensor, position: torch.Tensor,
                             page_table: torch.Tensor, cu_tokens: torch.Tensor, seq_lens: torch.Tensor,
                             positions: torch.Tensor, max_tokens: int, sm_scale: float,
                             tree: Optional[torch.Tensor] = None) -> torch.Tensor:
    return _pd.paged_attention(q, _pd.PagedKVCache(k_pool, v_pool, k_scale, v_scale), page_table, cu_tokens,
                               seq_lens, max_tokens, sm_scale=sm_scale, tree=tree,
                               weights=_pd.PagedWeights(weight, position), positions=positions)


_POOL = ("k_pool", "v_pool", "k_scale", "v_scale")


@torch.library.custom_op("spatten::paged_evict", mutates_args=_POOL + ("weight", "position"))
def paged_evict(k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                weight: torch.Tensor, position: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                keep: int, recent: int, per_head: bool) -> torch.Tensor:
    return _pd.paged_evict(_pd.PagedKVCache(k_pool, v_pool, k_scale, v_scale), _pd.PagedWeights(weight, position),
                           page_table, seq_lens, keep, recent=recent, per_head=per_head)


@torch.library.custom_op("spatten::paged_keep", mutates_args=_POOL)
def paged_keep(k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
               page_table: torch.Tensor, cu_tokens: torch.Tensor, seq_lens: torch.Tensor, accepted: torch.Tensor
               ) -> torch.Tensor:
    return _pd.paged_keep(_pd.PagedKVCache(k_pool, v_pool, k_scale, v_scale), page_table, cu_tokens, seq_lens, accepted)


@torch.library.custom_op("spatten::paged_keep_weighed", mutates_args=_POOL + ("weight", "position"))
def paged_keep_weighed(k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                       weight: torch.Tensor, position: torch.Tensor, page_table: torch.Tensor, cu_tokens: torch.Tensor,
                       seq_lens: torch.Tensor, accepted: torch.Tensor) -> torch.Tensor:
    return _pd.paged_keep(_pd.PagedKVCache(k_pool, v_pool, k_scale, v_scale), page_table, cu_tokens, seq_lens, accepted,
                          weights=_pd.PagedWeights(weight, position))
