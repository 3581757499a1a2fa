"""Drop-in SpAtten cascade for Hugging Face Qwen3 prefill, on the C-ABI kernels.

``SpattenQwen3Attention(config, layer_idx)`` subclasses HF ``Qwen3Attention``
(installed ``transformers/models/qwen3/modeling_qwen3.py``: the projections
are the HF module's own; for fp16 / bf16 its per-head RMSNorm QK-norm and
RoPE run as one kernel, ``qk_norm_rope``, with the HF arithmetic and the
query's int8 quantisation; fp32 keeps the HF modules) and replaces its
attention core with the progressive sparse attention kernel:

* GQA: Q heads share KV heads as in HF's ``repeat_kv`` (head h reads KV head
  h // (H / Hkv)); the kernel indexes the shared KV head, nothing is repeated.
* Cascade token pruning applied to the KV cache: every layer attends over the
  keys kept so far (all keys at layer 0), adds its token importance -- the sum
  over heads and queries of the pruned probabilities, as in SpAtten's BERT
  cascade (spatten_bert.py:136-150) -- to the kept keys' cumulative score and
  keeps ``max(1, ceil(token_keep_ratio * K))`` of them (radix-select top-k,
  ties to the smaller position) for the next layer. Queries are never pruned:
  every position's hidden state goes through every layer.
* Causality over a pruned key set: the kept keys stay sorted by position, so
  query position m sees the prefix of keys whose position is <= m
  (``key_limit``); CTAs skip key tiles none of their rows sees.
* The KV cache (``past_key_values``, e.g. HF ``DynamicCache``) of layer i holds
  the keys and values layer i attended over, post-RoPE, in HF's
  [B, Hkv, K_i, D] layout; ``kept_positions`` gives their positions.
* Knobs: ``enable_token_prune`` with ``token_keep_ratio`` (or
  ``token_prune_num``), ``enable_v_prune`` with ``v_prune_threshold`` or the
  count ``v_prune_num`` (<= 16), ``enable_prog_quant`` with ``quant_threshold``
  (the row max-probability below which the LSB plane of K is refetched).

* Generation: with a ``PagedQwen3Cache`` as ``past_key_values`` the prefill's
  keys and values of every layer go into a paged 8-bit cache (``paged.py``), and
  later forwards (a token, a few, or the next piece of a prompt) append to it and
  attend over it: QK-norm, RoPE and the append in one launch, the attention in
  two. A layer that pruned its keys keeps attending over the ones it kept. With
  ``keep_tokens`` the cascade goes on while it generates: a full layer forgets
  the tokens of the least accumulated attention. Trees of drafted tokens are
  checked in one forward (``draft_tree``, ``accept`` or ``drop_tree``).

Unpadded batches only (the HF attention mask is not read: the mask is the
causal one). The cascade state is shared by all layers of a model
(``patch_qwen3``) and restarts at layer 0 of every prefill.
"""
import math
from fractions import Fraction

import torch
from transformers.cache_utils import Cache
from transformers.models.qwen3.modeling_qwen3 import Qwen3Attention, apply_rotary_pos_emb

from . import _native as N
from . import paged
from .progressive import prog_attn, quant_k_planes, quant_q_int8
from .select import gather_rows, topk_indices


def keep_count(ratio, current):
    """``max(1, ceil(ratio * current))``, exact on the ratio's decimal repr."""
    return max(1, math.ceil(Fraction(repr(float(ratio))) * current))


_DT = {torch.float16: N.DTYPE_F16, torch.bfloat16: N.DTYPE_BF16}


def qk_norm_rope(q, k, q_norm, k_norm, cos, sin, Hq, Hk, D, quantize_q):
    """QK-norm + RoPE of the projections in one kernel (spatten_qk_norm_rope):
    q [B, S, Hq*D], k [B, S, Hk*D] (fp16 / bf16, rows contiguous), the HF
    Qwen3RMSNorm modules ``q_norm`` / ``k_norm``, cos / sin [B, S, D].
    Returns (q [B, S, Hq, D] or None, q8 [B, Hq, S, D] or None, q_scale
    [B, Hq, S] or None, k [B, S, Hk, D]); q8 / q_scale when ``quantize_q``,
    q otherwise."""
    B, S, _ = q.shape
    if q.stride(2) != 1 or q.stride(0) != S * q.stride(1):
        q = q.contiguous()
    if k.stride(2) != 1 or k.stride(0) != S * k.stride(1):
        k = k.contiguous()
    if cos.stride(-1) != 1 or sin.stride() != cos.stride():
        cos, sin = cos.contiguous(), sin.contiguous()
    wq, wk = q_norm.weight.contiguous(), k_norm.weight.contiguous()
    dev, dt = q.device, q.dtype
    a = N.QkNormRopeArgs()
    a.dtype = _DT[dt]
    a.B, a.S, a.Hq, a.Hk, a.D = B, S, Hq, Hk, D
    a.q, a.q_row_stride = q.data_ptr(), q.stride(1)
    a.k, a.k_row_stride = k.data_ptr(), k.stride(1)
    a.q_norm_w, a.k_norm_w = wq.data_ptr(), wk.data_ptr()
    if float(k_norm.variance_epsilon) != float(q_norm.variance_epsilon):
        raise ValueError("qk_norm_rope: q_norm and k_norm must share their epsilon")
    a.eps = float(q_norm.variance_epsilon)
    a.cos, a.sin = cos.data_ptr(), sin.data_ptr()
    a.cs_b_stride = cos.stride(0) if cos.shape[0] == B else 0
    a.cs_s_stride = cos.stride(1)
    k_out = torch.empty((B, S, Hk, D), dtype=dt, device=dev)
    a.k_out, a.k_out_row_stride = k_out.data_ptr(), Hk * D
    q_out = q8 = qs = None
    if quantize_q:
        q8 = torch.empty((B, Hq, S, D), dtype=torch.int8, device=dev)
        qs = torch.empty((B, Hq, S), dtype=torch.float32, device=dev)
        a.q8, a.q_scale = q8.data_ptr(), qs.data_ptr()
    else:
        q_out = torch.empty((B, S, Hq, D), dtype=dt, device=dev)
        a.q_out, a.q_out_row_stride = q_out.data_ptr(), Hq * D
    N.check(N.lib.spatten_qk_norm_rope(a, torch.cuda.current_stream(dev).cuda_stream))
    return q_out, q8, qs, k_out


class PagedQwen3Cache(Cache):
    """Paged 8-bit KV cache of every layer, for ``past_key_values`` of a model
    that ``patch_qwen3`` made. ``max_tokens`` slots per sequence are reserved in
    each layer's pool, sequence b's pages in a row; the layers share one page
    table. Layers may hold different numbers of tokens (token pruning).

    ``keep_tokens``: the layers keep account of the attention weight that each
    token gathers, and one that has no room for the next tokens keeps the
    ``recent_tokens`` newest and of the others those of the largest weight,
    ``keep_tokens`` in all (``paged_evict``), and goes on; so a text may be longer
    than ``max_tokens``. ``None``: a full cache refuses.

    HF's generation modes that change a cache are served: drafted tokens
    (``crop``), beams (``reorder_cache``), and changes of the batch
    (``batch_repeat_interleave``, ``batch_select_indices``)."""

    # tokens of a forward that accounts can be taken back for: drafts are fewer, and more are
    # a piece of the text (64 tokens of 32 x 128 are 0.5 MB a layer and sequence)
    drafted = 64

    def __init__(self, config, batch, max_tokens, page_size=64, kv_dtype=torch.int8, device="cuda", keep_tokens=None,
                 recent_tokens=0):
        super().__init__(layers=[])
        L, G, D = config.num_hidden_layers, config.num_key_value_heads, config.head_dim
        self.batch, self.max_tokens = batch, int(max_tokens)
        self.keep_tokens, self.recent_tokens = keep_tokens, int(recent_tokens)
        if keep_tokens is not None and not 1 <= keep_tokens < self.max_tokens:
            raise ValueError(f"PagedQwen3Cache: keep_tokens {keep_tokens} of {self.max_tokens}")
        if not 0 <= self.recent_tokens <= (keep_tokens or 0):
            raise ValueError(f"PagedQwen3Cache: {recent_tokens} recent tokens among {keep_tokens}")
        mp = -(-self.max_tokens // page_size)
        self.pools = [paged.new_paged_cache(batch * mp, G, D, page_size, kv_dtype, device) for _ in range(L)]
        self.weights = [paged.new_paged_weights(p) for p in self.pools] if keep_tokens is not None else [None] * L
        self.asked = [None] * L  # queries [B, n, H, D] of the last n tokens of a layer's last forward, and their scale
        self.tree = None  # (bits, parents, tokens per sequence, positions before) of drafted tokens
        self.page_table = self._pages(batch, mp, device)
        self.seq_lens = torch.zeros((L, batch), dtype=torch.int32, device=device)
        self.held = [0] * L  # slots of each layer, as the host counts them
        self.seen = [0] * L  # positions each layer has been given (kept or not)
        self.pruned = [0] * L  # positions of which each layer kept only some (0: all kept)

    @staticmethod
    def _pages(batch, per_sequence, device):
        return torch.arange(batch * per_sequence, dtype=torch.int32, device=device).view(batch, per_sequence)

    @property
    def max_batch_size(self):
        return self.batch

    @property
    def max_cache_len(self):
        return self.max_tokens

    def get_seq_length(self, layer_idx=0):
        return self.seen[layer_idx]

    def get_mask_sizes(self, query_length, layer_idx=0):
        return self.seen[layer_idx or 0] + int(query_length), 0

    def get_max_cache_shape(self, layer_idx=0):
        return self.max_tokens

    def reset(self):
        """Forget every token; the pools stay."""
        self.tree = None
        self.seq_lens.zero_()
        L = len(self.pools)
        self.asked = [None] * L
        self.held, self.seen, self.pruned = [0] * L, [0] * L, [0] * L

    def crop(self, max_length):
        """Forget the positions from ``max_length`` on (negative: that many of
        the last ones), in every layer; their slots are written again by the next
        tokens. Positions of which a layer kept only some (a pruned prompt, or what
        there was at an eviction) can only be forgotten as a whole: which it kept is
        not known here. With ``keep_tokens`` the attention weight that the forgotten ones
        gave the others goes too, up to its rounding, for as many as were among the last
        ``drafted`` (64) tokens of the last forward; that of earlier ones stays."""
        self._no_tree("crop")
        keep = int(max_length)
        if keep < 0:
            keep = max(self.seen[0] + keep, 0)
        drop = [max(n - keep, 0) for n in self.seen]
        if not any(drop):
            return
        if keep == 0:
            return self.reset()
        for n, d, fixed in zip(self.seen, drop, self.pruned):
            if d and n - d < fixed:
                raise NotImplementedError(f"PagedQwen3Cache: crop to {keep} inside {fixed} pruned tokens")
        for i, d in enumerate(drop):
            if d:
                self._take_back(i, d)
        if len(set(drop)) == 1:
            self.seq_lens.sub_(drop[0])
        else:  # layers that were given different numbers of tokens
            for lens, d in zip(self.seq_lens, drop):
                lens.sub_(d)
        self.held = [n - d for n, d in zip(self.held, drop)]
        self.seen = [n - d for n, d in zip(self.seen, drop)]

    def _rows_of(self, idx):
        rows = torch.arange(self.batch)[idx.cpu()].tolist() if idx.dtype == torch.bool else idx.tolist()
        if not rows or not all(0 <= r < self.batch for r in rows):
            raise ValueError(f"PagedQwen3Cache: sequences {rows} of {self.batch}")
        return rows

    def _by_sequence(self, t, pages=None):
        """A pool's tensor as [batch, pages, ..] of each sequence's first pages
        (codes as int8: copies need no more)."""
        t = t.view(torch.int8) if t.dtype.itemsize == 1 else t
        return t.view(self.batch, -1, *t.shape[1:])[:, :pages]

    def reorder_cache(self, beam_idx):
        """Sequence b becomes a copy of sequence beam_idx[b], on pages of its own
        (the next tokens of two beams differ)."""
        self._no_tree("reorder_cache")
        rows = self._rows_of(beam_idx)
        if len(rows) != self.batch:
            raise ValueError(f"PagedQwen3Cache: {len(rows)} beams for {self.batch} sequences")
        moved = [b for b, r in enumerate(rows) if r != b]
        if not moved:
            return
        dev = self.seq_lens.device
        dst, src = torch.tensor([moved, [rows[b] for b in moved]], device=dev)
        for pool, w, held in zip(self.pools, self.weights, self.held):
            for t in (*pool, *(w or ())):
                t = self._by_sequence(t, -(-held // pool.k.shape[2]))
                t.index_copy_(0, dst, t.index_select(0, src))
        self.seq_lens.index_copy_(1, dst, self.seq_lens.index_select(1, src))
        self._ask_for(torch.tensor(rows, device=dev))

    def _ask_for(self, idx):
        """The noted queries of sequences idx."""
        self.asked = [a and (a[0].index_select(0, idx), a[1]) for a in self.asked]

    def _select(self, rows):
        """Sequence b of a new batch is a copy of sequence rows[b]."""
        self._no_tree("a change of the batch")
        idx = torch.tensor(rows, device=self.seq_lens.device)

        def select(t):
            return self._by_sequence(t).index_select(0, idx).flatten(0, 1).view(t.dtype)
        self.pools = [paged.PagedKVCache(*map(select, pool)) for pool in self.pools]
        self.weights = [w and paged.PagedWeights(*map(select, w)) for w in self.weights]
        self.seq_lens = self.seq_lens.index_select(1, idx)
        self._ask_for(idx)
        self.batch = len(rows)
        self.page_table = self._pages(self.batch, self.page_table.shape[1], idx.device)

    def batch_repeat_interleave(self, repeats):
        """``repeats`` copies of each sequence, beside one another."""
        if repeats < 1:
            raise ValueError(f"PagedQwen3Cache: {repeats} copies")
        self._select([b for b in range(self.batch) for _ in range(repeats)])

    def batch_select_indices(self, indices):
        """The sequences ``indices`` (numbers or a mask) alone."""
        self._select(self._rows_of(indices))

    def packed(self, S):
        """cu_tokens of a batch that brings S tokens per sequence."""
        return torch.arange(0, (self.batch + 1) * S, S, dtype=torch.int32, device=self.seq_lens.device)

    def append(self, layer_idx, n, seen, cu, k, v, **kw):
        """``paged_append`` of n tokens per sequence (rows k, v, packed by cu =
        ``packed(n)``) to one layer, counted as ``seen`` more positions; nothing
        counts when the call is refused."""
        before = self.held[layer_idx]
        if before + n > self.max_tokens:
            if self.keep_tokens is None or self.keep_tokens + n > self.max_tokens or before <= self.keep_tokens:
                raise ValueError(f"PagedQwen3Cache: {before} + {n} tokens, room for {self.max_tokens}")
            if self.seq_lens.is_cuda:  # (elsewhere the eviction itself refuses)
                paged._check_append(self.pools[layer_idx], k, v, self.page_table, cu, self.seq_lens[layer_idx], n, **kw)
            before = self._evict(layer_idx)
        held = before + n
        lens = self.seq_lens[layer_idx]
        lens.add_(n)
        try:
            q = paged.paged_append(self.pools[layer_idx], k, v, self.page_table, cu, lens, n, **kw)
        except Exception:
            lens.sub_(n)
            raise
        self.held[layer_idx] = held
        self.asked[layer_idx] = None
        self.seen[layer_idx] += seen
        if n < seen:
            self.pruned[layer_idx] = self.seen[layer_idx]
        return q

    def _evict(self, layer_idx):
        """Cut a layer to ``keep_tokens``; returns the slots it holds."""
        lens = self.seq_lens[layer_idx]
        lens.copy_(paged.paged_evict(self.pools[layer_idx], self.weights[layer_idx], self.page_table, lens,
                                     self.keep_tokens, recent=self.recent_tokens))
        self.held[layer_idx] = self.keep_tokens
        self.pruned[layer_idx] = self.seen[layer_idx]
        return self.keep_tokens

    def note(self, layer_idx, q, sm_scale):
        """The queries [B, S, H, D] that a forward asked a layer with. Those of a drafted tree count
        once it is known which of them stay (``accept``), others until they are cropped."""
        if self.keep_tokens is not None:
            if self.tree is None and q.shape[1] > self.drafted:
                q = q[:, -self.drafted:].clone()
            self.asked[layer_idx] = q, sm_scale

    def _account(self, layer_idx, q, sm_scale, weights, positions=None):
        """Adds what the queries [B, n, H, D] of a layer's last n tokens give its cached ones to ``weights``."""
        B, n, H, D = q.shape
        if q.is_cuda:
            q.record_stream(torch.cuda.current_stream(q.device))
        paged._attend(q.reshape(B * n, H, D), self.pools[layer_idx], self.page_table, self.packed(n),
                      self.seq_lens[layer_idx], n, sm_scale=sm_scale, weights=weights, positions=positions)

    def _take_back(self, layer_idx, n):
        """Before a layer's last n tokens leave: what they gave the others leaves with them."""
        if self.asked[layer_idx] is None:
            return
        q, sm_scale = self.asked[layer_idx]
        stay = max(q.shape[1] - n, 0)
        gone = paged.new_paged_weights(self.pools[layer_idx])
        self._account(layer_idx, q[:, stay:], sm_scale, gone)
        self.weights[layer_idx].weight.sub_(gone.weight)  # (of the slots that are let go: anything)
        self.asked[layer_idx] = (q[:, :stay], sm_scale) if stay else None

    def positions(self, layer_idx, S):
        """Positions int32 [batch * S] of the next S tokens of each sequence."""
        first = self.seen[layer_idx]
        return torch.arange(first, first + S, dtype=torch.int32, device=self.seq_lens.device).repeat(self.batch)

    def store(self, layer_idx, k, v, seen, importance=None, positions=None):
        """Append finished (normed and rotated) keys and values [B, K, G, D];
        ``seen``: the positions that they were chosen from. With ``keep_tokens``
        their attention weights (fp32 [B, K], spread over the KV heads; default
        0) and positions ([B, K]; default: the next ones) start as given."""
        B, K, G, D = k.shape
        if B != self.batch:
            raise ValueError(f"PagedQwen3Cache: batch {B}, made for {self.batch}")
        if positions is None and self.keep_tokens is not None:
            positions = self.positions(layer_idx, K).view(B, K)
        self.append(layer_idx, K, seen, self.packed(K), k.reshape(B * K, G, D), v.reshape(B * K, G, D))
        if self.keep_tokens is not None:
            page = self.pools[layer_idx].k.shape[2]
            slot = torch.arange(self.held[layer_idx] - K, self.held[layer_idx], device=k.device)
            weight, position = (self._by_sequence(t) for t in self.weights[layer_idx])  # [B, pages, G, page]
            weight[:, slot // page, :, slot % page] = 0.0 if importance is None else (importance.t() / G)[..., None]
            position[:, slot // page, :, slot % page] = positions.t().to(torch.int32)[..., None]

    def _no_tree(self, what):
        if self.tree is not None:
            raise RuntimeError(f"PagedQwen3Cache: {what} before the drafted tree's tokens were accepted (accept) or given up "
                               "(drop_tree)")

    def draft_tree(self, parents):
        """The next forward's tokens [B, S] are a tree (or several): ``parents``
        [B, S] holds the place of each one's parent among them, before its own, or
        -1 for a child of the text so far. Returns their positions, int64 [B, S],
        for the model's ``position_ids``; ``accept`` has to follow that forward, or
        ``drop_tree``."""
        self._no_tree("another tree")
        B, S = parents.shape
        if B != self.batch or S < 1:
            raise ValueError(f"PagedQwen3Cache: parents of {B} sequences x {S} tokens, made for {self.batch}")
        if len(set(self.seen)) > 1 or self.seen[0] == 0:
            raise ValueError("PagedQwen3Cache: a drafted tree follows a prompt")
        dev = self.seq_lens.device
        lens = torch.full((B,), self.seen[0] + S, dtype=torch.int32, device=dev)
        parents = parents.to(dev, torch.int32, copy=True)
        bits, positions = paged.paged_tree(parents.reshape(-1), self.packed(S), lens, S)
        self.tree = bits, parents, S, self.seen[0]
        return positions.view(B, S).long()

    def accept(self, paths):
        """Of the drafted tree's tokens the ones at ``paths`` (per sequence their
        places, ascending, equally many for each) stay, in every layer: a branch from the
        text on, each of them one position behind the one before it. With
        ``keep_tokens`` the accepted ones' attention weights are added here, as if the
        text had been given without a draft: the rejected ones' never count."""
        if self.tree is None or any(n != self.tree[3] + self.tree[2] for n in self.seen):
            raise RuntimeError("PagedQwen3Cache: no forward of a drafted tree")
        S = self.tree[2]
        paths = [[int(i) for i in p] for p in paths]
        if len(paths) != self.batch or len(set(map(len, paths))) != 1:
            raise ValueError(f"PagedQwen3Cache: need as many accepted tokens for each of {self.batch} sequences")
        if any(p != sorted(set(p)) or (p and not 0 <= p[0] <= p[-1] < S) for p in paths):
            raise ValueError(f"PagedQwen3Cache: accepted places {paths} of {S} tokens (need them ascending)")
        for up, path in zip(self.tree[1].tolist(), paths):
            depth = []
            for i, a in enumerate(up):  # (as paged_tree: another value makes a child of the text)
                depth.append(depth[a] + 1 if 0 <= a < i else 0)
            if [depth[i] for i in path] != list(range(len(path))):
                raise ValueError(f"PagedQwen3Cache: accepted places {path} are {[depth[i] for i in path]} positions behind "
                                 "the text (need a branch: 0, 1, ..)")
        accepted = torch.tensor(paths, dtype=torch.int32, device=self.seq_lens.device).view(self.batch, -1)
        gone, cu = S - accepted.shape[1], self.packed(S)
        for pool, lens in zip(self.pools, self.seq_lens):  # (the new tokens have no weights yet)
            lens.copy_(paged.paged_keep(pool, self.page_table, cu, lens, accepted))
        self.held = [n - gone for n in self.held]
        before, self.tree = self.tree[3], None
        for i, asked in enumerate(self.asked):
            self.seen[i] = before
            if asked is not None and S > gone:
                q = asked[0][torch.arange(self.batch, device=accepted.device)[:, None], accepted.long()]
                self._account(i, q, asked[1], self.weights[i], self.positions(i, S - gone))
                self.note(i, q, asked[1])
            else:
                self.asked[i] = None
            self.seen[i] = before + S - gone

    def drop_tree(self):
        """Give a drafted tree up, if there is one: before its forward, after it, or where that
        failed on the way. Its tokens leave the layers that they had come to."""
        if self.tree is None:
            return
        before, self.tree = self.tree[3], None
        for i, n in enumerate(self.seen):
            if n > before:
                self.seq_lens[i].sub_(n - before)
                self.held[i] -= n - before
                self.seen[i], self.asked[i] = before, None

    def update(self, key_states, value_states, layer_idx, *args, **kwargs):
        """HF's form of ``store`` ([B, G, K, D]); only a prefill's first call may
        use it, as attention modules that read a dense cache expect all keys
        back."""
        if self.held[layer_idx]:
            raise NotImplementedError("PagedQwen3Cache: read by SpattenQwen3Attention only")
        self.store(layer_idx, key_states.transpose(1, 2), value_states.transpose(1, 2), key_states.shape[2])
        return key_states, value_states


class CascadeState:
    """Kept key positions [B, K] (int64, ascending) and their cumulative
    token importance [B, K] (fp32), handed from layer to layer."""

    def __init__(self):
        self.positions = None
        self.cumulative = None
        self.kept_per_layer = []


class SpattenQwen3Attention(Qwen3Attention):
    """HF Qwen3Attention with the SpAtten cascade, on the B200 kernels."""

    def __init__(self, config, layer_idx):
        super().__init__(config, layer_idx)
        self.num_heads = config.num_attention_heads
        self.num_kv_heads = config.num_key_value_heads
        self.enable_token_prune = False
        self.token_keep_ratio = None
        self.token_prune_num = 0
        self.enable_v_prune = False
        self.v_prune_threshold = None
        self.v_prune_num = 2
        self.enable_prog_quant = False
        self.quant_threshold = 0.1
        self.cascade = CascadeState()
        # diagnostics of the last forward
        self.kept_positions = None      # [B, K] positions this layer attended over
        self.token_importance = None    # [B, K] cumulative importance after this layer
        self.last_refetch = None

    def _v_prune(self, K):
        v_thr, v_count = 0.0, 0
        if self.enable_v_prune:
            if self.v_prune_threshold is not None:
                v_thr = float(self.v_prune_threshold)
            elif self.v_prune_num > 0 and K > self.v_prune_num:
                v_count = int(self.v_prune_num)
                if v_count > N.MAX_V_PRUNE_COUNT:
                    raise NotImplementedError(
                        f"v_prune_num={v_count}: at most {N.MAX_V_PRUNE_COUNT} keys per row by count")
        return v_thr, v_count

    def _extend(self, hidden_states, position_embeddings, cache):
        """Forward of further tokens over a ``PagedQwen3Cache`` that holds some."""
        B, S, _ = hidden_states.shape
        H, Hkv, d = self.num_heads, self.num_kv_heads, self.head_dim
        dt = hidden_states.dtype
        if dt not in _DT or d not in (64, 128):
            raise NotImplementedError(f"PagedQwen3Cache: {dt}, head dim {d} (need fp16 / bf16, 64 or 128)")
        if B != cache.batch:
            raise ValueError(f"PagedQwen3Cache: batch {B}, made for {cache.batch}")
        if float(self.k_norm.variance_epsilon) != float(self.q_norm.variance_epsilon):
            raise ValueError("q_norm and k_norm must share their epsilon")
        q = self.q_proj(hidden_states).view(B * S, H, d)
        k = self.k_proj(hidden_states).view(B * S, Hkv, d)
        v = self.v_proj(hidden_states).view(B * S, Hkv, d)
        cos, sin = position_embeddings  # [B or 1, S, d]: a row per token
        rows = torch.arange(cos.shape[0] * S, dtype=torch.int32, device=q.device)
        positions = rows if cos.shape[0] == B else rows.repeat(B)
        cu, more = cache.packed(S), {}
        if cache.tree is not None:
            more["tree"], _, drafted, before = cache.tree
            if S != drafted or cache.seen[self.layer_idx] != before:
                raise RuntimeError(f"PagedQwen3Cache: {S} tokens after a drafted tree of {drafted} that was not accepted")
        elif cache.keep_tokens is not None:
            more["weights"], more["positions"] = cache.weights[self.layer_idx], cache.positions(self.layer_idx, S)
        q = cache.append(self.layer_idx, S, S, cu, k, v, q=q, cos=cos.reshape(-1, d), sin=sin.reshape(-1, d),
                         positions=positions, q_norm_w=self.q_norm.weight, k_norm_w=self.k_norm.weight,
                         eps=self.q_norm.variance_epsilon)
        out = paged.paged_attention(q, cache.pools[self.layer_idx], cache.page_table, cu,
                                    cache.seq_lens[self.layer_idx], S, sm_scale=self.scaling, **more)
        cache.note(self.layer_idx, q.view(B, S, H, d), self.scaling)
        return self.o_proj(out.view(B, S, H * d)), None

    @torch.no_grad()
    def forward(self, hidden_states, position_embeddings, attention_mask=None, past_key_values=None,
                **kwargs):
        if not hidden_states.is_cuda:
            raise ValueError("SpattenQwen3Attention runs on the CUDA kernels only")
        B, S, _ = hidden_states.shape
        if past_key_values is not None and past_key_values.get_seq_length(self.layer_idx) > 0:
            if isinstance(past_key_values, PagedQwen3Cache):
                return self._extend(hidden_states, position_embeddings, past_key_values)
            raise NotImplementedError("SpattenQwen3Attention: prefill only (the cache already holds keys); "
                                      "a PagedQwen3Cache can be extended")
        H, Hkv, d = self.num_heads, self.num_kv_heads, self.head_dim
        dev = hidden_states.device
        cos, sin = position_embeddings
        q8 = qs = None
        if hidden_states.dtype in _DT and d in (64, 128):
            # QK-norm + RoPE (+ the query's int8) in one kernel: the HF
            # arithmetic without its dozen elementwise launches
            q, q8, qs, k = qk_norm_rope(self.q_proj(hidden_states), self.k_proj(hidden_states), self.q_norm,
                                        self.k_norm, cos, sin, H, Hkv, d, self.enable_prog_quant)
        else:
            q = self.q_norm(self.q_proj(hidden_states).view(B, S, H, d))
            k = self.k_norm(self.k_proj(hidden_states).view(B, S, Hkv, d))
            q, k = apply_rotary_pos_emb(q, k, cos, sin, unsqueeze_dim=2)
        v = self.v_proj(hidden_states).view(B, S, Hkv, d)

        st = self.cascade
        if self.layer_idx == 0 or st.positions is None or st.positions.shape[0] != B:
            st.positions = torch.arange(S, device=dev).expand(B, S).contiguous()
            st.cumulative = None
            st.kept_per_layer = []
        pos = st.positions
        K = pos.shape[1]
        if K < S:  # the kept keys: a gather of rows [B, S, Hkv*d] -> [B, K, Hkv*d]
            k = gather_rows(k.reshape(B, S, Hkv * d), pos).view(B, K, Hkv, d)
            v = gather_rows(v.contiguous().view(B, S, Hkv * d), pos).view(B, K, Hkv, d)
        else:
            k = k.contiguous()
            v = v.contiguous()
        # query position m sees the kept keys at positions <= m
        qpos = torch.arange(S, device=dev).expand(B, S).contiguous()
        key_limit = torch.searchsorted(pos, qpos, right=True).to(torch.int32)

        out = torch.empty(B, S, H, d, dtype=hidden_states.dtype, device=dev)
        v_thr, v_count = self._v_prune(K)
        qh = q.permute(0, 2, 1, 3) if q is not None else None  # [B, H, S, d] views
        kh = k.permute(0, 2, 1, 3)   # [B, Hkv, K, d]
        vh = v.permute(0, 2, 1, 3)
        # a cache that keeps accounts is given this layer's own weights, whole: as a difference of the
        # cascade's fp32 sums over layers they would lose the bits that those have no room for
        own = isinstance(past_key_values, PagedQwen3Cache) and past_key_values.keep_tokens is not None
        common = dict(sm_scale=self.scaling, v_thr=v_thr, v_prune_count=v_count, key_limit=key_limit,
                      tok_in=None if own else st.cumulative, want_tok=True, out=out.permute(0, 2, 1, 3))
        if self.enable_prog_quant:
            if q8 is None:
                q8, qs = quant_q_int8(qh)
            kp = quant_k_planes(kh)
            r = prog_attn(q8, kp.msb, vh, k1=kp.lsb, mode=N.MODE_QUANT, q_scale=qs, k_scale=kp.scale,
                          refetch_thr=float(self.quant_threshold), want_refetch=True, **common)
            self.last_refetch = r.refetch
        else:
            r = prog_attn(qh, kh, vh, mode=N.MODE_DENSE, **common)
        importance = cum = r.token_importance
        if own and st.cumulative is not None:
            cum = st.cumulative + importance  # (the sum that the kernel would have made)
        self.kept_positions = pos
        self.token_importance = cum
        st.kept_per_layer.append(K)

        if isinstance(past_key_values, PagedQwen3Cache):
            past_key_values.store(self.layer_idx, k, v, S, positions=pos, importance=importance)
            if K == S and own:  # (else it cannot be cropped into)
                if q8 is not None:
                    last = slice(-past_key_values.drafted, None)
                    q = (q8[:, :, last] * qs[:, :, last, None]).transpose(1, 2).to(v.dtype)
                past_key_values.note(self.layer_idx, q, self.scaling)
        elif past_key_values is not None:
            # the cache concatenates into a new contiguous [B, Hkv, K, d] tensor
            # itself: the head-major views go in as they are (one copy, not two)
            past_key_values.update(kh, vh, self.layer_idx)

        if self.enable_token_prune:
            keep = keep_count(self.token_keep_ratio, K) if self.token_keep_ratio is not None \
                else max(1, K - int(self.token_prune_num))
            if keep < K:
                idx = topk_indices(cum, keep)
                st.positions = pos.gather(1, idx)
                st.cumulative = cum.gather(1, idx)
            else:
                st.positions, st.cumulative = pos, cum
        else:
            st.positions, st.cumulative = pos, cum
        return self.o_proj(out.view(B, S, H * d)), None


def patch_qwen3(model, **knobs):
    """Swap every decoder layer's self-attention for SpattenQwen3Attention
    (weights carried over with load_state_dict), share one cascade state
    across the layers, and set ``knobs`` on every layer. ``model`` is a HF
    Qwen3Model or Qwen3ForCausalLM."""
    base = model.model if hasattr(model, "model") else model
    state = CascadeState()
    for i, layer in enumerate(base.layers):
        old = layer.self_attn
        new = SpattenQwen3Attention(base.config, old.layer_idx)
        new.load_state_dict(old.state_dict())
        new.to(device=old.q_proj.weight.device, dtype=old.q_proj.weight.dtype)
        new.cascade = state
        for k, v in knobs.items():
            setattr(new, k, v)
        layer.self_attn = new
    return model
