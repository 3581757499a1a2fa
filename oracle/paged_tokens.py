"""Oracle: trees of drafted tokens and eviction over the paged 8-bit KV cache
(CPU, torch float64), beside ``oracle/paged.py``.

Test infrastructure only (see ``oracle/__init__.py``): restates
``spatten_paged_tree``, ``spatten_paged_attend_ext``, ``spatten_paged_evict`` and
``spatten_paged_keep`` in plain loops, in 64 bits from the stored codes.
"""
import torch

from .paged import code_values, dense, round_codes, scale_for


def tree(parents, cu, lens, max_tokens):
    """(sees: list of sets per row, positions) of each row that is laid out."""
    sees, pos = {}, {}
    for b in range(len(lens)):
        n = cu[b + 1] - cu[b]
        for i in range(min(n, max_tokens)):
            a = parents[cu[b] + i]
            up = cu[b] + a if 0 <= a < i else None
            sees[cu[b] + i] = (sees[up] if up is not None else frozenset()) | {i}
            pos[cu[b] + i] = lens[b] - n + len(sees[cu[b] + i]) - 1
    return sees, pos


def words(sees, T, W):
    """Bits of ``sees`` as int32 [T, W] (rows that it lacks: zeros)."""
    out = torch.zeros(T, W, dtype=torch.int64)
    for t, s in sees.items():
        for j in s:
            out[t, j // 32] |= 1 << (j % 32)
    return torch.where(out >= 1 << 31, out - (1 << 32), out).to(torch.int32)


def attend(q, cache, table, cu, lens, sm_scale, sees=None, max_tokens=None):
    """As ``oracle.paged.attend`` with a tree's masks (None: causal), and the
    weights: (out, A, S, weight [B][G, len], err [B][G, len]); err is the sum
    over rows of p S, which the error bound of a weight is made of."""
    T, H, D = q.shape
    G = cache[0].shape[1]
    R = H // G
    out = torch.zeros(T, H, D, dtype=torch.float64)
    A = torch.zeros_like(out)
    S = torch.zeros(T, H, 1, dtype=torch.float64)
    weight, err = [], []
    for b in range(len(lens)):
        n = cu[b + 1] - cu[b]
        L = max(lens[b], 0)
        weight.append(torch.zeros(G, L, dtype=torch.float64))
        err.append(torch.zeros(G, L, dtype=torch.float64))
        if n == 0:
            continue
        K, V, has = dense(cache, table, b, L)
        old = lens[b] - n
        slot = torch.arange(L)
        for i in range(n if max_tokens is None else min(n, max_tokens)):
            t = cu[b] + i
            if sees is None:
                seen = slot < old + i + 1
            else:
                seen = slot < old
                for j in sees.get(t, ()):  # (tokens behind max_tokens are not the call's)
                    if j < (n if max_tokens is None else min(n, max_tokens)) and 0 <= old + j < L:
                        seen[old + j] = True
            seen = seen & has
            if not seen.any():
                continue
            qs = q[t].double().view(G, R, D)
            z = torch.einsum("grd,gnd->grn", qs, K) * sm_scale
            za = torch.einsum("grd,gnd->grn", qs.abs(), K.abs()) * abs(sm_scale)
            p = torch.zeros_like(z)
            p[..., seen] = torch.softmax(z[..., seen], -1)
            out[t] = torch.einsum("grn,gnd->grd", p, V).reshape(H, D)
            A[t] = torch.einsum("grn,gnd->grd", p, V.abs()).reshape(H, D)
            S[t] = za[..., seen].amax(-1).reshape(H, 1)
            weight[b] += p.sum(1)
            err[b] += (p * S[t].view(G, R, 1)).sum(1)
    return out, A, S, weight, err


def select(weight, position, keep, recent):
    """Moves [(to, from)] of one choice: weight (float32, as ranked), position: lists over the slots."""
    L = len(weight)
    if L <= keep:
        return []
    w = [float(x) if x > 0 else 0.0 for x in weight]  # (NaN > 0 is false)
    newest = max(position)
    order = sorted(range(L), key=lambda s: (not position[s] > newest - recent, -w[s], s))
    kept = set(order[:keep])
    return list(zip([s for s in range(keep) if s not in kept], [s for s in range(keep, L) if s in kept]))


def move(cache, table, moves, new_lens):
    """moves[b][g]: (to, from) pairs. Returns (codes, scales, ys) as
    ``oracle.paged.append``: the pools after the moves in float64, and for every
    code its value before rounding, in code units."""
    kv = cache[0].dtype
    page = cache[0].shape[2]
    codes = [code_values(cache[t]).clone() for t in range(2)]
    scales = [cache[2 + t].double().clone() for t in range(2)]
    ys = [c.clone() for c in codes]
    was = [c.clone() for c in codes], [s.clone() for s in scales]
    for b, heads in enumerate(moves):
        for g, pairs in enumerate(heads):
            for blk in sorted({to // page for to, _ in pairs}):
                here = [(to % page, fr) for to, fr in pairs if to // page == blk]
                pid = int(table[b, blk])
                gone = {r for r, _ in here}
                stay = [r for r in range(page) if blk * page + r < new_lens[b] and r not in gone]
                for t in range(2):
                    rows = {}
                    for r, fr in here:
                        ps = int(table[b, fr // page])
                        rows[r] = (was[0][t][ps, g, fr % page], float(was[1][t][ps, g]))
                    amax = max(float(c.abs().max()) * s for c, s in rows.values())
                    s_old = float(was[1][t][pid, g]) if stay else 0.0
                    s = max(s_old, scale_for(amax, kv))
                    if s > s_old:
                        for r in stay:
                            ys[t][pid, g, r] = was[0][t][pid, g, r] * (s_old / s)
                    for r, (c, sc) in rows.items():
                        ys[t][pid, g, r] = c * (sc / s) if s > 0 else c * 0
                    for r in list(rows) + (stay if s > s_old else []):
                        codes[t][pid, g, r] = round_codes(ys[t][pid, g, r], kv)
                    scales[t][pid, g] = s
    return codes, scales, ys


def move_beside(pool, table, moves):
    """The same moves of a pool [P, G, page]."""
    out, page = pool.clone(), pool.shape[2]
    for b, heads in enumerate(moves):
        for g, pairs in enumerate(heads):
            for to, fr in pairs:
                out[int(table[b, to // page]), g, to % page] = pool[int(table[b, fr // page]), g, fr % page]
    return out


def evict(cache, weight, position, table, lens, keep, recent=0, per_head=False):
    """(moves[b][g], new_lens)."""
    P, G, page, _ = cache[0].shape
    moves, new = [], []
    for b, L in enumerate(lens):
        pages = [int(table[b, s // page]) if s // page < table.shape[1] else -1 for s in range(0, max(L, 0), page)]
        if L <= keep or not all(0 <= p < P for p in pages):
            moves.append([[]] * G)
            new.append(L)
            continue
        w = weight[pages].transpose(0, 1).reshape(G, -1)[:, :L]
        p = position[pages].transpose(0, 1).reshape(G, -1)[:, :L]
        if per_head:
            moves.append([select(w[g].tolist(), p[g].tolist(), keep, recent) for g in range(G)])
        else:
            moves.append([select(w.double().sum(0).float().tolist(), p[0].tolist(), keep, recent)] * G)
        new.append(keep)
    return moves, new


def keep(cache, table, cu, lens, accepted):
    """(moves[b][g], new_lens)."""
    P, G, page, _ = cache[0].shape
    moves, new = [], []
    for b, L in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if n <= 0:
            moves.append([[]] * G)
            new.append(L)
            continue
        old, path, last = L - n, [], -1
        for a in accepted[b]:
            s = old + a
            if not last < a < n or s < 0 or s // page >= table.shape[1] or not 0 <= int(table[b, s // page]) < P:
                break
            path.append(a)
            last = a
        # (where a token moves to no page, it is gone)
        moves.append([[(old + j, old + a) for j, a in enumerate(path)
                       if j != a and old + j >= 0 and 0 <= int(table[b, (old + j) // page]) < P]] * G)
        new.append(max(old + len(path), 0))
    return moves, new
