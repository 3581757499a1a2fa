"""Oracle: the paged 8-bit KV cache (CPU, torch float64).

Test infrastructure only (see ``oracle/__init__.py``). The reference has no
decoding, so this restatement defines ``spatten_paged_*``: plain loops over
sequences, pages and heads, in 64 bits from the stored codes and scales.
"""
import math

import torch


def code_values(codes):
    """Codes (int8 or e4m3) as float64."""
    return codes.double() if codes.dtype == torch.int8 else codes.float().double()


def scale_for(amax, kv_dtype):
    """Scale of a block whose largest finite magnitude is ``amax``."""
    if amax == 0:
        return 0.0
    if kv_dtype == torch.int8:
        return amax / 127
    m, e = math.frexp(amax / 448)  # m in [0.5, 1)
    return 2.0 ** max(e if m > 0.5 else e - 1, -126)


def in_range(y, kv_dtype):
    """y (in code units) saturated, NaN to 0."""
    top = 127 if kv_dtype == torch.int8 else 448
    return torch.nan_to_num(y, nan=0.0, posinf=top, neginf=-top).clamp(-top, top)


def round_codes(y, kv_dtype):
    """y (in range) rounded to codes; float64."""
    return y.round() if kv_dtype == torch.int8 else y.float().to(torch.float8_e4m3fn).double()


def turn(x, w, eps, cos, sin, pos):
    """RMS norm and rotation of one row [heads, D] in 64 bits."""
    x = x.double()
    if w is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    if cos is not None:
        h = x.shape[-1] // 2
        r = min(max(pos, 0), cos.shape[0] - 1)
        c, s = cos[r, :h].double(), sin[r, :h].double()
        x = torch.cat([x[..., :h] * c - x[..., h:] * s, x[..., h:] * c + x[..., :h] * s], -1)
    return x


def append(cache, k, v, table, cu, lens, q=None, cos=None, sin=None, positions=None, wq=None, wk=None, eps=1e-6):
    """Returns (q_out or None, codes, scales, y), all float64: codes, scales
    and y as [K's, V's], the pool after the call; y holds, for every code that
    the call rounded, its value before rounding in code units (a rounded
    evaluation may end at either neighbour of a border), else the code."""
    kv = cache[0].dtype
    out = [code_values(cache[0]).clone(), code_values(cache[1]).clone(), cache[2].double().clone(),
           cache[3].double().clone()]
    ys = [out[0].clone(), out[1].clone()]
    P, G, page, D = cache[0].shape
    qo = None if q is None else torch.zeros(q.shape, dtype=torch.float64)
    for b in range(len(lens)):
        n = cu[b + 1] - cu[b]
        old = lens[b] - n
        rows_k, rows_v = [], []
        for i in range(n):
            t = cu[b] + i
            pos = positions[t] if positions is not None else old + i
            if q is not None:
                qo[t] = turn(q[t], wq, eps, cos, sin, pos)
            rows_k.append(turn(k[t], wk, eps, cos, sin, pos))
            rows_v.append(v[t].double())
        for pi in range(max(old, 0) // page, -(-lens[b] // page)):
            if pi >= table.shape[1] or not 0 <= int(table[b, pi]) < P:
                continue
            pid, first = int(table[b, pi]), pi * page
            lo, hi = max(old - first, 0), min(lens[b] - first, page)
            if hi <= lo:
                continue
            for which, rows in ((0, rows_k), (1, rows_v)):
                x = torch.stack(rows[first + lo - old:first + hi - old], 1)  # [G, hi - lo, D]
                for g in range(G):
                    fin = x[g][torch.isfinite(x[g])]
                    s_old = float(out[2 + which][pid, g]) if lo > 0 else 0.0
                    s = max(s_old, scale_for(float(fin.abs().max()) if fin.numel() else 0.0, kv))
                    if s > s_old and lo > 0:
                        y = out[which][pid, g, :lo] * (s_old / s)
                        ys[which][pid, g, :lo] = y
                        out[which][pid, g, :lo] = round_codes(y, kv)
                    y = in_range(x[g] / s, kv) if s > 0 else torch.zeros_like(x[g])
                    ys[which][pid, g, lo:hi] = y
                    out[which][pid, g, lo:hi] = round_codes(y, kv)
                    out[2 + which][pid, g] = s
    return qo, out[:2], out[2:], ys


def dense(cache, table, b, n):
    """K, V [G, n, D] float64 of slots 0 .. n-1, and which of them have memory."""
    P, G, page, D = cache[0].shape
    kv = [torch.zeros(G, n, D, dtype=torch.float64) for _ in range(2)]
    has = torch.zeros(n, dtype=torch.bool)
    for s in range(n):
        if s // page >= table.shape[1]:
            break
        pid = int(table[b, s // page])
        if 0 <= pid < P:
            has[s] = True
            for t in range(2):
                kv[t][:, s] = code_values(cache[t][pid, :, s % page]) * cache[2 + t][pid].double()[:, None]
    return kv[0], kv[1], has


def attend(q, cache, table, cu, lens, sm_scale):
    """(out, A, S): the attention in float64; A = sum p |v| per output and S =
    the largest sm_scale * sum |q k| of a row's scores, which the error bounds
    of a rounded evaluation are made of."""
    T, H, D = q.shape
    G = cache[0].shape[1]
    out = torch.zeros(T, H, D, dtype=torch.float64)
    A = torch.zeros_like(out)
    S = torch.zeros(T, H, 1, dtype=torch.float64)
    for b in range(len(lens)):
        n = cu[b + 1] - cu[b]
        if n == 0:
            continue
        K, V, has = dense(cache, table, b, max(lens[b], 0))
        qs = q[cu[b]:cu[b + 1]].double().view(n, G, H // G, D)
        z = torch.einsum("igrd,gnd->igrn", qs, K) * sm_scale
        za = torch.einsum("igrd,gnd->igrn", qs.abs(), K.abs()) * sm_scale
        seen = has[None] & (torch.arange(K.shape[1])[None] < (lens[b] - n + 1 + torch.arange(n))[:, None])
        for i in range(n):
            if not seen[i].any():
                continue
            p = torch.softmax(z[i][..., seen[i]], -1)  # [G, R, keys]
            out[cu[b] + i] = torch.einsum("grn,gnd->grd", p, V[:, seen[i]]).reshape(H, D)
            A[cu[b] + i] = torch.einsum("grn,gnd->grd", p, V[:, seen[i]].abs()).reshape(H, D)
            S[cu[b] + i] = za[i][..., seen[i]].amax(-1).reshape(H, 1)
    return out, A, S
