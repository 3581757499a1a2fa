"""Cases of what a serving loop does with the paged 8-bit KV cache beside appending and attending: trees of
drafted tokens (their masks, attention under them, the accepted ones kept) and eviction by accumulated attention
weight (attention that accumulates it, and the eviction itself).

The cache is that of perf/operators.py: codes [pages, G, page, D] (int8 or e4m3) with one fp32 scale per page and
KV head, sequence b's slot s in row s % page of page table[b, s // page], packed new tokens. Beside it, where
weights are accumulated, the pools weight (fp32) and position (int32), [pages, G, page].

* tree: `parents` (per new token the place of its parent among its sequence's new tokens, -1 for a child of the
  cached ones) -> words of a bit mask (bit j of a token's words: it sees new token j) and positions.
* tree_attend: every new token sees the cached tokens and those new ones that its words name.
* weigh: causal (or tree) attention that adds to the weight of every cached token the softmax weights that the new
  tokens gave it, summed over their query heads; a new token's own slot starts at 0 and takes its position.
* evict: sequences of more than `keep` tokens keep those of the `recent` newest positions and then those of the
  largest weight (the sum over the heads rounded to 32 bits, or each head by itself; ties to the lower slot).
  Kept tokens in slots behind `keep` move into the free slots before it, both ascending.
* keep: of the new tokens the accepted ones stay (places, ascending), moved to the front of them.

A token that moves into another page is rounded to that page's scale, which grows where it has to, as in appending
(and starts over in a page that keeps nothing).
"""
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one user's drafted tree, masks and positions for all layers of a step: all latency
        dict(name="tree_b1", op="tree", B=1, new_lo=26, new_hi=26, width=3),
        # a serving batch's trees
        dict(name="tree_b64", op="tree", B=64, new_lo=20, new_hi=64, width=4),
        # one user's tree checked over a short context
        dict(name="tree_attend_b1", op="tree_attend", B=1, H=32, G=8, D=128, page=64, kv="int8", dt="bf16",
             len_lo=777, len_hi=777, new_lo=26, new_hi=26, width=3),
        # small trees of a ragged batch, 64-wide heads, small pages (few query rows per KV head)
        dict(name="tree_attend_b24_ragged", op="tree_attend", B=24, H=12, G=4, D=64, page=16, kv="e4m3", dt="fp16",
             len_lo=20, len_hi=4096, new_lo=3, new_hi=17, width=2),
        # large trees over long contexts
        dict(name="tree_attend_b16", op="tree_attend", B=16, H=32, G=8, D=128, page=64, kv="int8", dt="bf16",
             len_lo=4097, len_hi=8192, new_lo=33, new_hi=64, width=4),
        # one user's next token while its cache keeps account of the weights, all latency
        dict(name="weigh_step_b1", op="weigh", B=1, H=32, G=8, D=128, page=64, kv="int8", dt="bf16",
             len_lo=777, len_hi=777, new_lo=1, new_hi=1, width=0),
        # the decode benchmark's batch and cache length
        dict(name="weigh_step_b64_n32768", op="weigh", B=64, H=32, G=8, D=128, page=64, kv="int8", dt="bf16",
             len_lo=32768, len_hi=32768, new_lo=1, new_hi=1, width=0),
        # the next piece of long prompts, whose queries say which of the earlier tokens matter
        dict(name="weigh_prompt_piece_b2", op="weigh", B=2, H=16, G=8, D=128, page=64, kv="e4m3", dt="bf16",
             len_lo=6000, len_hi=8192, new_lo=700, new_hi=1024, width=0),
        # a long document's cache cut to half, one choice for all heads
        dict(name="evict_b1_long", op="evict", B=1, G=8, D=128, page=128, kv="e4m3", dt="bf16",
             len_lo=131001, len_hi=131001, keep=65536, recent=1000, per_head=False),
        # a serving batch whose caches are full, every KV head by its own weights
        dict(name="evict_heads_b48", op="evict", B=48, G=8, D=128, page=64, kv="int8", dt="bf16",
             len_lo=3000, len_hi=5000, keep=4096, recent=256, per_head=True),
        # one user's accepted branch
        dict(name="keep_b1", op="keep", B=1, G=8, D=128, page=64, kv="int8", dt="bf16", old_lo=1000, old_hi=1000,
             new_lo=26, new_hi=26, width=3, weights=False),
        # a serving batch's, with the weights moving along
        dict(name="keep_b64", op="keep", B=64, G=8, D=64, page=16, kv="e4m3", dt="fp16", old_lo=1, old_hi=2000,
             new_lo=20, new_hi=64, width=4, weights=True),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["tree", "tree_attend", "tree_attend", "weigh", "weigh", "weigh", "evict", "evict", "keep"])
    if op == "tree":
        hi = _log(rng, 1, 256)
        return dict(op=op, B=_log(rng, 1, 128), new_lo=rng.randint(1, hi), new_hi=hi, width=rng.randint(1, 6))
    c = dict(op=op, G=rng.choice([1, 2, 4, 8]), D=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]),
             kv=rng.choice(["int8", "e4m3"]), dt=rng.choice(["bf16", "fp16"]))
    if op in ("tree_attend", "weigh"):
        c["B"] = _log(rng, 1, 64)
        c["H"] = c["G"] * rng.choice([1, 2, 3, 4, 5, 8, 16])
        tree = op == "tree_attend" or rng.random() < 0.3
        c["width"] = rng.randint(1, 6) if tree else 0
        kind = rng.random()
        c["new_hi"] = _log(rng, 2, 200) if tree else 1 if kind < 0.5 else rng.randint(2, 8)
        if not tree and kind > 0.75:  # a piece of a prompt
            c["new_hi"] = _log(rng, 9, 1024)
            c["H"] = min(c["H"], 2 * c["G"])
        # a bounded number of scores, of keys, and of the rows' (padded) keys
        most = min(131072, (48 * 32768) // c["B"], (1 << 31) // (c["B"] * c["new_hi"] * c["H"]))
        c["len_hi"] = max(c["new_hi"], _log(rng, 16, max(16, most)))
        c["len_lo"] = rng.choice([1, c["len_hi"], rng.randint(1, c["len_hi"])])
        c["new_lo"] = rng.randint(1, c["new_hi"])
    elif op == "evict":
        c["B"] = _log(rng, 1, 64)
        c["len_hi"] = _log(rng, 4, min(131072, (64 * 6000) // c["B"]))
        c["len_lo"] = rng.choice([1, c["len_hi"], rng.randint(1, c["len_hi"])])
        c["keep"] = rng.randint(1, c["len_hi"])
        c["recent"] = rng.choice([0, rng.randint(0, c["keep"]), _log(rng, 1, c["keep"])])
        c["per_head"] = rng.random() < 0.5
    else:
        c["B"] = _log(rng, 1, 96)
        c["old_lo"], c["old_hi"] = 0, _log(rng, 1, 4000)
        c["new_hi"] = _log(rng, 1, 200)
        c["new_lo"] = rng.randint(1, c["new_hi"])
        c["width"] = rng.randint(1, 6)
        c["weights"] = rng.random() < 0.5
    return c


# ---------------------------------------------------------------------------- inputs

def _values(shape, D, gen):
    """Activations: normal, a few channels much larger, as keys have them."""
    x = torch.randn(*shape, D, device="cuda", generator=gen)
    return x * (1.0 + 4.0 * (torch.arange(D, device="cuda") % 17 == 3))


def _scale(amax, kv):
    """The scale that a block whose largest magnitude is `amax` needs."""
    if kv == "int8":
        return amax / 127
    m, e = torch.frexp(amax.double() / 448)  # amax / 448 = m 2^e, m in [0.5, 1)
    s = torch.ldexp(torch.ones_like(m), torch.where(m > 0.5, e, e - 1)).float()
    return torch.where(amax > 0, s, torch.zeros_like(s))


def _round(y, kv):
    """Values in code units as codes."""
    return y.round().to(torch.int8) if kv == "int8" else y.to(torch.float8_e4m3fn)


def _codes(x, s, kv):
    """x / s in 8 bits (0 where the scale is 0)."""
    y = torch.where(s > 0, x / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(x))
    return _round(y.clamp(-127, 127) if kv == "int8" else y.clamp(-448, 448), kv)


def _trees(new, width, rng):
    """Parents of each sequence's drafted tokens: the first is the last accepted token, the others hang on one of
    the `width` before them or, as the first tokens' further candidates, on the first."""
    out = []
    for n in new:
        p = [-1]
        for i in range(1, n):
            p.append(rng.randint(max(0, i - width), i - 1) if rng.random() < 0.8 else rng.randint(0, min(i - 1, 3)))
        out.append(p)
    return out


def _words(parents, W):
    """Bit masks [T, W] (int32) of trees, and the tokens' depths."""
    rows, depth = [], []
    for p in parents:
        seen, d = [], []
        for i, a in enumerate(p):
            seen.append((seen[a] if a >= 0 else 0) | 1 << i)
            d.append(d[a] + 1 if a >= 0 else 0)
        rows += [[(m >> (32 * w) & 0xFFFFFFFF) for w in range(W)] for m in seen]
        depth += d
    words = torch.tensor(rows, dtype=torch.int64).view(-1, W)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32).cuda(), depth


def prepare(case, seed):
    c = dict(case)
    op, B = c["op"], c["B"]
    # the lengths go by the case alone: the outputs of every seed have the same shapes
    rng = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    gen = torch.Generator(device="cuda").manual_seed(seed)
    seeded = random.Random(seed)
    if op in ("tree", "keep"):
        new = [rng.randint(c["new_lo"], c["new_hi"]) for _ in range(B)]
        old = [rng.randint(c["old_lo"], c["old_hi"]) if op == "keep" else seeded.randint(0, 3000) for _ in range(B)]
        lens = [o + n for o, n in zip(old, new)]
    else:
        lens = [rng.randint(c["len_lo"], c["len_hi"]) for _ in range(B)]
        lens[0] = c["len_hi"]
        new = [0] * B if op == "evict" else [min(n, rng.randint(c["new_lo"], c["new_hi"])) for n in lens]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s = dict(case=c, lens=torch.tensor(lens, device="cuda", dtype=torch.int32),
             cu=torch.tensor(cu, device="cuda", dtype=torch.int32),
             new=torch.tensor(new, device="cuda", dtype=torch.int32), max_new=max(new))
    T, W = cu[-1], -(-max(new) // 32)
    if c.get("width"):
        trees = _trees(new, c["width"], seeded)
        s["parents"] = torch.tensor([p for t in trees for p in t], device="cuda", dtype=torch.int32)
    if op == "tree":
        return s
    G, D, page, kv, dt = c["G"], c["D"], c["page"], c["kv"], _DT[c["dt"]]
    # pages: every sequence's in any order of the pool, a few of the pool unused
    need = [-(-n // page) for n in lens]
    P = sum(need) + 3
    perm = torch.randperm(P, device="cuda", generator=gen).to(torch.int32)
    MP = max(need)
    cum = [0]
    for n in need:
        cum.append(cum[-1] + n)
    col = torch.arange(MP, device="cuda")[None, :]
    first = torch.tensor(cum[:-1], device="cuda")[:, None]
    have = torch.tensor(need, device="cuda")[:, None]
    s["table"] = torch.where(col < have, perm[(first + col).clamp(max=P - 1)],
                             torch.full((), -1, device="cuda", dtype=torch.int32))
    kc = torch.empty(P, G, page, D, device="cuda", dtype=torch.int8 if kv == "int8" else torch.float8_e4m3fn)
    vc = torch.empty_like(kc)
    ks = torch.empty(P, G, device="cuda")
    vs = torch.empty(P, G, device="cuda")
    step = max(1, (1 << 27) // (G * page * D))
    for a in range(0, P, step):  # the pool's contents, a part at a time
        n = min(step, P - a)
        for codes, scale in ((kc, ks), (vc, vs)):
            x = _values((n, G, page), D, gen)
            t = _scale(x.abs().amax(dim=(2, 3)), kv)
            codes[a:a + n] = _codes(x, t[:, :, None, None], kv)
            scale[a:a + n] = t
    s["cache"] = (kc, vc, ks, vs)
    if op in ("weigh", "evict") or c.get("weights"):
        # what earlier tokens' weights add up to: a few tokens have most of it, many next to none
        s["weight"] = torch.exp(2.5 * torch.randn(P, G, page, device="cuda", generator=gen) - 3)
        s["weight"] *= torch.rand(P, G, page, device="cuda", generator=gen) > 0.03  # (and some none at all)
        # positions: in order at the end, mixed where an earlier eviction filled free slots
        pos = torch.zeros(P, G, page, device="cuda", dtype=torch.int32)
        heads = G if c.get("per_head") else 1
        for b in range(B):
            n, m = lens[b], lens[b] * 3 // 4
            at = torch.rand(heads, 2 * m, device="cuda", generator=gen).argsort(1)[:, :m]
            p = torch.cat([at, 2 * m + torch.arange(n - m, device="cuda").expand(heads, n - m)], 1).to(torch.int32)
            p = torch.nn.functional.pad(p, (0, need[b] * page - n)).view(heads, need[b], page).transpose(0, 1)
            pos[s["table"][b, :need[b]].long()] = p.expand(-1, G, -1).contiguous()
        s["position"] = pos
    if op == "evict":
        return s
    s["tok_b"] = torch.repeat_interleave(torch.arange(B, device="cuda"), s["new"].long())
    s["tok_i"] = torch.arange(T, device="cuda") - s["cu"].long()[s["tok_b"]]
    if op == "keep":
        paths = []
        for p in trees:
            at, path = seeded.randrange(len(p)), []
            while at >= 0:
                path.append(at)
                at = p[at]
            paths.append(path[::-1])
        wide = max(new)
        s["accepted"] = torch.tensor([p + [-1] * (wide - len(p)) for p in paths], device="cuda", dtype=torch.int32)
        start = torch.tensor([o // page * page for o in old], device="cuda")
        s["idx"] = start[:, None] + torch.arange(wide + page, device="cuda")[None, :]
        return s
    s["q"] = torch.randn(T, c["H"], D, device="cuda", generator=gen).to(dt)
    s["tree"] = None
    depth = s["tok_i"]
    if c["width"]:
        s["tree"], d = _words(trees, W)
        depth = torch.tensor(d, device="cuda")
    if op == "weigh":  # positions of a sequence some of whose tokens were evicted before
        s["positions"] = ((s["lens"] - s["new"]).long() * 2 + 5)[s["tok_b"]].add(depth).to(torch.int32)
    return s


# ---------------------------------------------------------------------------- plain forms

def _take(codes, *at):
    """codes[at] (indexing goes by bytes: not every 8-bit type has it)."""
    return codes.view(torch.int8)[at].view(codes.dtype)


def _tree_plain(st):
    """Ancestors by repeated products of the relation `sees itself or its parent`."""
    B, n, T = st["case"]["B"], st["max_new"], st["parents"].shape[0]
    W = -(-n // 32)
    i = torch.arange(n, device="cuda")
    row = (st["cu"].long()[:-1, None] + i).clamp(max=T - 1)
    live = i < st["new"].long()[:, None]
    up = torch.where(live, st["parents"].long()[row], torch.full((), -1, device="cuda"))
    sees = ((i[None, None, :] == i[None, :, None]) | (i[None, None, :] == up[:, :, None])).float()
    step = 1
    while step < n:
        sees = ((sees @ sees) > 0).float()
        step *= 2
    depth = sees.sum(-1).long() - 1
    bits = torch.nn.functional.pad(sees.long(), (0, 32 * W - n)).view(B, n, W, 32)
    words = (bits << torch.arange(32, device="cuda")).sum(-1)
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
    pos = ((st["lens"] - st["new"]).long()[:, None] + depth).to(torch.int32)
    return {"tree": words[live], "positions": pos[live]}


def _attend_plain(st):
    c = st["case"]
    B, H, G, D = c["B"], c["H"], c["G"], c["D"]
    R, Q = H // G, st["max_new"]
    pid = st["table"].long().clamp(min=0)
    k, v = [(_take(codes, pid).float() * scale[pid][..., None, None]).transpose(1, 2).flatten(2, 3)
            for codes, scale in (st["cache"][0::2], st["cache"][1::2])]  # [B, G, L, D]
    i = torch.arange(Q, device="cuda")
    row = (st["cu"].long()[:-1, None] + i).clamp(max=st["q"].shape[0] - 1)
    q = st["q"][row].float().view(B, Q, G, R, D).permute(0, 2, 1, 3, 4).reshape(B, G, Q * R, D)
    s = (q @ k.transpose(2, 3)) * D ** -0.5
    slot, old = torch.arange(k.shape[2], device="cuda"), (st["lens"] - st["new"]).long()
    if st["tree"] is None:
        seen = slot < (old[:, None] + i + 1)[:, :, None]
    else:
        j = slot[None, :] - old[:, None]  # [B, L]
        words = st["tree"].long()[row]  # [B, Q, W]
        at = j.clamp(0, 32 * words.shape[2] - 1)[:, None, :].expand(-1, Q, -1)
        bit = words.gather(2, at // 32) >> (at % 32) & 1
        seen = (j < 0)[:, None, :] | ((bit == 1) & (j < st["new"].long()[:, None])[:, None, :])
    seen = seen & (i < st["new"].long()[:, None])[:, :, None]  # rows behind a shorter sequence's: none
    s = s.masked_fill(~seen.repeat_interleave(R, dim=1)[:, None], float("-inf"))
    top = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(top > float("-inf"), top, torch.zeros_like(top)))
    p = p / p.sum(dim=-1, keepdim=True).clamp(min=1e-30)
    o = (p @ v).view(B, G, Q, R, D).permute(0, 2, 1, 3, 4).reshape(B, Q, H, D)
    out = {"out": o[st["tok_b"], st["tok_i"]].to(st["q"].dtype)}
    if c["op"] == "weigh":
        add = p.sum(dim=2, dtype=torch.float64).float()  # [B, G, L]
        b, n = (slot[None, :] < st["lens"].long()[:, None]).nonzero(as_tuple=True)
        page = pid[b, n // c["page"]]
        was = torch.where((n < old[b])[:, None], st["weight"][page, :, n % c["page"]], torch.zeros((), device="cuda"))
        st["weight"][page, :, n % c["page"]] = was + add[b, :, n]
        n = (st["lens"].long() - st["new"])[st["tok_b"]] + st["tok_i"]
        st["position"][pid[st["tok_b"], n // c["page"]], :, n % c["page"]] = st["positions"][:, None].expand(-1, G)
        out.update(weight=st["weight"], position=st["position"])
    return out


def _move(st, b, g, dst, src, lens):
    """Tokens of head g[i] (None: all heads) of sequence b[i] from slot src[i] to dst[i]; the others of the first
    lens[b] slots stay where they are."""
    c = st["case"]
    page, kv, G = c["page"], c["kv"], c["G"]
    if g is None:
        b, dst, src = [x.repeat_interleave(G) for x in (b, dst, src)]
        g = torch.arange(G, device="cuda").repeat(b.shape[0] // G)
    table = st["table"].long()
    pd, ps = table[b, dst // page], table[b, src // page]
    moved = torch.zeros(st["cache"][0].shape[:3], dtype=torch.bool, device="cuda")
    moved[pd, g, dst % page] = True
    sb, slot = (torch.arange(table.shape[1] * page, device="cuda") < lens.long()[:, None]).nonzero(as_tuple=True)
    stays = torch.zeros_like(moved)
    stays[table[sb, slot // page], :, slot % page] = True
    stays &= ~moved
    touched = moved.any(-1)
    tp, tg = touched.nonzero(as_tuple=True)
    for codes, scale in (st["cache"][0::2], st["cache"][1::2]):
        row, was = _take(codes, ps, g, src % page).float(), scale.clone()
        need = torch.zeros_like(scale).view(-1).scatter_reduce(0, pd * G + g, row.abs().amax(-1) * was[ps, g], "amax")
        s_old = torch.where(stays.any(-1), was, torch.zeros_like(was))
        s = torch.where(touched, torch.maximum(s_old, _scale(need.view_as(scale), kv)), was)
        some = torch.where(s > 0, s, torch.ones_like(s))
        kept = _take(codes, tp, tg)
        grown = _round(kept.float() * (was / some)[tp, tg, None, None], kv)
        grown = torch.where((stays[tp, tg] & (s > was)[tp, tg, None])[..., None], grown.float(), kept.float())
        codes.view(torch.int8)[tp, tg] = grown.to(codes.dtype).view(torch.int8)
        new = _round(row * (was[ps, g] / some[pd, g])[:, None], kv)
        codes.view(torch.int8)[pd, g, dst % page] = new.view(torch.int8)
        scale.copy_(s)
    if "weight" in st:
        for t in (st["weight"], st["position"]):
            t[pd, g, dst % page] = t[ps, g, src % page]


def _values_of(st, idx, lens):
    """Slots idx [B, n] in 16 bits, zeros behind lens."""
    c = st["case"]
    live = idx < lens.long()[:, None]
    at = torch.where(live, idx, torch.zeros_like(idx))
    pid = st["table"].long().gather(1, at // c["page"])
    return [torch.where(live[:, :, None, None],
                        _take(codes, pid, slice(None), at % c["page"]).float() * scale[pid][..., None],
                        torch.zeros((), device="cuda")).to(_DT[c["dt"]])
            for codes, scale in (st["cache"][0::2], st["cache"][1::2])]


def _evict_plain(st):
    c = st["case"]
    page, keep = c["page"], c["keep"]
    pid = st["table"].long().clamp(min=0)
    w, pos = [t[pid].transpose(1, 2).flatten(2) for t in (st["weight"], st["position"])]  # [B, G, L]
    if not c["per_head"]:
        w, pos = w.sum(1, keepdim=True, dtype=torch.float64).float(), pos[:, :1]
    lens = st["lens"].long()
    slot = torch.arange(w.shape[2], device="cuda")
    live = slot < lens[:, None, None]
    pos = torch.where(live, pos, torch.full_like(pos, -2 ** 31)).long()
    recent = live & (pos > pos.amax(2, keepdim=True) - c["recent"])
    # dead slots last, then by recency, weight and slot: stable sorts from the last criterion to the first
    order = torch.where(live, w, torch.full_like(w, -1.0)).sort(dim=2, descending=True, stable=True).indices
    order = order.gather(2, recent.long().gather(2, order).sort(dim=2, descending=True, stable=True).indices)
    kept = torch.zeros_like(order, dtype=torch.bool).scatter(2, order[:, :, :keep], True) & live
    new_lens = torch.minimum(lens, torch.full_like(lens, keep))
    front = slot < new_lens[:, None, None]
    b, g, dst = (front & ~kept).nonzero(as_tuple=True)  # sequence, head, slot ascending
    _, _, src = (kept & ~front & live).nonzero(as_tuple=True)
    _move(st, b, g if c["per_head"] else None, dst, src, new_lens)
    k, v = _values_of(st, torch.arange(keep, device="cuda").expand(c["B"], -1), new_lens)
    return {"k": k, "v": v, "lens": new_lens.to(torch.int32), "weight": st["weight"], "position": st["position"]}


def _keep_plain(st):
    c = st["case"]
    acc, new = st["accepted"].long(), st["new"].long()
    before = torch.nn.functional.pad(acc, (1, 0), value=-1)[:, :-1]
    ok = ((acc > before) & (acc < new[:, None])).long().cumprod(1).bool()
    old = st["lens"].long() - new
    new_lens = old + ok.sum(1)
    j = torch.arange(acc.shape[1], device="cuda")
    b, i = (ok & (acc != j)).nonzero(as_tuple=True)
    _move(st, b, None, old[b] + i, old[b] + acc[b, i], new_lens)
    k, v = _values_of(st, st["idx"], new_lens)
    out = {"k": k, "v": v, "lens": new_lens.to(torch.int32)}
    if c["weights"]:
        out.update(weight=st["weight"], position=st["position"])
    return out


def run(state):
    st, c = state, state["case"]
    if not own:
        return {"tree": _tree_plain, "tree_attend": _attend_plain, "weigh": _attend_plain, "evict": _evict_plain,
                "keep": _keep_plain}[c["op"]](st)
    from spatten_b200 import paged
    if c["op"] == "tree":
        tree, positions = paged.paged_tree(st["parents"], st["cu"], st["lens"], st["max_new"])
        return {"tree": tree, "positions": positions}
    cache = paged.PagedKVCache(*st["cache"])
    weights = paged.PagedWeights(st["weight"], st["position"]) if "weight" in st else None
    if c["op"] == "tree_attend":
        return {"out": paged.paged_attention(st["q"], cache, st["table"], st["cu"], st["lens"], st["max_new"],
                                             tree=st["tree"])}
    if c["op"] == "weigh":
        out = paged.paged_attention(st["q"], cache, st["table"], st["cu"], st["lens"], st["max_new"], tree=st["tree"],
                                    weights=weights, positions=st["positions"])
        return {"out": out, "weight": weights.weight, "position": weights.position}
    if c["op"] == "evict":
        lens = paged.paged_evict(cache, weights, st["table"], st["lens"], c["keep"], recent=c["recent"],
                                 per_head=c["per_head"])
        k, v = paged.paged_read(cache, st["table"], lens, n_tokens=c["keep"], dtype=_DT[c["dt"]])
    else:
        lens = paged.paged_keep(cache, st["table"], st["cu"], st["lens"], st["accepted"], weights=weights)
        k, v = paged.paged_read(cache, st["table"], lens, idx=st["idx"], dtype=_DT[c["dt"]])
    out = {"k": k, "v": v, "lens": lens}
    if weights is not None:
        out.update(weight=weights.weight, position=weights.position)
    return out


# ---------------------------------------------------------------------------- work and 64-bit values

def _mean(lo, hi):
    return (lo + hi) / 2


def work(case):
    c = case
    B = c["B"]
    if c["op"] == "tree":
        T = B * _mean(c["new_lo"], c["new_hi"])
        return {"bytes": T * (8 + 4 * -(-c["new_hi"] // 32)), "flops": T * max(1, _mean(c["new_lo"], c["new_hi"]) / 4)}
    G, D = c["G"], c["D"]
    if c["op"] in ("tree_attend", "weigh"):
        n, new = B * _mean(c["len_lo"], c["len_hi"]), _mean(c["new_lo"], c["new_hi"])
        seen = max(n / B - new / 2, 1)
        work = {"bytes": n * G * D * 2 + 4 * B * new * c["H"] * D, "flops": 4 * B * new * seen * c["H"] * D}
        if c["op"] == "weigh":
            work["bytes"] += n * G * 8 + B * new * G * 4
            work["flops"] += B * new * seen * c["H"]
        return work
    if c["op"] == "evict":
        n = _mean(c["len_lo"], c["len_hi"])
        kept = min(n, c["keep"])
        moved = kept * max(0.0, 1 - c["keep"] / n)  # free slots among the first, as many as go
        heads = G if c["per_head"] else 1
        return {"bytes": B * (n * (4 * G + (4 * heads if c["recent"] else 0)) + moved * G * (4 * D + 16)
                              + kept * G * D * 6), "flops": B * (n + kept * D * 2) * G}
    n = _mean(c["new_lo"], c["new_hi"])
    path = max(1, n / (1 + c["width"]))
    return {"bytes": B * (path * G * (4 * D + (16 if c["weights"] else 0)) + (path + c["page"] / 2) * G * D * 6),
            "flops": B * (path + c["page"] / 2) * G * D * 2}


def _exact_moved(st, moves, new_lens):
    """moves[b][g]: a list of (slot to, slot from); the pools afterwards, in 64 bits: (K, V as dicts of page and head
    to values, scales), computed per page from what it holds at the end."""
    c = st["case"]
    page, kv = c["page"], c["kv"]
    top = 127.0 if kv == "int8" else 448.0
    values = []
    for codes, scale in (st["cache"][0::2], st["cache"][1::2]):
        was = scale.double()
        whole = codes.float().double() * was[:, :, None, None]
        values.append(whole.clone())
        for b, heads in enumerate(moves):
            for g, pairs in enumerate(heads):
                if not pairs:
                    continue
                to, fr = torch.tensor(pairs, device="cuda").T
                table = st["table"][b].long()
                for i in (to // page).unique().tolist():
                    here = to // page == i
                    pid, at = int(table[i]), to[here] % page
                    rows = whole[table[fr[here] // page], g, fr[here] % page]
                    stay = torch.arange(page, device="cuda") + i * page < new_lens[b]
                    stay[at] = False
                    s = rows.abs().amax() / top
                    if kv != "int8" and s > 0:
                        s = torch.exp2(torch.ceil(torch.log2(s)))
                    if stay.any():
                        s = torch.maximum(s, was[pid, g])
                    new = whole[pid, g].clone()
                    new[at] = rows
                    y = new / s if s > 0 else torch.zeros_like(new)
                    y = y.round() if kv == "int8" else y.float().to(torch.float8_e4m3fn).double()
                    values[-1][pid, g] = y * s
    return values


def exact(case, seed):
    c = case
    B = c["B"]
    st = prepare(c, seed)
    lens, cu = st["lens"].tolist(), st["cu"].tolist()
    if c["op"] == "tree":
        up, rows, pos = st["parents"].tolist(), [], []
        W = -(-st["max_new"] // 32)
        for b in range(B):
            n = cu[b + 1] - cu[b]
            for i in range(n):
                chain, a = [], i
                while a >= 0:
                    chain.append(a)
                    a = up[cu[b] + a]
                words = [0] * W
                for a in chain:
                    words[a >> 5] += 1 << (a & 31)
                rows.append([x - (1 << 32) if x >> 31 else x for x in words])
                pos.append(lens[b] - n + len(chain) - 1)
        return {"tree": torch.tensor(rows, dtype=torch.int32, device="cuda"),
                "positions": torch.tensor(pos, dtype=torch.int32, device="cuda")}
    page, G, D = c["page"], c["G"], c["D"]
    table = st["table"].long()
    if c["op"] in ("tree_attend", "weigh"):
        R = c["H"] // G
        out = torch.zeros(cu[-1], c["H"], D, device="cuda", dtype=torch.float64)
        total = st["weight"].double() if c["op"] == "weigh" else None
        for b in range(B):
            L, n = lens[b], cu[b + 1] - cu[b]
            old = L - n
            pages = table[b, :-(-L // page)]
            may = torch.ones(n, L, dtype=torch.bool, device="cuda")
            if st["tree"] is None:
                may = may.tril(old)
            else:
                j = torch.arange(n, device="cuda")
                may[:, old:] = (st["tree"][cu[b]:cu[b + 1]].long()[:, j >> 5] >> (j & 31)) % 2 == 1
            for g in range(G):
                K, V = [(st["cache"][t].view(torch.int8)[pages, g].view(st["cache"][t].dtype).double()
                         * st["cache"][2 + t].double()[pages, g, None, None]).reshape(-1, D)[:L] for t in range(2)]
                mass = torch.zeros(L, dtype=torch.float64, device="cuda")
                for h in range(g * R, (g + 1) * R):
                    z = st["q"][cu[b]:cu[b + 1], h].double() @ K.T / D ** 0.5
                    p = torch.softmax(z.masked_fill(~may, float("-inf")), -1)
                    out[cu[b]:cu[b + 1], h] = p @ V
                    mass += p.sum(0)
                if total is not None:
                    flat = total[pages, g].reshape(-1)
                    flat[old:L] = 0
                    flat[:L] += mass
                    total[pages, g] = flat.view(-1, page)
        if total is None:
            return {"out": out}
        position = st["position"].clone()
        for b in range(B):
            for i in range(cu[b + 1] - cu[b]):
                s = lens[b] - (cu[b + 1] - cu[b]) + i
                position[table[b, s // page], :, s % page] = st["positions"][cu[b] + i]
        return {"out": out, "weight": total, "position": position}
    moves, new_lens = [], []
    if c["op"] == "evict":
        for b in range(B):
            L = lens[b]
            new_lens.append(min(L, c["keep"]))
            pages = table[b, :-(-L // page)]
            w = st["weight"][pages].transpose(0, 1).reshape(G, -1)[:, :L].double()
            p = st["position"][pages].transpose(0, 1).reshape(G, -1)[:, :L].long()
            heads = []
            for g in range(G if c["per_head"] else 1):
                if L <= c["keep"]:
                    heads.append([])
                    continue
                score = (w[g] if c["per_head"] else w.sum(0)).float().tolist()
                place = p[g].tolist()
                newest = max(place)
                best = sorted(range(L), key=lambda n: (place[n] <= newest - c["recent"], -score[n], n))[:c["keep"]]
                chosen = set(best)
                heads.append(list(zip([n for n in range(c["keep"]) if n not in chosen],
                                      [n for n in range(c["keep"], L) if n in chosen])))
            moves.append(heads if c["per_head"] else heads * G)
        idx = torch.arange(c["keep"], device="cuda").expand(B, -1)
    else:
        for b, path in enumerate(st["accepted"].tolist()):
            n = cu[b + 1] - cu[b]
            path = [a for a in path if a >= 0]
            new_lens.append(lens[b] - n + len(path))
            moves.append([[(lens[b] - n + i, lens[b] - n + a) for i, a in enumerate(path) if a != i]] * G)
        idx = st["idx"]
    values = _exact_moved(st, moves, new_lens)
    got = {"k": None, "v": None}
    for name, val in zip(got, values):
        x = torch.zeros(B, idx.shape[1], G, D, dtype=torch.float64, device="cuda")
        for b in range(B):
            at = idx[b][idx[b] < new_lens[b]]
            x[b, :at.shape[0]] = val[table[b, at // page], :, at % page]
        got[name] = x
    got["lens"] = torch.tensor(new_lens, dtype=torch.int32, device="cuda")
    if "weight" in st:
        weight, position = st["weight"].double(), st["position"].clone()
        for b in range(B):
            for g in range(G):
                if moves[b][g]:
                    to, fr = torch.tensor(moves[b][g], device="cuda").T
                    for t in (weight, position):
                        t[table[b, to // page], g, to % page] = t[table[b, fr // page], g, fr % page]
        got.update(weight=weight, position=position)
    return got
