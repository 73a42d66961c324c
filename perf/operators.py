"""The key/value cache operators of a decode step: what is measured of them, and their plain forms.

Five operators that a decoder runs around its projections, on a cache of keys and values [batch, kv heads, slots, head
width] whose sequences are as long as a device array `lens` says:

  append     rotate (and optionally norm) the new tokens' queries and keys, write keys and values behind each sequence
  attention  a tree of drafted tokens attends to the sequence before it and to its own ancestors
  mass       add up, per cached slot, the attention weight that the accepted tokens gave it
  evict      keep the first slots, the last ones and the heaviest of the others, in order, in a smaller cache
  accept     walk the drafted tree along the target's tokens, move the accepted tokens' keys and values into place

A case is a dict of plain values; `run` is one call. With `own` false it is the operator in elementary torch operations
in 32 bits, with `own` true the framework's call. `exact` is the definition in 64 bits, written on its own.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    """Head layouts and layer counts are those of the decoder's two architectures (32 query heads over 8 of 128; 36
    layers), or generic (14 over 2 of 64)."""
    return [
        # plain decoding at the start of a chat: nothing but latency
        {"name": "attention one token", "op": "attention", "type": "bf16", "batch": 1, "tokens": 1, "heads": 32, "kv": 8, "width": 128, "longest": 129, "shortest": 129, "tree": False},
        # the decoder's own 32-bit cache, twelve drafted tokens
        {"name": "attention tree 32-bit cache", "op": "attention", "type": "fp32", "batch": 1, "tokens": 12, "heads": 32, "kv": 8, "width": 128, "longest": 2047, "shortest": 2047, "tree": True},
        # a serving batch, every sequence of another length, small trees
        {"name": "attention ragged batch", "op": "attention", "type": "fp16", "batch": 24, "tokens": 7, "heads": 32, "kv": 8, "width": 128, "longest": 8192, "shortest": 501, "tree": True},
        # one long document, the largest tree
        {"name": "attention long document", "op": "attention", "type": "bf16", "batch": 1, "tokens": 64, "heads": 32, "kv": 8, "width": 128, "longest": 131000, "shortest": 131000, "tree": True},
        # plain decoding with an eviction budget: one token's weights, narrow heads in groups of seven
        {"name": "mass one token", "op": "mass", "type": "bf16", "batch": 1, "tokens": 1, "heads": 14, "kv": 2, "width": 64, "longest": 1000, "shortest": 1000, "accepted": 1, "path": False},
        # the end of a prompt votes for what of it is kept
        {"name": "mass prompt window", "op": "mass", "type": "fp16", "batch": 2, "tokens": 64, "heads": 32, "kv": 8, "width": 128, "longest": 32768, "shortest": 30001, "accepted": 64, "path": False},
        # one layer that is 64 slots over its budget
        {"name": "evict one layer", "op": "evict", "type": "bf16", "layers": 1, "batch": 1, "kv": 8, "width": 128, "longest": 2112, "shortest": 2112, "budget": 2048, "sinks": 4, "recent": 64},
        # all layers after a long prompt
        {"name": "evict all layers", "op": "evict", "type": "bf16", "layers": 36, "batch": 1, "kv": 8, "width": 128, "longest": 16384, "shortest": 16384, "budget": 2048, "sinks": 4, "recent": 128},
        # one sequence, eight drafted tokens, three of them taken
        {"name": "accept small tree", "op": "accept", "type": "fp16", "layers": 36, "batch": 1, "tokens": 8, "kv": 8, "width": 128, "longest": 1500, "shortest": 1500, "accepted": 3},
        # a batch with the largest trees
        {"name": "accept batch", "op": "accept", "type": "bf16", "layers": 32, "batch": 16, "tokens": 64, "kv": 8, "width": 128, "longest": 1024, "shortest": 77, "accepted": 6},
        # one decoded token of an architecture that norms its queries and keys
        {"name": "append one token", "op": "append", "type": "fp16", "batch": 1, "tokens": 1, "heads": 32, "kv": 8, "width": 128, "longest": 777, "shortest": 777, "norm": True},
        # a prompt
        {"name": "append prompt", "op": "append", "type": "bf16", "batch": 1, "tokens": 4099, "heads": 32, "kv": 8, "width": 128, "longest": 0, "shortest": 0, "norm": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "mass", "evict", "accept", "append"])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 4, 5, 7, 8])
    c = {"op": op, "type": rng.choice(["bf16", "fp16", "fp32"]), "batch": _log(rng, 1, 32), "kv": kv, "width": rng.choice([64, 128])}
    if op in ("attention", "mass"):
        c["tokens"], c["heads"], c["longest"] = _log(rng, 1, 64), kv * group, _log(rng, 1, 131000)
        if op == "attention":
            c["tree"] = rng.random() < 0.7
        else:
            c["accepted"] = rng.randint(1, c["tokens"])
            c["path"] = rng.random() < 0.6
    elif op == "evict":
        c["layers"], c["longest"] = rng.choice([1, 1, rng.randint(2, 36)]), _log(rng, 16, 131000)
    elif op == "accept":
        c["layers"], c["tokens"], c["longest"] = rng.randint(1, 36), _log(rng, 1, 64), _log(rng, 1, 1500)
        c["accepted"] = rng.randint(1, max(1, min(c["tokens"], 12)))
    else:
        c["tokens"], c["heads"], c["longest"] = _log(rng, 1, 4096), kv * group, _log(rng, 1, 8192)
        c["norm"] = rng.random() < 0.5
    shorter = rng.choice([0.0, rng.random()])

    def costs():
        slots = c["batch"] * kv * (c["longest"] + c.get("tokens", 0)) * c.get("layers", 1)
        size = c["width"] * SIZE[c["type"]]
        if op in ("attention", "mass"):  # products of 32-bit values cost more
            return max(slots * size / (1 << 28), slots * c["tokens"] * group * c["width"] / (8e8 if c["type"] == "fp32" else 8e9))
        if op == "append":
            return c["batch"] * c["tokens"] * (c["heads"] + 2 * kv) * (c["width"] * 4 + size) / 150e6
        return slots * size / (150e6 if op == "evict" else 500e6)

    while costs() > 1:  # no more than the largest listed cases
        big = max((x for x in (("batch", "tokens") if op == "append" else ("batch", "layers", "longest")) if x in c), key=lambda x: c[x])
        c[big] = c[big] * 2 // 3
    c["shortest"] = int(c["longest"] * (1 - shorter))
    if op == "evict":
        c["budget"] = min(_log(rng, 8, 8192), c["longest"])
        c["sinks"] = rng.randint(0, min(8, c["budget"] // 2))
        c["recent"] = rng.randint(0, c["budget"] // 2)
    return c


def _lens(c):
    """The sequences' lengths: from the longest down to the shortest in even steps."""
    return [c["longest"] - (b * (c["longest"] - c["shortest"])) // max(1, c["batch"] - 1) for b in range(c["batch"])]


def work(case):
    """Each key, value, query and weight that the operator needs read once, each result written once."""
    c, e = case, SIZE[case["type"]]
    row = c["width"] * e
    total = sum(_lens(c))
    if c["op"] == "attention":
        slots = (total + c["batch"] * c["tokens"]) * c["kv"]
        rows = c["batch"] * c["tokens"] * c["heads"]
        return {"bytes": 2 * slots * row + rows * (2 * row + 4), "flops": 4 * c["width"] * (c["heads"] // c["kv"]) * c["tokens"] * slots}
    if c["op"] == "mass":
        slots = (total + c["batch"] * c["accepted"]) * c["kv"]
        rows = c["batch"] * c["accepted"] * c["heads"]
        return {"bytes": slots * (row + 8) + rows * (row + 4), "flops": 2 * c["width"] * (c["heads"] // c["kv"]) * c["accepted"] * slots}
    if c["op"] == "evict":
        kept = sum(min(n, c["budget"]) for n in _lens(c))
        return {"bytes": c["layers"] * c["kv"] * (4 * total + kept * (4 * row + 4 + 4)), "flops": 0}
    if c["op"] == "accept":
        return {"bytes": c["batch"] * (c["tokens"] * 24 + 24 + 4 * row * c["layers"] * c["kv"] * (c["accepted"] - 1)), "flops": 0}
    rows, keys = c["batch"] * c["tokens"] * c["heads"], c["batch"] * c["tokens"] * c["kv"]
    return {"bytes": (rows + 2 * keys) * c["width"] * (4 + e) + c["batch"] * c["tokens"] * (4 * c["width"] + 4), "flops": 6 * (rows + keys) * c["width"]}


# ------------------------------------------------------------------------------------------------------------ inputs
def _visible(mask, lens, tokens, cap):
    """[batch, tokens, cap]: a token sees the slots before its sequence's end and the drafted ones of its bits"""
    at = torch.arange(cap, device=lens.device)[None, None, :] - lens[:, None, None]
    bit = (mask[..., None] >> at.clamp(0, 63)) & 1
    return (at < 0) | ((at < tokens) & (bit != 0))


def _tree(g, batch, tokens, tree):
    """parents [batch, tokens] (a tree whose nodes mostly hang on recent ones, or a chain) and the ancestor bits"""
    t = torch.arange(tokens, device="cuda")
    back = torch.randint(1, 9, (batch, tokens), device="cuda", generator=g) if tree else torch.ones(batch, tokens, dtype=torch.int64, device="cuda")
    parents = (t[None] - back).clamp(min=0)
    parents[:, 0] = -1
    sees = torch.eye(tokens, dtype=torch.float32, device="cuda").repeat(batch, 1, 1)
    up = torch.nn.functional.one_hot(parents.clamp(min=0), tokens).float()
    up[:, 0] = 0
    for _ in range(6):  # paths of length up to 64 by squaring
        sees, up = ((sees + up @ sees) > 0).float(), ((up @ up) > 0).float()
    bits = (sees.long() << t).sum(-1)
    return parents.int(), bits


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = TYPES[c["type"]]
    B, kv, D = c["batch"], c["kv"], c["width"]
    lens = torch.tensor(_lens(c), dtype=torch.int32, device="cuda")

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32 if dtype == torch.float32 else dtype) * scale)

    s = {"case": c, "lens": lens}
    if c["op"] in ("attention", "mass"):
        T, H = c["tokens"], c["heads"]
        cap = c["longest"] + T + 5
        s["k"], s["v"] = normal(B, kv, cap, D), normal(B, kv, cap, D)
        s["k"] += normal(B, kv, 1, D, scale=0.5)  # keys share a direction
        s["q"] = normal(B, T, H, D, scale=1.5)
        s["scale"] = 1.0 / math.sqrt(D)
    if c["op"] == "attention":
        _, s["mask"] = _tree(g, B, T, c["tree"])
        s["out"], s["lse"] = torch.empty_like(s["q"]), torch.empty(B, T, H, device="cuda")
    elif c["op"] == "mass":
        n = c["accepted"]
        del s["v"]
        s["counts"] = torch.full((B,), n, dtype=torch.int32, device="cuda")
        order = torch.argsort(torch.rand(B, T, device="cuda", generator=g), dim=-1)[:, :n] if c["path"] else torch.arange(n, device="cuda").repeat(B, 1)
        s["rows"] = torch.full((B, T), -1, dtype=torch.int32, device="cuda")
        s["rows"][:, :n] = torch.sort(order, dim=-1).values
        s["path"] = c["path"]
        s["mass"] = torch.rand(B, kv, cap, device="cuda", generator=g).square() * 4
        s["out"] = torch.zeros_like(s["mass"])
        s["lse"] = torch.zeros(B, T, H, device="cuda")
        for b in range(B):  # what the attention call left for these rows
            n_b, G = int(_lens(c)[b]) + n, H // kv
            take = s["rows"][b, :n].long()
            x = s["q"][b, take].float().reshape(n, kv, G, D).permute(1, 0, 2, 3).reshape(kv, n * G, D)
            y = (x @ s["k"][b, :, :n_b].float().transpose(-1, -2)).mul_(s["scale"]).reshape(kv, n, G, n_b)
            late = torch.arange(n_b, device="cuda")[None, :] > n_b - n + torch.arange(n, device="cuda")[:, None]
            y.masked_fill_(late[None, :, None, :], -math.inf)
            s["lse"][b, take] = torch.logsumexp(y.double() if y.numel() < 1 << 26 else y, -1).permute(1, 0, 2).reshape(n, H).float()
    elif c["op"] == "evict":
        N, cap = c["layers"], c["longest"] + 3
        s["k"], s["v"] = normal(N, B, kv, cap, D), normal(N, B, kv, cap, D)
        # a few heavy slots, many light ones, some that nothing ever looked at
        m = torch.rand(N, B, kv, cap, device="cuda", generator=g)
        s["mass"] = torch.where(m < 0.1, torch.zeros_like(m), m.pow(8) * 50)
        b = c["budget"]
        s["k_out"], s["v_out"] = (torch.zeros(N, B, kv, b, D, dtype=dt, device="cuda") for _ in range(2))
        s["mass_out"] = torch.zeros(N, B, kv, b, device="cuda")
        s["kept"] = torch.empty(N, B, kv, b, dtype=torch.int32, device="cuda")
        s["new_lens"] = torch.empty_like(lens)
    elif c["op"] == "accept":
        N, T, n = c["layers"], c["tokens"], c["accepted"]
        cap = c["longest"] + T + 5
        s["k"], s["v"] = normal(N, B, kv, cap, D), normal(N, B, kv, cap, D)
        s["parents"], _ = _tree(g, B, T, True)
        s["tokens"] = torch.randint(0, 30000, (B, T), device="cuda", generator=g)
        s["target"] = torch.randint(30000, 32000, (B, T), device="cuda", generator=g)
        # the accepted path: the root and n - 1 later nodes, each hung on the one before and holding what the target says
        at = torch.sort(torch.argsort(torch.rand(B, T - 1, device="cuda", generator=g), dim=-1)[:, : n - 1] + 1, dim=-1).values
        at = torch.cat([torch.zeros(B, 1, dtype=torch.int64, device="cuda"), at], dim=1)
        s["parents"].scatter_(1, at[:, 1:], at[:, :-1].int())
        s["tokens"].scatter_(1, at[:, 1:], s["target"].gather(1, at[:, :-1]))
        s["res"] = {"path": torch.empty(B, T, dtype=torch.int32, device="cuda"), "accepted": torch.empty_like(lens), "next_token": torch.empty(B, dtype=torch.int64, device="cuda"), "new_lens": torch.empty_like(lens)}
    else:
        T, H = c["tokens"], c["heads"]
        cap = c["longest"] + T + 5
        x = normal(B * T, (H + 2 * kv) * D, dtype=torch.float32)  # the projections' outputs, one behind the other
        s["xq"], s["xk"], s["xv"] = (y.unflatten(1, (-1, D)).unflatten(0, (B, T)) for y in x.split([H * D, kv * D, kv * D], dim=1))
        s["k"], s["v"] = torch.zeros(B, kv, cap, D, dtype=dt, device="cuda"), torch.zeros(B, kv, cap, D, dtype=dt, device="cuda")
        s["pos"] = lens[:, None] + torch.arange(T, dtype=torch.int32, device="cuda")
        angle = torch.arange(cap, dtype=torch.float64, device="cuda")[:, None] * 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
        s["cos"], s["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
        s["q_norm"], s["k_norm"] = (normal(D, scale=0.1, dtype=torch.float32) + 1 if c["norm"] else None for _ in range(2))
        s["q_out"] = torch.empty(B, T, H, D, dtype=dt, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------------- plain forms
def _rows(q, kv):
    """[B, T, H, D] -> [B, kv, T * group, D] in 32 bits"""
    B, T, H, D = q.shape
    return q.float().reshape(B, T, kv, H // kv, D).permute(0, 2, 1, 3, 4).reshape(B, kv, -1, D)


def _attention(s):
    q, kv, cap = s["q"], s["k"].shape[1], s["k"].shape[2]
    B, T, H, D = q.shape
    seen = _visible(s["mask"], s["lens"], T, cap)
    x = (_rows(q, kv) @ s["k"].float().transpose(-1, -2)).mul_(s["scale"])
    x.masked_fill_(~seen[:, None, :, None, :].expand(B, 1, T, H // kv, cap).reshape(B, 1, -1, cap), -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p @ s["v"].float()) / total.clamp(min=1e-30)
    back = lambda y: y.reshape(B, kv, T, H // kv, -1).permute(0, 2, 1, 3, 4).reshape(B, T, H, -1)  # noqa: E731
    return {"out": back(o).to(q.dtype), "lse": back(top + total.log())[..., 0]}


def _mass(s):
    kv, cap, n = s["k"].shape[1], s["k"].shape[2], s["case"]["accepted"]
    B, T, H, D = s["q"].shape
    rows = s["rows"][:, :n].long()
    q = torch.gather(s["q"], 1, rows[..., None, None].expand(-1, -1, H, D))
    lse = torch.gather(s["lse"], 1, rows[..., None].expand(-1, -1, H))
    x = (_rows(q, kv) @ s["k"].float().transpose(-1, -2)).mul_(s["scale"])
    x.sub_(_rows(lse[..., None], kv))
    at = torch.arange(cap, device="cuda")[None, None, :] - s["lens"][:, None, None]
    seen = at <= torch.arange(n, device="cuda")[None, :, None]
    x.masked_fill_(~seen[:, None, :, None, :].expand(B, 1, n, H // kv, cap).reshape(B, 1, -1, cap), -math.inf)
    add = x.exp_().sum(2)
    at = at.expand(B, kv, cap)
    return {"mass": torch.where(at < 0, s["mass"] + add, torch.where(at < n, add, s["out"]))}


def _evict(s):
    k, m, lens, c = s["k"], s["mass"], s["lens"].long(), s["case"]
    N, B, kv, cap, D = k.shape
    budget, sinks, recent = c["budget"], c["sinks"], c["recent"]
    at = torch.arange(cap, device="cuda").expand(B, cap)
    group = torch.where((at < sinks) | (at >= lens[:, None] - recent), 0, 1)
    group = torch.where(at >= lens[:, None], 2, group)[None, :, None].expand(N, B, kv, cap)
    order = torch.sort(m, dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, torch.sort(group.gather(-1, order), dim=-1, stable=True).indices)
    new = lens.clamp(max=budget)
    live = torch.arange(budget, device="cuda") < new[:, None]
    live = live[None, :, None].expand(N, B, kv, budget)
    kept = torch.sort(torch.where(live, order[..., :budget], cap), dim=-1).values
    take = kept.clamp(max=cap - 1)
    rows = take[..., None].expand(N, B, kv, budget, D)
    return {"k": torch.where(live[..., None], k.gather(3, rows), s["k_out"]), "v": torch.where(live[..., None], s["v"].gather(3, rows), s["v_out"]),
            "mass": torch.where(live, m.gather(3, take), s["mass_out"]), "kept": torch.where(live, kept, -1).int(), "new_lens": new.int()}


def _accept(s):
    tokens, parents, target, lens = s["tokens"], s["parents"].long(), s["target"], s["lens"]
    B, T = tokens.shape
    up = parents.clamp(min=0)
    fits = (tokens == target.gather(1, up)) & (parents >= 0)
    first = torch.tril(torch.ones(T, T, dtype=torch.bool, device="cuda"), -1)  # an earlier child of the same parent that fits as well
    fits &= ~((up[:, :, None] == up[:, None, :]) & fits[:, None, :] & first).any(-1)
    fits[:, 0] = True
    for _ in range(6):  # a node is accepted where all of its ancestors are: paths of length up to 64 by doubling
        fits, up = fits & fits.gather(1, up), up.gather(1, up)
    n = fits.sum(1)
    t = torch.arange(T, device="cuda")
    path = torch.sort(torch.where(fits, t, T), dim=1).values
    last = path.gather(1, n[:, None] - 1)
    live = t < n[:, None]
    src = (lens[:, None] + torch.where(live, path, t))[None, :, None, :, None]
    dst = (lens[:, None] + t)[None, :, None, :, None]
    shape = (*s["k"].shape[:3], T, s["k"].shape[4])
    src, dst = src.expand(shape), dst.expand(shape)
    s["k"].scatter_(3, dst, s["k"].gather(3, src))
    s["v"].scatter_(3, dst, s["v"].gather(3, src))
    return {"path": torch.where(live, path, -1).int(), "accepted": n.int(), "next_token": target.gather(1, last)[:, 0], "new_lens": (lens + n).int(), "k": s["k"], "v": s["v"]}


def _append(s):
    lens, pos, T = s["lens"].long(), s["pos"].long(), s["pos"].shape[1]

    def turn(x, w):
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        a, b = x.chunk(2, dim=-1)
        cos, sin = s["cos"][pos][:, :, None], s["sin"][pos][:, :, None]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)

    slot = (lens[:, None] + torch.arange(T, device="cuda"))[:, None, :, None].expand(s["k"].shape[0], s["k"].shape[1], T, s["k"].shape[3])
    s["k"].scatter_(2, slot, turn(s["xk"], s["k_norm"]).transpose(1, 2).to(s["k"].dtype))
    s["v"].scatter_(2, slot, s["xv"].transpose(1, 2).to(s["v"].dtype))
    return {"q": turn(s["xq"], s["q_norm"]).to(s["k"].dtype), "k": s["k"], "v": s["v"]}


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"attention": _attention, "mass": _mass, "evict": _evict, "accept": _accept, "append": _append}[op](s)
    from pingala8_llm_b200 import cache

    if op == "attention":
        out, lse = cache.tree_attention(s["q"], s["k"], s["v"], s["lens"], mask=s["mask"], scale=s["scale"], out=s["out"], lse=s["lse"])
        return {"out": out, "lse": lse}
    if op == "mass":
        return {"mass": cache.attention_mass(s["q"], s["lse"], s["k"], s["lens"], s["mass"], rows=s["rows"] if s["path"] else None, counts=s["counts"], scale=s["scale"], out=s["out"])}
    if op == "evict":
        c = s["case"]
        cache.kv_evict(s["k"], s["v"], s["mass"], s["lens"], c["budget"], sinks=c["sinks"], recent=c["recent"], k_out=s["k_out"], v_out=s["v_out"], mass_out=s["mass_out"], kept=s["kept"], new_lens=s["new_lens"])
        return {"k": s["k_out"], "v": s["v_out"], "mass": s["mass_out"], "kept": s["kept"], "new_lens": s["new_lens"]}
    if op == "accept":
        cache.tree_accept(s["tokens"], s["parents"], s["target"], s["k"], s["v"], s["lens"], **s["res"])
        return {**s["res"], "k": s["k"], "v": s["v"]}
    q = cache.kv_append(s["xq"], s["xk"], s["xv"], s["k"], s["v"], s["lens"], s["pos"], s["cos"], s["sin"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6, q_out=s["q_out"])
    return {"q": q, "k": s["k"], "v": s["v"]}


# ----------------------------------------------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    c, lens = case, _lens(case)
    B, kv, D = c["batch"], c["kv"], c["width"]
    if c["op"] == "attention":
        T, H = c["tokens"], c["heads"]
        out, lse = torch.zeros(B, T, H, D, dtype=torch.float64, device="cuda"), torch.empty(B, T, H, dtype=torch.float64, device="cuda")
        for b in range(B):
            n = lens[b] + T
            bits = torch.stack([(s["mask"][b] >> j) & 1 for j in range(T)], dim=1).bool()
            see = torch.cat([torch.ones(T, lens[b], dtype=torch.bool, device="cuda"), bits], dim=1)
            for h in range(kv):
                key, val = s["k"][b, h, :n].double(), s["v"][b, h, :n].double()
                for g in range(H // kv):
                    i = h * (H // kv) + g
                    z = torch.where(see, (s["q"][b, :, i].double() @ key.T) * s["scale"], -math.inf)
                    lse[b, :, i] = torch.logsumexp(z, -1)
                    out[b, :, i] = torch.softmax(z, -1) @ val
        return {"out": out, "lse": lse}
    if c["op"] == "mass":
        H, n, res = c["heads"], c["accepted"], s["out"].double()
        for b in range(B):
            res[b, :, : lens[b]] = s["mass"][b, :, : lens[b]].double()
            for i in range(n):
                r, end = int(s["rows"][b, i]), lens[b] + i + 1
                for h in range(kv):
                    hs = slice(h * (H // kv), (h + 1) * (H // kv))
                    z = (s["q"][b, r, hs].double() @ s["k"][b, h, :end].double().T) * s["scale"]
                    res[b, h, :end] += torch.exp(z - s["lse"][b, r, hs].double()[:, None]).sum(0)
        return {"mass": res}
    if c["op"] == "evict":
        ko, vo, mo = s["k_out"].double(), s["v_out"].double(), s["mass_out"].double()
        for b in range(B):
            n, keep = lens[b], min(lens[b], c["budget"])
            m = s["mass"][:, b, :, :n].double().clone()
            if n > keep:
                m[..., : c["sinks"]] = math.inf
                m[..., n - c["recent"]:] = math.inf
            best = torch.argsort(m, dim=-1, descending=True, stable=True)[..., :keep]
            best = torch.sort(best, dim=-1).values
            ko[:, b, :, :keep] = torch.take_along_dim(s["k"][:, b], best[..., None], 2).double()
            vo[:, b, :, :keep] = torch.take_along_dim(s["v"][:, b], best[..., None], 2).double()
            mo[:, b, :, :keep] = torch.take_along_dim(s["mass"][:, b], best, 2).double()
        return {"k": ko, "v": vo, "mass": mo, "kept": None, "new_lens": None}
    if c["op"] == "accept":
        k, v = s["k"].double(), s["v"].double()
        par, tok, tgt = s["parents"].tolist(), s["tokens"].tolist(), s["target"].tolist()
        for b in range(B):
            path = [0]
            while True:
                kids = [j for j in range(1, c["tokens"]) if par[b][j] == path[-1] and tok[b][j] == tgt[b][path[-1]]]
                if not kids:
                    break
                path.append(kids[0])
            src = [lens[b] + j for j in path]
            k[:, b, :, lens[b]: lens[b] + len(path)] = s["k"][:, b][:, :, src].double()
            v[:, b, :, lens[b]: lens[b] + len(path)] = s["v"][:, b][:, :, src].double()
        return {"path": None, "accepted": None, "next_token": None, "new_lens": None, "k": k, "v": v}
    T, H, half = c["tokens"], c["heads"], D // 2
    k, v, q = s["k"].double(), s["v"].double(), torch.empty(B, T, H, D, dtype=torch.float64, device="cuda")

    def turned(x, w, cos, sin):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.double()
        z = torch.complex(x[..., :half], x[..., half:]) * torch.complex(cos, sin)[:, None]
        return torch.cat([z.real, z.imag], dim=-1)

    for b in range(B):
        p = s["pos"][b].long()
        cos, sin = s["cos"][p].double(), s["sin"][p].double()
        q[b] = turned(s["xq"][b], s["q_norm"], cos, sin)
        k[b, :, lens[b]: lens[b] + T] = turned(s["xk"][b], s["k_norm"], cos, sin).transpose(0, 1)
        v[b, :, lens[b]: lens[b] + T] = s["xv"][b].double().transpose(0, 1)
    return {"q": q, "k": k, "v": v}
