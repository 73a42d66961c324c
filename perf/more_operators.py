"""The operators of serving from a paged key/value cache and of beam search on it: what is measured of them, and their plain forms.

Keys and values lie in pages [(layers,) pages, kv heads, page slots, head width]; slot s of a sequence is slot s % page of the
page that its row of `tables` names at s / page. A device array `lens` says how long the sequences are.

  append     rotate (and optionally norm) the new tokens' queries and keys, write keys and values through the tables
  attention  one new token per sequence attends to everything up to itself
  select     the best continuations of a group of beams: log-probabilities of beams x vocabulary, the n largest
  reorder    beams go on from their parents: page tables change places, started pages are copied for a second child

A case is a dict of plain values; `run` is one call. With `own` false it is the operator in elementary torch operations,
with `own` true the framework's call. `exact` is the definition in 64 bits, written on its own.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    """Head layouts, layer counts and vocabularies are those of the decoder's two architectures (32 query heads over 8 of
    128; 36 and 32 layers; 151,936 and 128,256 tokens), or generic."""
    return [
        # plain decoding at the start of a chat: nothing but latency
        {"name": "attention one sequence", "op": "attention", "type": "bf16", "batch": 1, "heads": 32, "kv": 8, "width": 128, "page": 16, "longest": 129, "shortest": 129},
        # the decoder's own 32-bit cache, four beams
        {"name": "attention 32-bit cache", "op": "attention", "type": "fp32", "batch": 4, "heads": 32, "kv": 8, "width": 128, "page": 64, "longest": 2047, "shortest": 2047},
        # a serving batch, every sequence of another length
        {"name": "attention ragged batch", "op": "attention", "type": "fp16", "batch": 64, "heads": 32, "kv": 8, "width": 128, "page": 16, "longest": 8192, "shortest": 501},
        # one long document: the length is split over the whole GPU
        {"name": "attention long document", "op": "attention", "type": "bf16", "batch": 1, "heads": 32, "kv": 8, "width": 128, "page": 64, "longest": 131000, "shortest": 131000},
        # one decoded token for each of eight sequences, queries and keys normed
        {"name": "append one token", "op": "append", "type": "fp16", "batch": 8, "tokens": 1, "heads": 32, "kv": 8, "width": 128, "page": 16, "rotary": 128, "interleaved": False, "norm": True, "longest": 777, "shortest": 30, "stretch": 1},
        # pieces of prompts of a batch, half of each head turned, in neighbouring pairs, positions stretched for a longer context
        {"name": "append pieces", "op": "append", "type": "fp32", "batch": 6, "tokens": 129, "heads": 14, "kv": 2, "width": 64, "page": 24, "rotary": 32, "interleaved": True, "norm": False, "longest": 2000, "shortest": 3, "stretch": 4},
        # a prompt
        {"name": "append prompt", "op": "append", "type": "bf16", "batch": 1, "tokens": 4099, "heads": 32, "kv": 8, "width": 128, "page": 16, "rotary": 128, "interleaved": False, "norm": False, "longest": 0, "shortest": 0, "stretch": 1},
        # four beams of one prompt
        {"name": "select four beams", "op": "select", "type": "fp32", "batch": 1, "beams": 4, "vocab": 128256, "candidates": 4, "done": 0.0, "first": False},
        # twice as many candidates as beams, an odd vocabulary, 16-bit logits
        {"name": "select odd vocabulary", "op": "select", "type": "bf16", "batch": 12, "beams": 5, "vocab": 50001, "candidates": 10, "done": 0.2, "first": False},
        # a batch of prompts, eight beams each, the largest vocabulary
        {"name": "select batch", "op": "select", "type": "fp32", "batch": 32, "beams": 8, "vocab": 151936, "candidates": 8, "done": 0.1, "first": False},
        # four beams of one prompt, all layers
        {"name": "reorder four beams", "op": "reorder", "type": "fp16", "layers": 36, "batch": 1, "beams": 4, "kv": 8, "width": 128, "page": 16, "longest": 777, "shortest": 777},
        # a batch of prompts, eight beams each, all layers, larger pages
        {"name": "reorder batch", "op": "reorder", "type": "bf16", "layers": 32, "batch": 16, "beams": 8, "kv": 8, "width": 128, "page": 32, "longest": 2047, "shortest": 100},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "select", "select", "reorder"])
    c = {"op": op, "type": rng.choice(["bf16", "fp16", "fp32"]), "batch": _log(rng, 1, 64)}
    if op == "select":
        c["beams"], c["vocab"] = _log(rng, 1, 16), _log(rng, 100, 151936)
        c["candidates"] = max(1, min(rng.choice([c["beams"], 2 * c["beams"], rng.randint(1, 32)]), c["vocab"] // 4))
        c["done"], c["first"] = rng.choice([0.0, rng.random() * 0.6]), rng.random() < 0.2
    else:
        kv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 4, 5, 7, 8, 12])
        c |= {"kv": kv, "width": rng.choice([64, 128]), "page": rng.choice([1, 8, 10, 16, 16, 24, 32, 64, 128])}
        if op == "reorder":
            c["layers"], c["beams"], c["longest"] = rng.choice([1, rng.randint(2, 36)]), rng.randint(1, 16), _log(rng, 1, 2047)
        else:
            c["heads"], c["longest"] = kv * group, _log(rng, 1, 131000 if op == "attention" else 8192)
        if op == "append":
            c["tokens"] = _log(rng, 1, 4096)
            c["rotary"], c["interleaved"], c["norm"] = rng.choice([c["width"], c["width"], c["width"] // 2, 24]), rng.random() < 0.5, rng.random() < 0.5
            c["stretch"] = rng.choice([1, 1, 4, 32])
        shorter = rng.choice([0.0, rng.random()])

    def costs():  # against the largest listed cases
        size = SIZE[c["type"]]
        if op == "select":
            return c["batch"] * c["beams"] * c["vocab"] * size / 156e6
        if op == "attention":
            return c["batch"] * c["kv"] * c["longest"] * c["width"] * size * 2 / 537e6
        if op == "append":
            return (c["batch"] * c["tokens"] * (c["heads"] + 2 * c["kv"]) * c["width"] * (4 + size) + c["batch"] * c["longest"] * 4 * c["kv"]) / 151e6
        return c["batch"] * c["beams"] * c["layers"] * c["kv"] * c["page"] * c["width"] * size / 268e6

    while costs() > 1:  # no more than the largest listed cases
        big = max((x for x in {"select": ("batch", "beams", "vocab"), "attention": ("batch", "longest"), "append": ("batch", "tokens"), "reorder": ("batch", "beams", "layers")}[op]), key=lambda x: c[x])
        c[big] = c[big] * 2 // 3
    if op == "select":
        c["candidates"] = max(1, min(c["candidates"], c["vocab"] // 4))
    else:
        c["shortest"] = int(c["longest"] * (1 - shorter))
    return c


def _lens(c):
    """The sequences' (groups') lengths: from the longest down to the shortest in even steps."""
    return [c["longest"] - (b * (c["longest"] - c["shortest"])) // max(1, c["batch"] - 1) for b in range(c["batch"])]


def work(case):
    """Each key, value, query, logit and table entry that the operator needs read once, each result written once."""
    c, e = case, SIZE[case["type"]]
    if c["op"] == "select":
        rows = c["batch"] * c["beams"]
        live = c["batch"] * (1 if c["first"] else c["beams"] * (1 - c["done"]))
        return {"bytes": live * c["vocab"] * e + rows * 5 + c["batch"] * c["candidates"] * 17, "flops": 3 * live * c["vocab"]}
    row, lens = c["width"] * e, _lens(c)
    if c["op"] == "attention":
        slots = sum(lens) + c["batch"]
        pages = sum(n // c["page"] + 1 for n in lens)
        return {"bytes": 2 * slots * c["kv"] * row + c["batch"] * c["heads"] * (2 * row + 4) + 4 * pages, "flops": 4 * c["width"] * c["heads"] * slots}
    if c["op"] == "append":
        tokens = c["batch"] * c["tokens"]
        return {"bytes": tokens * ((c["heads"] + 2 * c["kv"]) * c["width"] * (4 + e) + 4 * c["rotary"] + 4 + 4 / c["page"]), "flops": 6 * tokens * (c["heads"] + c["kv"]) * c["width"]}
    W = c["beams"]
    further = W * (1 - 1 / W) ** W if W > 1 else 0  # beams without a child, of parents drawn evenly: as many second children
    return {"bytes": sum(W * (8 * (n // c["page"]) + 4) + further * (n % c["page"]) * c["layers"] * c["kv"] * 4 * row for n in lens), "flops": 0}


# ------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt, B = TYPES[c["type"]], c["batch"]

    def normal(*shape, scale=1.0, dtype=dt):
        return torch.randn(*shape, device="cuda", generator=g, dtype=dtype) * scale

    s = {"case": c}
    if c["op"] == "select":
        W, V, n = c["beams"], c["vocab"], c["candidates"]
        # a few likely tokens in front of many, some forbidden ones
        s["logits"] = normal(B, 1 if c["first"] else W, V, scale=2.5)
        u = torch.rand(V, device="cuda", generator=g)
        s["logits"] += (3 * u.pow(12)).to(dt)
        s["logits"].masked_fill_(torch.rand(B, 1, V, device="cuda", generator=g) < 0.01, -math.inf)
        s["logits"] = s["logits"].expand(B, W, V)
        s["scores"] = -torch.sort(torch.rand(B, W, device="cuda", generator=g), dim=1).values * 4 - 20
        s["done"] = torch.rand(B, W, device="cuda", generator=g) < c["done"]
        if c["first"]:  # one beam is all there is
            s["scores"][:, 0], s["scores"][:, 1:] = 0, -math.inf
            s["done"].fill_(False)
        s["end"] = V // 2
        s["res"] = {"out_scores": torch.empty(B, n, device="cuda"), "parents": torch.empty(B, n, dtype=torch.int32, device="cuda"),
                    "tokens": torch.empty(B, n, dtype=torch.int64, device="cuda"), "out_done": torch.empty(B, n, dtype=torch.bool, device="cuda")}
        return s
    kv, D, P = c["kv"], c["width"], c["page"]
    lens = _lens(c)
    if c["op"] == "reorder":
        W, N = c["beams"], c["layers"]
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda").repeat_interleave(W)
        cols = c["longest"] // P + 2
        pages = B * W + 32
        s["k"], s["v"] = normal(N, pages, kv, P, D), normal(N, pages, kv, P, D)
        s["parents"] = torch.randint(0, W, (B, W), dtype=torch.int32, device="cuda", generator=g)
        # every beam has a started page of its own; which the full ones are is nothing to the operator
        s["tables"] = torch.randint(0, pages, (B * W, cols), dtype=torch.int32, device="cuda", generator=g)
        started = torch.randperm(pages, device="cuda", generator=g)[: B * W].int()
        s["tables"].scatter_(1, (s["lens"] // P).long()[:, None], started[:, None])
        return s
    T = c.get("tokens", 1)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    need = [(n + T - 1) // P + 1 for n in lens]
    cols = max(need) + 2
    pages = sum(need) + 5
    order = torch.randperm(pages, device="cuda", generator=g).int()
    s["tables"] = torch.full((B, cols), -1, dtype=torch.int32, device="cuda")  # pages that a sequence does not have yet
    at = 0
    for b, n in enumerate(need):
        s["tables"][b, :n] = order[at: at + n]
        at += n
    H = c["heads"]
    if c["op"] == "attention":
        s["k"], s["v"] = normal(pages, kv, P, D), normal(pages, kv, P, D)
        s["k"] += normal(kv, 1, D, scale=0.5)  # keys share a direction
        s["q"] = normal(B, H, D, scale=1.5)
        s["scale"] = 1.0 / math.sqrt(D)
        s["out"], s["lse"] = torch.empty_like(s["q"]), torch.empty(B, H, device="cuda")
        return s
    x = normal(B * T, (H + 2 * kv) * D, dtype=torch.float32)  # the projections' outputs, one behind the other
    s["xq"], s["xk"], s["xv"] = (y.unflatten(1, (-1, D)).unflatten(0, (B, T)) for y in x.split([H * D, kv * D, kv * D], dim=1))
    s["k"], s["v"] = (torch.zeros(pages, kv, P, D, dtype=dt, device="cuda") for _ in range(2))
    s["pos"] = s["lens"][:, None] + torch.arange(T, dtype=torch.int32, device="cuda")
    R = c["rotary"]
    angle = torch.arange(c["longest"] + T, dtype=torch.float64, device="cuda")[:, None] / c["stretch"] * 1e6 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
    s["cos"], s["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
    s["q_norm"], s["k_norm"] = (normal(D, scale=0.1, dtype=torch.float32) + 1 if c["norm"] else None for _ in range(2))
    s["q_out"] = torch.empty(B, T, H, D, dtype=dt, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------------- plain forms
def _attention(s):
    q, P = s["q"], s["k"].shape[2]
    B, H, D = q.shape
    kv = s["k"].shape[1]
    take = s["tables"].clamp(min=0).long()
    flat = lambda x: x[take].transpose(1, 2).reshape(B, kv, -1, D).float()  # noqa: E731
    x = (q.float().reshape(B, kv, H // kv, D) @ flat(s["k"]).transpose(-1, -2)).mul_(s["scale"])
    at = torch.arange(take.shape[1] * P, device="cuda")
    x.masked_fill_(at > s["lens"][:, None, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p @ flat(s["v"])) / total
    return {"out": o.reshape(B, H, D).to(q.dtype), "lse": (top + total.log()).reshape(B, H)}


def _append(s):
    lens, pos, T = s["lens"].long(), s["pos"].long(), s["pos"].shape[1]
    P, R, spread = s["k"].shape[2], 2 * s["cos"].shape[1], s["case"]["interleaved"]

    def turn(x, w):
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        x, rest = x[..., :R], x[..., R:]
        a, b = (x[..., ::2], x[..., 1::2]) if spread else x.chunk(2, dim=-1)
        cos, sin = s["cos"][pos][:, :, None], s["sin"][pos][:, :, None]
        y = (a * cos - b * sin, b * cos + a * sin)
        return torch.cat([torch.stack(y, dim=-1).flatten(-2) if spread else torch.cat(y, dim=-1), rest], dim=-1)

    slot = lens[:, None] + torch.arange(T, device="cuda")
    page = s["tables"].long().gather(1, slot // P)
    s["k"][page, :, slot % P] = turn(s["xk"], s["k_norm"]).to(s["k"].dtype)
    s["v"][page, :, slot % P] = s["xv"].to(s["k"].dtype)
    return {"q": turn(s["xq"], s["q_norm"]).to(s["k"].dtype), "k": s["k"], "v": s["v"]}


def _select(s):
    """in 64 bits: two beams' continuations may be as near to one another as they like"""
    x, n, done = s["logits"].double(), s["case"]["candidates"], s["done"][..., None]
    B, W, V = x.shape
    top = x.amax(-1, keepdim=True)
    p = s["scores"].double()[..., None] + (x - (top + (x - top).exp_().sum(-1, keepdim=True).log()))
    p.masked_fill_(done, -math.inf)
    p[..., s["end"]] = torch.where(done[..., 0], s["scores"].double(), p[..., s["end"]])
    best, at = torch.sort(p.reshape(B, W * V), dim=-1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    live = best > -math.inf
    parents, tokens = torch.where(live, at // V, -1), torch.where(live, at % V, -1)
    return {"out_scores": best.float(), "parents": parents.int(), "tokens": tokens, "out_done": tokens == s["end"]}


def _reorder(s):
    k, v, tables = s["k"], s["v"], s["tables"]
    B, W = s["parents"].shape
    N, _, kv, P, D = k.shape
    parents = s["parents"].long()
    old = tables.reshape(B, W, -1)
    n = s["lens"].reshape(B, W)[:, :1].long()
    full, rest = n // P, n % P
    same = parents[:, :, None] == parents[:, None, :]
    further = (same & torch.tril(torch.ones(W, W, dtype=torch.bool, device="cuda"), -1)).any(-1)  # a lower beam has the same parent
    childless = ~(parents[:, :, None] == torch.arange(W, device="cuda")).any(1)
    started = old.gather(2, full[:, :, None].expand(B, W, 1))[..., 0]
    free = torch.where(childless, torch.arange(W, device="cuda"), W).sort(-1).values.clamp(max=W - 1)  # beams without children first
    spare = started.gather(1, free).gather(1, (further.cumsum(-1) - 1).clamp(min=0))  # one for each further child, in order
    own_page = torch.where(further, spare, started.gather(1, parents))
    own_page = torch.where(rest > 0, own_page, started)
    src = torch.where(further & (rest > 0), started.gather(1, parents), own_page).reshape(-1).long()
    dst = own_page.reshape(-1).long()
    keep = (torch.arange(P, device="cuda") < rest).repeat_interleave(W, 0)[None, :, None, :, None]
    for x in (k, v):
        x[:, dst] = torch.where(keep, x[:, src], x[:, dst])
    col = torch.arange(old.shape[2], device="cuda")
    new = torch.where(col < full[:, :, None], old.gather(1, parents[:, :, None].expand_as(old)), torch.where(col == full[:, :, None], own_page[:, :, None], old))
    tables.copy_(new.reshape(tables.shape))
    return {"tables": tables, "k": k, "v": v}


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"attention": _attention, "append": _append, "select": _select, "reorder": _reorder}[op](s)
    from pingala8_llm_b200 import paged

    if op == "attention":
        out, lse = paged.paged_attention(s["q"], s["k"], s["v"], s["tables"], s["lens"], scale=s["scale"], out=s["out"], lse=s["lse"])
        return {"out": out, "lse": lse}
    if op == "append":
        q = paged.paged_append(s["xq"], s["xk"], s["xv"], s["k"], s["v"], s["tables"], s["lens"], s["pos"], s["cos"], s["sin"], interleaved=s["case"]["interleaved"], q_norm=s["q_norm"],
                               k_norm=s["k_norm"], eps=1e-6, q_out=s["q_out"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    if op == "select":
        paged.beam_select(s["logits"], s["scores"], done=s["done"], end=s["end"], candidates=s["case"]["candidates"], **s["res"])
        return s["res"]
    paged.beam_reorder(s["parents"], s["k"], s["v"], s["tables"], s["lens"])
    return {"tables": s["tables"], "k": s["k"], "v": s["v"]}


# ----------------------------------------------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    c = case
    B, lens = c["batch"], None if c["op"] == "select" else _lens(c)
    if c["op"] == "attention":
        H, kv, D, P = c["heads"], c["kv"], c["width"], c["page"]
        out, lse = torch.zeros(B, H, D, dtype=torch.float64, device="cuda"), torch.empty(B, H, dtype=torch.float64, device="cuda")
        for b in range(B):
            n = lens[b] + 1
            ids = s["tables"][b, : (n + P - 1) // P].long()
            for h in range(kv):
                key, val = s["k"][ids, h].reshape(-1, D)[:n].double(), s["v"][ids, h].reshape(-1, D)[:n].double()
                hs = slice(h * (H // kv), (h + 1) * (H // kv))
                z = (s["q"][b, hs].double() @ key.T) * s["scale"]
                lse[b, hs] = torch.logsumexp(z, -1)
                out[b, hs] = torch.softmax(z, -1) @ val
        return {"out": out, "lse": lse}
    if c["op"] == "select":
        res = torch.full((B, c["candidates"]), -math.inf, dtype=torch.float64, device="cuda")
        for b in range(B):
            every = []
            for w in range(c["beams"]):
                score = s["scores"][b, w].double()
                if bool(s["done"][b, w]):
                    every.append(score[None])
                elif math.isfinite(float(score)):
                    every.append(score + torch.topk(torch.log_softmax(s["logits"][b, w].double(), -1), c["candidates"]).values)
            best = torch.sort(torch.cat(every), descending=True).values[: c["candidates"]]
            res[b, : len(best)] = best
        return {"out_scores": res, "parents": None, "tokens": None, "out_done": None}
    if c["op"] == "append":
        T, H, D, P, R = c["tokens"], c["heads"], c["width"], c["page"], c["rotary"]
        k, v, q = s["k"].double(), s["v"].double(), torch.empty(B, T, H, D, dtype=torch.float64, device="cuda")

        def turned(x, w, cos, sin):
            x = x.double()
            if w is not None:
                x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.double()
            first, second = (slice(0, R, 2), slice(1, R, 2)) if c["interleaved"] else (slice(0, R // 2), slice(R // 2, R))
            z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * torch.complex(cos, sin)[:, None]
            y = x.clone()
            y[..., first], y[..., second] = z.real, z.imag
            return y

        for b in range(B):
            p = s["pos"][b].long()
            cos, sin = s["cos"][p].double(), s["sin"][p].double()
            slot = lens[b] + torch.arange(T, device="cuda")
            page = s["tables"][b, slot // P].long()
            q[b] = turned(s["xq"][b], s["q_norm"], cos, sin)
            k[page, :, slot % P] = turned(s["xk"][b], s["k_norm"], cos, sin)
            v[page, :, slot % P] = s["xv"][b].double()
        return {"q": q, "k": k, "v": v}
    W, P = c["beams"], c["page"]
    k, v, parents, tables = s["k"].double(), s["v"].double(), s["parents"].tolist(), s["tables"].tolist()
    for b in range(B):
        full, rest = lens[b] // P, lens[b] % P
        if not rest:
            continue
        page = [tables[b * W + w][full] for w in range(W)]
        free = [page[w] for w in range(W) if w not in parents[b]]
        taken = set()
        for w in range(W):
            if parents[b][w] in taken:
                to = free.pop(0)
                k[:, to, :, :rest] = s["k"][:, page[parents[b][w]], :, :rest].double()
                v[:, to, :, :rest] = s["v"][:, page[parents[b][w]], :, :rest].double()
            taken.add(parents[b][w])
    return {"tables": None, "k": k, "v": v}
