"""Paged cache and beam search operators against their definitions in 64 bits.

Tolerances. u = eps / 2 is the error of one rounding to the tensors' type, e = 2^-24 that of one fp32 rounding (2 e where a tensor core
may cut).
  append: a norm is off by a factor 1 +- (D + 12) e (a sum of D squares in any order, division, root, two products), a turned
    pair by 3 e more of |x0 c| + |x1 s|; then u of the result.
  attention: a score is a dot product of D terms: off by at most ds = 2 (D + 16) e A, A = scale max |q||k| (16: scale, exponent's
    argument); its exponential by a factor 1 +- 2 ds (its own score's and the reference's). 4 e for the exponential; weights go in as two cut pieces:
    2^-14 (bf16), 2^-20 (fp16), nothing (fp32). Sums of L terms with independent errors: 16 sqrt(L) e, 128 e for the joining of
    lanes, warps and parts. So
        |o - o*| <= (w + 2 ds + (132 + 16 sqrt(L)) e) sum p |v| + u |o*|,    |lse - lse*| <= ds + (132 + 16 sqrt(L)) e + 2 e |lse*|
  selection: the log of a sum of positive terms; a term 2^a (a <= 0) is off by a factor 1 +- (4 + 2 |a|) e (argument, exponential), and the weighted mean of
    |a| is at most log2 V; sums of 16, of a lane's rounds and of 512 lanes and pieces add (16 + V / 4096 + 30) e. So a total is off by
    (50 + 2 log2 V + V / 4096) e, and e of itself for its rounding to fp32. Parents and tokens have to be equal.
Moved rows and tables have to be equal.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

import pingala8_llm_b200 as p8  # noqa: E402
from pingala8_llm_b200 import paged  # noqa: E402

E = 2.0 ** -24
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
INF, NAN = math.inf, math.nan


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def ended(bits=0):
    torch.cuda.synchronize()
    assert p8.device_error() == bits


def close(got, want, tol, what=""):
    got = got.double()
    odd = ~torch.isfinite(want)
    assert torch.equal(got[odd], want[odd]), what
    assert not torch.isnan(got).any(), what
    d = (got - want)[~odd].abs() - tol[~odd]
    assert d.numel() == 0 or float(d.max()) <= 0, f"{what}: {float(d.max())} over the bound"


def make_pages(g, pages, kv, page, D, dtype, layout="heads", fill=None):
    """k, v [pages, kv, page, D]; "slots": slots before heads in memory; "pair": keys and values of a page side by side"""
    shape = (pages, kv, page, D)
    if layout == "slots":
        out = [randn(g, pages, page, kv, D, dtype=dtype).transpose(1, 2) for _ in range(2)]
    elif layout == "pair":
        both = randn(g, pages, 2, kv, page, D, dtype=dtype)
        out = [both[:, 0], both[:, 1]]
    else:
        out = [randn(g, *shape, dtype=dtype) for _ in range(2)]
    if fill is not None:
        for x in out:
            x.fill_(fill)
    return out


def make_tables(g, lens, extra, page, pages, spare=2):
    """every sequence its own pages, in any order; entries behind them are no pages"""
    need = [(n + extra + page - 1) // page for n in lens]
    assert sum(need) <= pages
    order = torch.randperm(pages, device="cuda", generator=g).int()
    t = torch.full((len(lens), max(need) + spare), -7, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n]
        at += n
    return t


# ------------------------------------------------------------------------------------------------------------ append
def append_ref(q, k, v, kp, vp, tables, lens, pos, cos, sin, interleaved, qn, kn, eps, counts):
    """(queries, keys, values, their bounds) in 64 bits, the pages whole"""
    B, T, H, D = q.shape
    R, P = 2 * cos.shape[1], kp.shape[2]
    u = torch.finfo(kp.dtype).eps / 2 if kp.dtype != torch.float32 else E

    def turn(x, w, p):
        x = x.double()
        rel = 0.0
        if w is not None:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
            rel = (D + 12) * E
        c, s = cos[p].double()[:, None], sin[p].double()[:, None]
        i0, i1 = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
        y, size = x.clone(), x.abs()
        y[..., i0], y[..., i1] = x[..., i0] * c - x[..., i1] * s, x[..., i1] * c + x[..., i0] * s
        size[..., i0], size[..., i1] = (x[..., i0] * c).abs() + (x[..., i1] * s).abs(), (x[..., i1] * c).abs() + (x[..., i0] * s).abs()
        return y, (rel + 3 * E) * size * (1 + 2 * u) + u * y.abs() + torch.finfo(kp.dtype).tiny

    qo, qt = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    ko, vo = kp.double().clone(), vp.double().clone()
    kt, vt = torch.zeros_like(ko), torch.zeros_like(vo)
    for b in range(B):
        for t in range(T if counts is None else int(counts[b])):
            p, s = int(pos[b, t]), int(lens[b]) + t
            qo[b, t], qt[b, t] = (x[0] for x in turn(q[b, t][None], qn, [p]))
            at, r = int(tables[b, s // P]), s % P
            ky, kb = turn(k[b, t][None], kn, [p])
            ko[at, :, r], kt[at, :, r] = ky[0], kb[0]
            vo[at, :, r] = v[b, t].double()
            vt[at, :, r] = u * v[b, t].double().abs() + torch.finfo(kp.dtype).tiny
    return qo, ko, vo, qt, kt, vt


# type, D, page, R, interleaved, norm, T, H, kv, lens, counts, layout
APPENDS = [
    ("fp32", 64, 1, 64, False, False, 1, 1, 1, [0], None, "heads"),
    ("fp16", 128, 16, 128, False, True, 1, 32, 8, [15, 16, 777], None, "heads"),
    ("bf16", 128, 16, 64, True, True, 5, 8, 2, [14, 0, 31], [5, 0, 3], "slots"),
    ("fp32", 64, 24, 32, True, False, 33, 14, 2, [7, 23], None, "pair"),
    ("bf16", 64, 7, 8, False, True, 20, 6, 3, [1, 60], [20, 19], "pair"),
    ("fp16", 128, 10, 24, True, False, 3, 5, 5, [9, 10, 11, 0, 100], None, "slots"),
    ("fp32", 128, 64, 120, False, True, 130, 4, 1, [63], None, "heads"),
    ("bf16", 128, 1000, 128, True, False, 70, 9, 3, [0, 930], None, "heads"),
]


@pytest.mark.parametrize("case", APPENDS)
def test_append(case):
    name, D, page, R, inter, norm, T, H, kv, lens_, counts_, layout = case
    g, dt, B = gen(hash(case[1:9]) % 1000), TYPES[name], len(lens_)
    pages = sum((n + T + page - 1) // page for n in lens_) + 3
    kp, vp = make_pages(g, pages, kv, page, D, dt, layout)
    tables = make_tables(g, lens_, T, page, pages)
    lens, counts = ints(*lens_), None if counts_ is None else ints(*counts_)
    x = randn(g, B, T, (H + 2 * kv) * D)
    q, k, v = (y.unflatten(2, (-1, D)) for y in x.split([H * D, kv * D, kv * D], dim=2))
    cos, sin = paged.rotary_tables(1100, R, 1e4, device="cuda")
    pos = torch.randint(0, 1100, (B, T), dtype=torch.int32, device="cuda", generator=g)
    qn, kn = (randn(g, D) if norm else None for _ in range(2))
    want = append_ref(q, k, v, kp, vp, tables, lens, pos, cos, sin, inter, qn, kn, 1e-6, counts)
    out = paged.paged_append(q, k, v, kp, vp, tables, lens, pos, cos, sin, interleaved=inter, q_norm=qn, k_norm=kn, counts=counts)
    ended()
    for got, y, t, what in ((out, want[0], want[3], "q"), (kp, want[1], want[4], "k"), (vp, want[2], want[5], "v")):
        close(got, y, t, what)  # what was not written included: its bound is nothing


def test_append_in_place_and_into_a_given_tensor():
    g = gen(3)
    kp, vp = make_pages(g, 6, 2, 8, 64, torch.float32)
    tables, lens, pos = make_tables(g, [5, 11], 3, 8, 6), ints(5, 11), torch.arange(6, dtype=torch.int32, device="cuda").view(2, 3)
    q, k, v = randn(g, 2, 3, 4, 64), randn(g, 2, 3, 2, 64), randn(g, 2, 3, 2, 64)
    cos, sin = paged.rotary_tables(6, 64, device="cuda")
    a = paged.paged_append(q, k, v, kp, vp, tables, lens, pos, cos, sin)
    q2, k2, v2 = q.clone(), kp.clone(), vp.clone()
    assert paged.paged_append(q2, k, v, k2, v2, tables, lens, pos, cos, sin, q_out=q2) is q2
    wide = torch.zeros(2, 3, 9, 64, device="cuda")
    paged.paged_append(q, k, v, k2, v2, tables, lens, pos, cos, sin, q_out=wide[:, :, 2:6])
    ended()
    assert torch.equal(a, q2) and torch.equal(a, wide[:, :, 2:6]) and torch.equal(kp, k2) and float(wide[:, :, :2].abs().max()) == 0


def test_append_leaves_out_what_is_out_of_range():
    g = gen(4)
    cos, sin = paged.rotary_tables(40, 64, device="cuda")

    def call(lens_, tables_, pos_, counts_=None, T=2):
        kp, vp = make_pages(g, 5, 2, 4, 64, torch.bfloat16)
        k0, v0 = kp.clone(), vp.clone()
        B = len(lens_)
        q, k, v = randn(g, B, T, 2, 64), randn(g, B, T, 2, 64), randn(g, B, T, 2, 64)
        out = torch.full((B, T, 2, 64), 5.0, dtype=torch.bfloat16, device="cuda")
        paged.paged_append(q, k, v, kp, vp, torch.tensor(tables_, dtype=torch.int32, device="cuda"), ints(*lens_), torch.tensor(pos_, dtype=torch.int32, device="cuda"), cos, sin,
                           counts=None if counts_ is None else ints(*counts_), q_out=out)
        torch.cuda.synchronize()
        err = p8.device_error()
        return err, (kp != k0).flatten(2).any(-1), out

    ok = [[0, 1, 2], [3, 4, 2]]
    for lens_ in ([-1, 2], [11, 2], [-2 ** 31, 2], [2 ** 31 - 1, 2]):
        err, wrote, out = call(lens_, ok, [[0, 1], [2, 3]])
        assert err == 64 and not wrote[:3].any() and float(out[0].float().min()) == 5 and wrote[3].any() and wrote[4].sum() == 0
    err, wrote, out = call([0, 2], ok, [[0, 40], [-1, 3]])  # positions: one token of each
    assert err == 64 and float(out[0, 1].float().min()) == 5 and float(out[1, 0].float().min()) == 5 and float(out[0, 0].float().min()) < 5
    for bad in (5, -1, -2 ** 31, 2 ** 31 - 1):  # pages: the second token's
        err, wrote, out = call([3, 1], [[0, bad, 1], [3, 4, 2]], [[0, 1], [2, 3]])
        assert err == 64 and wrote[0].all() and not wrote[1:3].any() and wrote[3].all() and not wrote[4].any()
    err, wrote, out = call([3, 1], ok, [[0, 1], [2, 3]], counts_=[3, 1])
    assert err == 64 and not wrote[:3].any() and wrote[3].all()
    err, wrote, out = call([3, 1], [[0, -1, -1], [3, -1, -1]], [[0, -9], [2, 99]], counts_=[1, 0])  # behind the counts nothing is looked at
    assert err == 0 and wrote[0].all() and not wrote[1:].any()


# --------------------------------------------------------------------------------------------------------- attention
def attend(q, kp, vp, tables, lens, counts, scale):
    """(o, lse, bounds); slots of pages that are out of range count as not there; None where a row has no token"""
    B, H, D = q.shape
    kv, P = kp.shape[1], kp.shape[2]
    G = H // kv
    o, lse = torch.zeros(B, H, D, dtype=torch.float64, device="cuda"), torch.full((B, H), -INF, dtype=torch.float64, device="cuda")
    to, tl = torch.zeros_like(o), torch.zeros_like(lse)
    u = torch.finfo(q.dtype).eps / 2
    w = {torch.float32: 0.0, torch.float16: 2.0 ** -20, torch.bfloat16: 2.0 ** -14}[q.dtype]
    for b in range(B):
        if counts is not None and int(counts[b]) == 0:
            continue
        n = int(lens[b]) + 1
        slot = torch.arange(n, device="cuda")
        at = tables[b].long()[slot // P]
        live = (at >= 0) & (at < kp.shape[0])
        at, slot = at[live], slot[live] % P
        if not at.numel():
            continue
        acc = (132 + 16 * math.sqrt(at.numel())) * E
        for h in range(kv):
            K, V = kp[at, h, slot].double(), vp[at, h, slot].double()
            x = q[b, h * G:(h + 1) * G].double()
            s = x @ K.T * scale
            lse[b, h * G:(h + 1) * G] = torch.logsumexp(s, -1)
            p = torch.softmax(s, -1)
            y = p @ V
            o[b, h * G:(h + 1) * G] = y
            ds = 2 * (D + 16) * E * (x.abs() @ K.abs().T).amax(-1, keepdim=True) * abs(scale)
            to[b, h * G:(h + 1) * G] = (w + 2 * ds + acc) * (p @ V.abs()) + u * y.abs() + torch.finfo(q.dtype).tiny
            tl[b, h * G:(h + 1) * G] = (ds[:, 0] + acc) + 2 * E * lse[b, h * G:(h + 1) * G].abs()
    return o, lse, to, tl


# H, kv, D, page, lens, layout: lengths on either side of tiles (8, 16), pages, shares (128) and CTAs
ATTENTIONS = [
    (1, 1, 64, 1, [0], "heads"),
    (4, 4, 128, 16, [0, 1, 6, 7, 8], "heads"),
    (32, 8, 128, 16, [14, 15, 16, 17], "pair"),
    (5, 1, 64, 24, [126, 127, 128, 129], "slots"),
    (7, 1, 128, 10, [300, 0, 55], "heads"),
    (14, 2, 64, 7, [1000, 999], "pair"),
    (9, 1, 128, 32, [511, 77], "heads"),
    (24, 2, 128, 16, [255, 600, 3], "slots"),
    (40, 2, 64, 8, [90, 400], "heads"),
    (66, 2, 128, 16, [200], "heads"),
    (8, 8, 64, 128, [4000], "heads"),
    (32, 8, 128, 64, [20011], "pair"),
    (3, 3, 128, 1000, [2500, 999, 1000, 1], "slots"),
    (16, 4, 128, 3, [40 * i for i in range(37)], "heads"),
    (2, 1, 64, 16, [17 * (i % 9) for i in range(700)], "heads"),
]


@pytest.mark.parametrize("name", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("case", ATTENTIONS)
def test_attention(name, case):
    H, kv, D, page, lens_, layout = case
    g, dt = gen(H * 100 + D), TYPES[name]
    pages = sum((n + 1 + page - 1) // page for n in lens_) + 2
    kp, vp = make_pages(g, pages, kv, page, D, dt, layout)
    tables, lens, q = make_tables(g, lens_, 1, page, pages), ints(*lens_), randn(g, len(lens_), H, D, dtype=dt, scale=1.5)
    # what lies behind the sequences is nobody's business
    used = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens_):
        s = torch.arange(n + 1, device="cuda")
        used[tables[b].long()[s // page], s % page] = True
    hole = ~used[:, None, :, None].expand(kp.shape)
    kp[hole], vp[hole] = NAN, INF
    want = attend(q, kp, vp, tables, lens, None, D ** -0.5)
    out, lse = paged.paged_attention(q, kp, vp, tables, lens)
    ended()
    close(out, want[0], want[2], "out")
    close(lse, want[1], want[3], "lse")
    again, lse2 = paged.paged_attention(q, kp, vp, tables, lens)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


# H, kv, page, lens: heads of 128 whose rows come in blocks, in tables that are longer than the sequences (the eight warps' form),
# with lengths on either side of its tiles, rounds and shares, rows without a token and pages that are not there
@pytest.mark.parametrize("name", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("H,kv,page,lens_", [(32, 8, 16, [0, 15, 16, 127, 128, 129, 383, 384, 385, 2000]), (4, 4, 4, [3 * i for i in range(300)]), (16, 2, 64, [9000, 1, 191, 192]), (1, 1, 8, [30000])])
def test_attention_in_long_tables(name, H, kv, page, lens_):
    g, dt = gen(H + page), TYPES[name]
    pages = sum((n + page) // page for n in lens_) + 2
    kp, vp = make_pages(g, pages, kv, page, 128, dt)
    B, columns = len(lens_), (max(lens_) + page) // page + 3000 // page
    tables = torch.full((B, columns), -1, dtype=torch.int32, device="cuda")
    short = make_tables(g, lens_, 1, page, pages)
    tables[:, :short.shape[1]] = short
    lens, q = ints(*lens_), randn(g, B, H, 128, dtype=dt, scale=1.5)
    counts = torch.ones(B, dtype=torch.int32, device="cuda")
    if B > 1:
        counts[B // 2] = 0
        tables[0, 0], tables[B - 1, 0] = pages, -7  # all of a sequence of one page, and a beginning
    want = attend(q, kp, vp, tables, lens, counts, 128 ** -0.5)
    out, lse = paged.paged_attention(q, kp, vp, tables, lens, counts=counts)
    ended(64 if B > 1 else 0)
    live = counts.bool()
    close(out[live], want[0][live], want[2][live], "out")
    close(lse[live], want[1][live], want[3][live], "lse")
    assert not out[~live].any() and not lse[~live].any()
    again, lse2 = paged.paged_attention(q, kp, vp, tables, lens, counts=counts)
    ended(64 if B > 1 else 0)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("name", ["fp32", "fp16", "bf16"])
def test_attention_rows_without_a_token_and_pages_out_of_range(name):
    g, dt = gen(8), TYPES[name]
    kp, vp = make_pages(g, 12, 2, 16, 64, dt)
    tables = torch.tensor([[0, 1, 2, 3], [4, -1, 5, 99], [-1, 12, -2 ** 31, 2 ** 31 - 1], [6, 7, 8, 9], [10, 11, 0, 1]], dtype=torch.int32, device="cuda")
    lens, q = ints(40, 50, 63, 20, 5), randn(g, 5, 6, 64, dtype=dt)
    out, lse = torch.full((5, 6, 64), 3.0, dtype=dt, device="cuda"), torch.full((5, 6), 4.0, device="cuda")
    counts = ints(1, 1, 1, 0, 1)
    want = attend(q, kp, vp, tables, lens, counts, 0.3)
    paged.paged_attention(q, kp, vp, tables, lens, counts=counts, scale=0.3, out=out, lse=lse)
    ended(64)
    live = [0, 1, 2, 4]
    close(out[live], want[0][live], want[2][live], "out")
    close(lse[live], want[1][live], want[3][live], "lse")
    assert float(out[2].float().abs().max()) == 0 and float(lse[2].max()) == -INF  # nothing of it is there
    assert float(out[3].float().min()) == 3 == float(out[3].float().max()) and float(lse[3].min()) == 4
    for bad in ([-1, 3], [64, 3], [-2 ** 31, 3], [2 ** 31 - 1, 3]):  # lengths: the row is left alone
        out.fill_(3.0)
        paged.paged_attention(q[:2], kp, vp, tables[[0, 3]].contiguous(), ints(*bad), out=out[:2], lse=lse[:2])
        ended(64)
        assert float(out[0].float().min()) == 3 == float(out[0].float().max()) and float((out[1].float() - 3).abs().max()) > 0
    for counts_ in ([2, 1], [-1, 1]):
        out.fill_(3.0)
        paged.paged_attention(q[:2], kp, vp, tables[[0, 3]].contiguous(), ints(40, 3), counts=ints(*counts_), out=out[:2], lse=lse[:2])
        ended(64)
        assert float(out[0].float().min()) == 3 == float(out[0].float().max()) and float((out[1].float() - 3).abs().max()) > 0


@pytest.mark.parametrize("name", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("how", ["rising", "falling", "one", "flat", "large", "negative scale", "no scale"])
def test_attention_scores_of_all_kinds(name, how):
    """maxima that move often or never, one slot that takes all, far tails, scores of one size, thousands"""
    g, dt, n, D = gen(9), TYPES[name], 3000, 128
    kp, vp = make_pages(g, (n + 15) // 16, 1, 16, D, dt)
    tables = torch.arange(kp.shape[0], dtype=torch.int32, device="cuda")[None].contiguous()
    q = randn(g, 1, 4, D, dtype=dt)
    scale = {"negative scale": -0.2, "no scale": 0.0}.get(how, D ** -0.5)
    ramp = torch.linspace(0, 40, n + 8 & ~15 if False else kp.shape[0] * 16, device="cuda").view(-1, 16)
    dirn = q[0, 0].float() / q[0, 0].float().norm() ** 2 * D ** 0.5
    if how in ("rising", "falling"):
        r = ramp if how == "rising" else 40 - ramp
        kp[:, 0] = (r[..., None] * dirn).to(dt)
    elif how == "one":
        kp[77, 0, 3] = (60 * dirn).to(dt)
    elif how == "flat":
        kp.zero_()
    elif how == "large":
        kp *= 50
    lens = ints(n - 1)
    want = attend(q, kp, vp, tables, lens, None, scale)
    out, lse = paged.paged_attention(q, kp, vp, tables, lens, scale=scale)
    ended()
    close(out, want[0], want[2], "out")
    close(lse, want[1], want[3], "lse")


@pytest.mark.parametrize("name", ["fp32", "fp16", "bf16"])
def test_attention_infinities_that_are_seen(name):
    g, dt = gen(10), TYPES[name]
    kp, vp = make_pages(g, 8, 1, 16, 64, dt)
    tables, lens, q = torch.arange(8, dtype=torch.int32, device="cuda")[None].contiguous(), ints(100), randn(g, 1, 3, 64, dtype=dt)
    vp[2, 0, 5, 7], vp[3, 0, 0, 9], vp[1, 0, 1, 20] = INF, -INF, NAN
    out, lse = paged.paged_attention(q, kp, vp, tables, lens)
    ended()
    assert (out[0, :, 7] == INF).all() and (out[0, :, 9] == -INF).all() and torch.isnan(out[0, :, 20]).all()
    rest = [d for d in range(64) if d not in (7, 9, 20)]
    assert torch.isfinite(out[0][:, rest]).all() and torch.isfinite(lse).all()
    kp[4, 0, 0, 0] = NAN
    out, lse = paged.paged_attention(q, kp, vp, tables, lens)
    ended()
    assert torch.isnan(out).all() and torch.isnan(lse).all()


def test_attention_strides_broadcasts_and_shared_pages():
    """queries and outputs as slices, one table for all rows, lengths of their own: the tokens of a prompt, each over what is before it"""
    g, n, D = gen(11), 50, 128
    kp, vp = make_pages(g, 7, 2, 8, D, torch.float16)
    table = torch.randperm(7, device="cuda", generator=g).int()[None].expand(n, 7)
    wide = randn(g, n, 11, D, dtype=torch.float16)
    q, lens = wide[:, 2:10], torch.arange(n, dtype=torch.int32, device="cuda")
    out = torch.zeros(8, n, D, dtype=torch.float16, device="cuda").transpose(0, 1)
    lse = torch.empty(n, 8, device="cuda")
    want = attend(q, kp, vp, table, lens, None, D ** -0.5)
    paged.paged_attention(q, kp, vp, table, lens, out=out, lse=lse)
    ended()
    close(out, want[0], want[2], "out")
    close(lse, want[1], want[3], "lse")


def test_offsets_beyond_32_bits():
    """pages whose places in memory are more than 2^32 bytes apart, for all three that touch them"""
    g, D = gen(12), 64
    big = torch.zeros(3 * (5 << 30) // 2, dtype=torch.float16, device="cuda")
    kp = torch.as_strided(big, (3, 2, 8, D), ((5 << 30) // 2, 8 * D, D, 1))
    vp = torch.as_strided(big, (3, 2, 8, D), ((5 << 30) // 2, 8 * D, D, 1), storage_offset=4 * 8 * D)
    for x in (kp, vp):
        x.copy_(randn(g, 3, 2, 8, D, dtype=torch.float16))
    tables, lens = ints(2, 0, 1, 2, 1, 0).view(2, 3), ints(20, 20)
    cos, sin = paged.rotary_tables(30, D, device="cuda")
    q, k, v = randn(g, 2, 1, 4, D), randn(g, 2, 1, 2, D), randn(g, 2, 1, 2, D)
    tables = ints(2, 0, 1).view(1, 3)
    want = append_ref(q[:1], k[:1], v[:1], kp, vp, tables, lens[:1], lens[:1, None], cos, sin, False, None, None, 1e-6, None)
    qo = paged.paged_append(q[:1], k[:1], v[:1], kp, vp, tables, lens[:1], lens[:1, None], cos, sin)
    ended()
    for got, y, t in ((qo, want[0], want[3]), (kp, want[1], want[4]), (vp, want[2], want[5])):
        close(got, y, t)
    want = attend(qo[:, 0], kp, vp, tables, lens[:1], None, D ** -0.5)
    out, lse = paged.paged_attention(qo[:, 0], kp, vp, tables, lens[:1])
    ended()
    close(out, want[0], want[2])
    before = kp.clone(), vp.clone()
    two = ints(0, 2, 0, 1).view(2, 2)  # 0 full, then pages 2 and 1: beam 1's page takes a copy of beam 0's
    paged.beam_reorder(ints(0, 0).view(1, 2), kp, vp, two, ints(13, 13))
    ended()
    assert two.tolist() == [[0, 2], [0, 1]]
    for x, y in zip((kp, vp), before):
        assert torch.equal(x[1, :, :5], y[2, :, :5]) and torch.equal(x[1, :, 5:], y[1, :, 5:]) and torch.equal(x[[0, 2]], y[[0, 2]])


# --------------------------------------------------------------------------------------------------------- selection
def select_ref(logits, scores, done, end, n):
    """(totals, parents, tokens, ended) as lists of lists"""
    B, W, V = logits.shape
    res = []
    for b in range(B):
        every = []
        for w in range(W):
            s = float(scores[b, w])
            if not math.isfinite(s):
                continue
            if done is not None and bool(done[b, w]):
                every.append((-s, w, 0, end, True))
                continue
            x = logits[b, w].double()
            x = torch.where(torch.isnan(x), torch.full_like(x, -INF), x)
            if not math.isfinite(float(x.max())):
                continue
            lse = float(torch.logsumexp(x, -1))
            val, order = torch.sort(x, descending=True, stable=True)
            for i, (y, t) in enumerate(zip(val[:n].tolist(), order[:n].tolist())):
                if y > -INF:
                    every.append((-(s + (y - lse)), w, i, t, end is not None and t == end))
        every.sort(key=lambda c: c[:3])
        every = every[:n] + [(INF, -1, 0, -1, False)] * (n - len(every[:n]))
        res.append(every)
    return tuple([[f(c) for c in r] for r in res] for f in (lambda c: -c[0], lambda c: c[1], lambda c: c[3], lambda c: c[4]))


def check_select(best, want, V):
    tol = (50 + 2 * math.log2(V + 1) + V / 4096) * E
    w = torch.tensor(want[0], dtype=torch.float64, device="cuda")
    assert best.parents.tolist() == want[1] and best.tokens.tolist() == want[2] and best.done.tolist() == want[3]
    close(best.scores, w, tol + E * w.abs(), "scores")


# type, B, W, V, n, done
SELECTS = [
    ("fp32", 1, 1, 1, 1, False), ("fp16", 2, 3, 2, 8, False), ("bf16", 1, 1, 17, 5, False), ("fp32", 3, 4, 100, 4, True), ("bf16", 2, 5, 4095, 10, True), ("fp16", 2, 2, 4096, 64, False),
    ("fp32", 5, 3, 4097, 6, True), ("fp32", 1, 4, 50001, 4, False), ("bf16", 3, 5, 50001, 10, True), ("fp16", 1, 64, 1000, 64, True), ("fp32", 1, 1, 151936, 33, False), ("fp32", 2, 8, 151936, 8, True),
    ("bf16", 70, 2, 8192, 2, False), ("fp16", 1, 16, 33000, 32, False), ("fp32", 300, 2, 777, 3, True),
]


@pytest.mark.parametrize("case", SELECTS)
def test_select(case):
    name, B, W, V, n, some_done = case
    g = gen(V + n)
    logits = randn(g, B, W, V, scale=3.0, dtype=TYPES[name])
    logits[torch.rand(B, W, V, device="cuda", generator=g) < 0.05] = -INF
    scores = -torch.rand(B, W, device="cuda", generator=g) * 5
    done = torch.rand(B, W, device="cuda", generator=g) < 0.4 if some_done else None
    end = V // 3 if some_done else None
    best = paged.beam_select(logits, scores, done=done, end=end, candidates=n)
    ended()
    check_select(best, select_ref(logits, scores, done, end, n), V)
    again = paged.beam_select(logits, scores, done=done, end=end, candidates=n)
    assert all(torch.equal(x, y) for x, y in zip(best, again))


@pytest.mark.parametrize("name", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("V", [3000, 20001])
def test_select_ties_go_to_the_lowest(name, V):
    g = gen(20)
    few = torch.randint(0, 3, (2, 4, V), device="cuda", generator=g)
    row = few[:, :1].expand(2, 4, V).contiguous().to(TYPES[name])  # the same in all beams, three values, zeros of both signs
    row[..., ::7] *= -1
    scores = torch.full((2, 4), -1.25, device="cuda")
    for n in (1, 4, 13, 40, 64):
        check_select(paged.beam_select(row, scores, candidates=n), select_ref(row, scores, None, None, n), V)
    one = torch.zeros(1, 3, V, dtype=TYPES[name], device="cuda")
    best = paged.beam_select(one, torch.zeros(1, 3, device="cuda"), candidates=50)
    assert best.parents.tolist() == [[0] * 50] and best.tokens.tolist() == [list(range(50))]
    ended()


@pytest.mark.parametrize("order", ["rising", "falling", "late"])
@pytest.mark.parametrize("n", [1, 8, 40, 64])
def test_select_logits_in_order(order, n):
    """every logit above those before it, below them, and the best at the very end"""
    V = 30000
    x = torch.arange(V, dtype=torch.float32, device="cuda") * 1e-3
    x = x if order == "rising" else x.flip(0) if order == "falling" else torch.cat([torch.zeros(V - n, device="cuda"), x[:n] + 3])
    logits, scores = x.expand(1, 2, V), torch.tensor([[-1.0, -1.3]], device="cuda")
    check_select(paged.beam_select(logits, scores, candidates=n), select_ref(logits, scores, None, None, n), V)
    ended()


def test_select_what_is_no_continuation():
    g, V = gen(21), 5000
    logits = randn(g, 1, 8, V)
    logits[0, 0, 7], logits[0, 0, 4000] = NAN, NAN
    logits[0, 1] = -INF
    logits[0, 2, 9] = INF
    logits[0, 3] = NAN
    logits[0, 4, 5:] = -INF
    scores = torch.tensor([[-3.0, -1.0, -1.0, -1.0, -2.0, -INF, NAN, INF]], device="cuda")
    logits[0, 5:] = NAN
    for n in (3, 8, 64):
        check_select(paged.beam_select(logits, scores, candidates=n), select_ref(logits, scores, None, None, n), V)
    done = torch.zeros(1, 8, dtype=torch.bool, device="cuda")
    done[0, 1] = done[0, 5] = True  # one that has ended goes on whatever its logits; one that is not there does not
    best = paged.beam_select(logits, scores, done=done, end=11, candidates=6)
    check_select(best, select_ref(logits, scores, done, 11, 6), V)
    assert best.parents[0, 0] == 1 and best.tokens[0, 0] == 11 and bool(best.done[0, 0])
    few = paged.beam_select(logits[:, 4:5], scores[:, 4:5], candidates=8)
    assert few.tokens[0, 5:].tolist() == [-1] * 3 and few.parents[0, 5:].tolist() == [-1] * 3 and few.scores[0, 5:].tolist() == [-INF] * 3 and not few.done.any()
    none = paged.beam_select(logits[:, 5:], scores[:, 5:])
    assert none.tokens.tolist() == [[-1] * 3] and none.parents.tolist() == [[-1] * 3]
    ended()


def test_select_strides_first_step_and_far_scores():
    g, V = gen(22), 3001
    wide = randn(g, 3, 2, V + 7, dtype=torch.bfloat16)
    logits = wide[:, :, 3:3 + V]
    scores = torch.tensor([[-1.0, -2.0], [-1000.0, -1000.5], [-1e30, -1.0]], device="cuda")
    check_select(paged.beam_select(logits, scores, candidates=7), select_ref(logits, scores, None, None, 7), V)
    first = logits[:, :1].expand(3, 4, V)  # one beam is all there is
    scores = torch.tensor([[0.0] + [-INF] * 3] * 3, device="cuda")
    best = paged.beam_select(first, scores)
    check_select(best, select_ref(first, scores, None, None, 4), V)
    assert best.parents.eq(0).all()
    turned = randn(g, 4, 3, V).transpose(0, 1)  # beams before groups
    check_select(paged.beam_select(turned, torch.zeros(3, 4, device="cuda"), candidates=4), select_ref(turned, torch.zeros(3, 4), None, None, 4), V)
    for scale in (1e-30, 1e-3, 1e4, 1e7, 2e8, 4e8, 1e10, 1e37):
        big = randn(g, 1, 2, V, scale=scale)
        check_select(paged.beam_select(big, torch.zeros(1, 2, device="cuda")), select_ref(big, torch.zeros(1, 2), None, None, 2), V)
    ended()


# -------------------------------------------------------------------------------------------------------- reordering
def reorder_ref(parents, k, v, tables, lens, P):
    """pages and tables after it, by the text of its definition; groups that are left alone are not given"""
    k, v, t = k.clone(), v.clone(), tables.tolist()
    B, W = parents.shape
    k0, v0, t0 = k.clone(), v.clone(), tables.tolist()
    for b in range(B):
        n = int(lens[b * W])
        full, rest = n // P, n % P
        par = [int(p) if p >= 0 else i for i, p in enumerate(parents[b].tolist())]
        for i in range(W):
            t[b * W + i][:full] = t0[b * W + par[i]][:full]
        if not rest:
            continue
        begun = [t0[b * W + i][full] for i in range(W)]
        free, taken = [begun[i] for i in range(W) if i not in par], set()
        for i in range(W):
            if par[i] not in taken:
                t[b * W + i][full] = begun[par[i]]
                taken.add(par[i])
                continue
            to = free.pop(0)
            t[b * W + i][full] = to
            k[..., to, :, :rest, :], v[..., to, :, :rest, :] = k0[..., begun[par[i]], :, :rest, :], v0[..., begun[par[i]], :, :rest, :]
    return k, v, torch.tensor(t, dtype=torch.int32, device="cuda")


# type, layers (0: no dimension), B, W, kv, D, page, lens, kinds of parents
REORDERS = [
    ("fp16", 0, 1, 1, 1, 64, 16, [5], "any"), ("bf16", 2, 1, 4, 8, 128, 16, [777], "any"), ("fp32", 1, 3, 2, 2, 64, 24, [0, 23, 24], "any"), ("fp16", 3, 2, 33, 2, 64, 8, [100, 7], "any"),
    ("bf16", 2, 1, 64, 1, 128, 10, [55], "any"), ("fp32", 0, 4, 8, 3, 128, 7, [6, 7, 8, 0], "one"), ("bf16", 36, 1, 4, 8, 128, 128, [255], "one"), ("fp16", 1, 2, 6, 2, 64, 1, [9, 3], "any"),
    ("fp16", 2, 2, 16, 4, 64, 32, [64, 95], "turned"), ("bf16", 1, 2, 40, 1, 64, 16, [17, 4000], "last"), ("fp32", 1, 1, 5, 2, 128, 1000, [999], "some -1"), ("fp16", 2, 130, 3, 1, 64, 16, list(range(130)), "any"),
]


@pytest.mark.parametrize("case", REORDERS)
def test_reorder(case):
    name, layers, B, W, kv, D, page, lens_, kind = case
    g, dt = gen(W * 10 + B), TYPES[name]
    pages, cols = B * W + 3, max(lens_) // page + 2
    shape = ((layers,) if layers else ()) + (pages, kv, page, D)
    k, v = randn(g, *shape, dtype=dt), randn(g, *shape, dtype=dt)
    lens = torch.tensor(lens_, dtype=torch.int32, device="cuda").repeat_interleave(W)
    tables = torch.randint(0, 10 ** 6, (B * W, cols + 2), dtype=torch.int32, device="cuda", generator=g)[:, :cols]  # full pages are not looked into
    tables.scatter_(1, (lens // page).long()[:, None], torch.randperm(pages, device="cuda", generator=g)[:B * W].int()[:, None])
    parents = {"any": lambda: torch.randint(0, W, (B, W), device="cuda", generator=g), "one": lambda: torch.full((B, W), W // 2, device="cuda"),
               "turned": lambda: torch.arange(W, device="cuda").flip(0).expand(B, W), "last": lambda: torch.full((B, W), W - 1, device="cuda"),
               "some -1": lambda: torch.randint(-1, W, (B, W), device="cuda", generator=g)}[kind]().int().contiguous()
    want = reorder_ref(parents, k, v, tables, lens, page)
    assert paged.beam_reorder(parents, k, v, tables, lens) is tables
    ended()
    assert torch.equal(tables, want[2]) and torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_reorder_leaves_a_group_alone_that_is_out_of_range():
    g = gen(31)
    for bad in ("parent", "low parent", "lengths", "negative", "long", "huge"):
        k, v = randn(g, 2, 12, 2, 16, 64), randn(g, 2, 12, 2, 16, 64)
        tables = torch.randperm(12, device="cuda", generator=g).int().view(6, 2)
        parents, lens = ints(0, 0, 1, 2, 2, 0).view(2, 3), ints(21, 21, 21, 20, 20, 20)
        if bad == "parent":
            parents[0, 1] = 3
        elif bad == "low parent":
            parents[0, 2] = -2
        elif bad == "lengths":
            lens[1] = 22
        else:
            lens[:3] = {"negative": -1, "long": 33, "huge": 2 ** 31 - 1}[bad]
        want = reorder_ref(torch.cat([ints(-1, -1, -1)[None], parents[1:]]), k, v, tables, torch.cat([ints(0, 0, 0), lens[3:]]), 16)
        paged.beam_reorder(parents, k, v, tables, lens)
        ended(64)
        assert torch.equal(tables, want[2]) and torch.equal(k, want[0]) and torch.equal(v, want[1]), bad
    for page in (12, -1, -2 ** 31, 2 ** 31 - 1):  # a begun page that is none: it is not copied
        k, v = randn(g, 2, 12, 2, 16, 64), randn(g, 2, 12, 2, 16, 64)
        k0, v0 = k.clone(), v.clone()
        tables = ints(0, 1, 2, page, 4, 5).view(3, 2)
        paged.beam_reorder(ints(0, 0, 2).view(1, 3), k, v, tables, ints(21, 21, 21))
        ended(64)
        assert torch.equal(k, k0) and torch.equal(v, v0) and tables.tolist() == [[0, 1], [0, page], [4, 5]]


# ----------------------------------------------------------------------------------------------------- used together
def test_a_prompt_and_beams_from_it_on_a_side_stream():
    """pages shared under all beams, then some steps; every beam's attention is that over its own history"""
    g, W, kv, H, D, P, n0, steps = gen(40), 4, 2, 4, 64, 8, 21, 14
    dt = torch.float32
    pages = n0 // P + W * (steps // P + 3)
    k, v = (torch.full((1, pages, kv, P, D), NAN, device="cuda") for _ in range(2))
    cols = (n0 + steps) // P + 1
    tables = torch.full((W, cols), -1, dtype=torch.int32)
    tables[0, :n0 // P] = torch.arange(n0 // P)
    tables[:, n0 // P:] = n0 // P + torch.arange(W * (cols - n0 // P)).view(W, -1)
    tables = tables.cuda()
    cos, sin = paged.rotary_tables(64, D, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    hist = [[] for _ in range(W)]  # (key, value) of each beam's slots
    q, kk, vv = randn(g, 1, n0, H, D), randn(g, 1, n0, kv, D), randn(g, 1, n0, kv, D)
    lens = torch.zeros(W, dtype=torch.int32, device="cuda")
    paged.paged_append(q, kk, vv, k[0], v[0], tables[:1], lens[:1], torch.arange(n0, dtype=torch.int32, device="cuda")[None], cos, sin, stream=st)
    st.synchronize()
    flat = lambda x, row, n: x[0][tables[row].long().clamp(min=0)].transpose(1, 2).reshape(-1, kv, D)[:n]  # noqa: E731
    hist[0] = (flat(k, 0, n0).clone(), flat(v, 0, n0).clone())
    lens += n0
    parents = torch.zeros(1, W, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    for step in range(steps):
        paged.beam_reorder(parents, k, v, tables, lens, stream=st)
        hist = [hist[p] for p in parents[0].tolist()]
        q, kk, vv = randn(g, W, 1, H, D), randn(g, W, 1, kv, D), randn(g, W, 1, kv, D)
        torch.cuda.synchronize()
        qq = paged.paged_append(q, kk, vv, k[0], v[0], tables, lens, lens[:, None].contiguous(), cos, sin, stream=st)
        out, lse = paged.paged_attention(qq[:, 0], k[0], v[0], tables, lens, stream=st)
        st.synchronize()
        n = n0 + step + 1
        for w in range(W):
            a, b = flat(k, w, n), flat(v, w, n)
            assert torch.equal(a[:-1], hist[w][0]) and torch.equal(b[:-1], hist[w][1]), (step, w)
            hist[w] = (a.clone(), b.clone())
        want = attend(qq[:, 0], k[0], v[0], tables, lens, None, D ** -0.5)
        close(out, want[0], want[2])
        lens += 1
        parents = torch.randint(0, W, (1, W), dtype=torch.int32, device="cuda", generator=g)
    ended()


def test_a_step_in_a_graph_and_two_graphs_with_one_workspace():
    g, W, H, kv, D, P, V = gen(41), 3, 8, 2, 128, 16, 5003
    k, v = (randn(g, 2, 40, kv, P, D, dtype=torch.float16) for _ in range(2))
    tables0 = torch.randperm(40, device="cuda", generator=g)[:36].int().view(W, 12)
    tables0[:, :6] = tables0[0, :6]
    head = randn(g, H * D, V, scale=0.05)
    cos, sin = paged.rotary_tables(200, D, device="cuda")
    x = randn(g, W, 1, (H + 2 * kv) * D)
    ws = torch.empty(max(paged.attention_workspace_size(k[0], v[0], tables0, H), paged.select_workspace_size(head.T[None, :1].expand(1, W, H * D), 5), paged.select_workspace_size(torch.empty(1, W, V, device="cuda"), W)),
                     dtype=torch.uint8, device="cuda")

    def fresh():
        return {"k": k.clone(), "v": v.clone(), "tables": tables0.clone(), "lens": ints(100, 100, 100), "scores": torch.tensor([[0.0, -1.0, -1.5]], device="cuda"),
                "done": torch.zeros(1, W, dtype=torch.bool, device="cuda"), "tokens": torch.zeros(1, W, dtype=torch.int64, device="cuda"), "parents": torch.zeros(1, W, dtype=torch.int32, device="cuda")}

    def step(s):
        q, kk, vv = (y.unflatten(2, (-1, D)) for y in x.split([H * D, kv * D, kv * D], dim=2))
        acc = 0
        for L in range(2):
            qq = paged.paged_append(q + acc, kk, vv, s["k"][L], s["v"][L], s["tables"], s["lens"], s["lens"][:, None], cos, sin)
            out, _ = paged.paged_attention(qq[:, 0], s["k"][L], s["v"][L], s["tables"], s["lens"], workspace=ws)
            acc = out[:, None].float()
        logits = (acc.reshape(W, -1) @ head + s["tokens"].view(-1, 1) * 1e-4)[None]
        best = paged.beam_select(logits, s["scores"], done=s["done"], end=2, workspace=ws)
        s["scores"].copy_(best.scores), s["done"].copy_(best.done), s["tokens"].copy_(best.tokens), s["parents"].copy_(best.parents)
        s["lens"] += 1
        paged.beam_reorder(s["parents"], s["k"], s["v"], s["tables"], s["lens"])

    eager = fresh()
    for _ in range(30):
        step(eager)
    ended()
    states, graphs = [fresh(), fresh()], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fresh())
    torch.cuda.synchronize()
    for s in states:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            step(s)
        graphs.append(gr)
    for _ in range(30):
        for gr in graphs:
            gr.replay()
    ended()
    for s in states:
        for name in ("tables", "lens", "scores", "tokens", "parents"):
            assert torch.equal(s[name], eager[name]), name
        assert torch.equal(s["k"], eager["k"]) and torch.equal(s["v"], eager["v"])


# ------------------------------------------------------------------------------------------------ calls at the edges
def test_4096_sequences_some_without_a_token():
    g, B, H, kv, D, P = gen(50), 4096, 4, 2, 64, 16
    lens_ = [(7 * i) % 90 for i in range(B)]
    pages = sum(n // P + 1 for n in lens_) + 1
    kp, vp = make_pages(g, pages, kv, P, D, torch.float16)
    tables, lens = make_tables(g, lens_, 1, P, pages), ints(*lens_)
    counts = (torch.arange(B, device="cuda") % 5 != 3).int()
    q = randn(g, B, H, D, dtype=torch.float16)
    cos, sin = paged.rotary_tables(100, D, device="cuda")
    x = randn(g, B, 1, H + 2 * kv, D)
    before = kp.clone()
    paged.paged_append(x[:, :, :H], x[:, :, H:H + kv], x[:, :, H + kv:], kp, vp, tables, lens, lens[:, None].contiguous(), cos, sin, counts=counts)
    at = tables.gather(1, (lens // P).long()[:, None])[:, 0].long()
    wrote = (kp[at, :, (lens % P).long()] != before[at, :, (lens % P).long()]).flatten(1).any(1)
    assert torch.equal(wrote, counts.bool())
    out, lse = torch.full_like(q, 7.0), torch.full((B, H), 7.0, device="cuda")
    paged.paged_attention(q, kp, vp, tables, lens, counts=counts, out=out, lse=lse)
    ended()
    skipped = counts == 0
    assert (out[skipped] == 7).all() and (lse[skipped] == 7).all()
    some = torch.arange(0, B, 37, device="cuda")
    want = attend(q[some], kp, vp, tables[some], lens[some], counts[some], D ** -0.5)
    live = counts[some] == 1
    close(out[some][live], want[0][live], want[2][live])
    close(lse[some][live], want[1][live], want[3][live])
    none, l0 = torch.full_like(q, 7.0), torch.full((B, H), 7.0, device="cuda")
    paged.paged_attention(q, kp, vp, tables, lens, counts=torch.zeros_like(counts), out=none, lse=l0)
    ended()
    assert (none == 7).all() and (l0 == 7).all()


def test_calls_on_two_streams_at_once():
    g, D, P = gen(51), 128, 16
    kp, vp = make_pages(g, 700, 8, P, D, torch.bfloat16)
    sets = []
    for i in range(2):
        lens_ = [3000 - 500 * i, 17, 800]
        tables = make_tables(g, lens_, 1, P, 700)
        sets.append((randn(g, 3, 32, D, dtype=torch.bfloat16), tables, ints(*lens_), randn(g, 2, 4, 30011), -torch.rand(2, 4, device="cuda", generator=g)))
    one = [(paged.paged_attention(q, kp, vp, t, n), paged.beam_select(x, s)) for q, t, n, x, s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i, (q, t, n, x, s) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i].append((paged.paged_attention(q, kp, vp, t, n), paged.beam_select(x, s)))
    ended()
    for i in range(2):
        for (a, l), best in got[i]:
            assert torch.equal(a, one[i][0][0]) and torch.equal(l, one[i][0][1]) and all(torch.equal(x, y) for x, y in zip(best, one[i][1]))


def test_a_sequence_over_the_pages_of_another_and_one_page_twice():
    """the same page in several places of a table, and under several sequences"""
    g, D, P = gen(52), 64, 8
    kp, vp = make_pages(g, 4, 2, P, D, torch.float32)
    tables, lens, q = ints(1, 1, 1, 3, 1, 0).view(2, 3), ints(23, 20), randn(g, 2, 2, D)
    want = attend(q, kp, vp, tables, lens, None, D ** -0.5)
    out, lse = paged.paged_attention(q, kp, vp, tables, lens)
    ended()
    close(out, want[0], want[2])
    close(lse, want[1], want[3])


def test_select_of_equal_beams_of_an_odd_vocabulary():
    """two beams that are one another's copy tie in every continuation, wherever their rows begin in memory"""
    g = gen(53)
    for name in TYPES:
        row = randn(g, 1, 1, 20011, dtype=TYPES[name])
        logits, scores = row.expand(3, 4, 20011).contiguous(), torch.full((3, 4), -2.5, device="cuda")
        for n in (4, 20):
            check_select(paged.beam_select(logits, scores, candidates=n), select_ref(logits, scores, None, None, n), 20011)
    ended()


def test_select_of_the_largest_groups():
    g, W, V = gen(54), 64, 9001
    logits, scores = randn(g, 2, W, V, dtype=torch.float16, scale=0.1), -torch.rand(2, W, device="cuda", generator=g) * 0.01
    check_select(paged.beam_select(logits, scores, candidates=64), select_ref(logits, scores, None, None, 64), V)
    flat = torch.zeros(1, W, V, device="cuda")
    check_select(paged.beam_select(flat, torch.zeros(1, W, device="cuda"), candidates=64), select_ref(flat, torch.zeros(1, W), None, None, 64), V)
    done = torch.ones(2, W, dtype=torch.bool, device="cuda")
    check_select(paged.beam_select(logits, scores, done=done, end=5, candidates=64), select_ref(logits, scores, done, 5, 64), V)
    ended()
