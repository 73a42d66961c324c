"""Key/value cache operators without a GPU: the drafted trees' plan, and what the entry points refuse before they touch
a device (the C entries get addresses that nothing reads)."""
import struct

import pytest
import torch

import pingala8_llm_b200 as p8
from pingala8_llm_b200 import cache

PTR = 1 << 20  # an aligned address that is never read: every call below is refused first
KV = struct.Struct("=16q")
ARG, WORKSPACE, UNSUPPORTED = -1, -11, -13


def kv(k=PTR, v=2 * PTR, type=2, layers=1, batch=2, heads=2, slots=64, width=64, ks=None, vs=None):
    st = (batch * heads * slots * width, heads * slots * width, slots * width, width)
    return KV.pack(k, v, type, layers, batch, heads, slots, width, *(ks or st), *(vs or st))


def walk(parents):
    mask, depth = [], []
    for t in range(len(parents)):
        bits, d, c = 0, -1, t
        while c >= 0:
            bits |= 1 << c
            d += 1
            c = parents[c]
        mask.append(bits - (1 << 64) if bits >> 63 else bits)
        depth.append(d)
    return mask, depth


@pytest.mark.parametrize("n,seed", [(1, 0), (2, 1), (7, 2), (33, 3), (64, 4)])
def test_tree_plan_is_the_walk_to_the_root(n, seed):
    g = torch.Generator().manual_seed(seed)
    par = [-1] + [int(torch.randint(-1 if seed % 2 else 0, t, (1,), generator=g)) for t in range(1, n)]
    m, d = cache.tree_plan(torch.tensor(par, dtype=torch.int32))
    assert (m.tolist(), d.tolist()) == walk(par)
    both = torch.tensor([par, [-1] + list(range(n - 1))])
    m, d = cache.tree_plan(both)
    assert m[0].tolist() == walk(par)[0] and d[1].tolist() == list(range(n))
    assert m.dtype == torch.int64 and d.dtype == torch.int32


def test_tree_plan_refuses():
    for bad in (torch.zeros(65, dtype=torch.int32), torch.zeros(0, dtype=torch.int32), torch.zeros(3), torch.zeros(1, 1, 1, dtype=torch.int32)):
        with pytest.raises(ValueError):
            cache.tree_plan(bad)


def test_tensors_on_the_cpu_are_refused():
    k, i = torch.zeros(1, 1, 8, 64), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 1, 1, 64)
    t = torch.zeros(1, 1, dtype=torch.int64)
    for call in (lambda: cache.kv_append(q, q, q, k, k, i, i[None], k[0, 0], k[0, 0]), lambda: cache.tree_attention(q, k, k, i),
                 lambda: cache.attention_mass(q, q[..., 0], k, i, k[..., 0]), lambda: cache.kv_evict(k, k, k[..., 0], i, 4),
                 lambda: cache.tree_accept(t, t.int(), t, k, k, i)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


BAD_KV = [dict(k=0), dict(v=0), dict(k=PTR + 8), dict(type=3), dict(type=-1), dict(layers=0), dict(batch=0), dict(batch=4097), dict(heads=0),
          dict(slots=0), dict(slots=1 << 31), dict(width=96), dict(width=256), dict(ks=(0, 8192, 4100, 64)), dict(vs=(0, 8192, 4096, 65))]


def append_args(**o):
    d = dict(q=PTR, k=PTR, v=PTR, qs=(512, 256, 64), ks=(256, 128, 64), vs=(256, 128, 64), tokens=2, heads=4, lens=PTR, counts=0, pos=PTR, cos=PTR,
             sin=PTR, positions=10, qn=0, kn=0, eps=1e-6, out=PTR, os=(512, 256, 64)) | o
    return struct.pack("=3q9q2q3q2qq2qd4q", d["q"], d["k"], d["v"], *d["qs"], *d["ks"], *d["vs"], d["tokens"], d["heads"], d["lens"], d["counts"],
                       d["pos"], d["cos"], d["sin"], d["positions"], d["qn"], d["kn"], d["eps"], d["out"], *d["os"])


def attn_args(**o):
    d = dict(q=4 * PTR, qs=(512, 256, 64), tokens=2, heads=4, lens=PTR, counts=0, mask=0, ms=0, scale=0.1, out=5 * PTR, os=(512, 256, 64), lse=0) | o
    return struct.pack("=4q2q4qd5q", d["q"], *d["qs"], d["tokens"], d["heads"], d["lens"], d["counts"], d["mask"], d["ms"], d["scale"], d["out"], *d["os"], d["lse"])


def mass_args(**o):
    d = dict(q=4 * PTR, qs=(512, 256, 64), tokens=2, heads=4, lse=PTR, lens=PTR, counts=0, rows=0, scale=0.1, mass=PTR, ms=(128, 64), out=PTR, os=(128, 64)) | o
    return struct.pack("=4q2q4qd6q", d["q"], *d["qs"], d["tokens"], d["heads"], d["lse"], d["lens"], d["counts"], d["rows"], d["scale"], d["mass"], *d["ms"], d["out"], *d["os"])


def evict_args(**o):
    d = dict(mass=3 * PTR, ms=(256, 128, 64), out=3 * PTR, os=(256, 128, 64), lens=PTR, new=2 * PTR, kept=PTR, budget=8, sinks=2, recent=2) | o
    return struct.pack("=8q3q3q", d["mass"], *d["ms"], d["out"], *d["os"], d["lens"], d["new"], d["kept"], d["budget"], d["sinks"], d["recent"])


def accept_args(**o):
    d = dict(tokens=PTR, target=PTR, parents=PTR, n=4, lens=PTR, counts=0, path=PTR, accepted=PTR, new=2 * PTR, next=PTR) | o
    return struct.pack("=10q", *(d[x] for x in ("tokens", "target", "parents", "n", "lens", "counts", "path", "accepted", "new", "next")))


@pytest.mark.parametrize("bad", BAD_KV, ids=str)
def test_a_bad_cache_is_refused_by_every_entry(bad):
    L, c = p8.lib(), kv(**bad)
    assert L.p8_kv_append(c, append_args(), None) == ARG
    assert L.p8_tree_attn_workspace(c, 2, 4) == 0
    assert L.p8_tree_attn(c, attn_args(), None, 0, None) == ARG
    if "v" not in bad and "vs" not in bad:
        assert L.p8_attn_mass(c, mass_args(), None) == ARG
    assert L.p8_kv_evict(c, c, evict_args(), None) == ARG
    assert L.p8_tree_accept(c, accept_args(), None) == ARG


def test_bad_arguments_are_refused():
    L, c = p8.lib(), kv()
    for bad in (dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(lens=0), dict(pos=0), dict(cos=0), dict(sin=0), dict(q=PTR + 4), dict(cos=PTR + 4),
                dict(tokens=-1), dict(tokens=65), dict(heads=3), dict(heads=0), dict(positions=0), dict(eps=-1.0), dict(eps=float("nan")),
                dict(qs=(512, 254, 64)), dict(ks=(256, 128, 66)), dict(os=(512, 252, 64))):
        assert L.p8_kv_append(c, append_args(**bad), None) == ARG, bad
    for bad in (dict(q=0), dict(out=0), dict(lens=0), dict(tokens=0), dict(tokens=65), dict(heads=5), dict(scale=float("inf")), dict(scale=float("nan")),
                dict(mask=PTR, ms=3), dict(qs=(512, 256, 68)), dict(os=(512, 260, 64)), dict(out=4 * PTR), dict(out=PTR), dict(out=2 * PTR + 4096)):
        assert L.p8_tree_attn(c, attn_args(**bad), PTR, 1 << 40, None) == ARG, bad
    for bad in (dict(q=0), dict(lse=0), dict(lens=0), dict(mass=0), dict(out=0), dict(tokens=0), dict(tokens=65), dict(heads=3), dict(out=PTR + 64),
                dict(os=(64, 128)), dict(scale=float("nan"))):
        assert L.p8_attn_mass(c, mass_args(**bad), None) == ARG, bad
    for bad in (dict(mass=0), dict(out=0), dict(lens=0), dict(new=0), dict(kept=0), dict(new=PTR), dict(budget=0), dict(budget=65), dict(sinks=-1),
                dict(recent=-1), dict(sinks=5, recent=4), dict(sinks=9), dict(recent=9), dict(out=3 * PTR + 4), dict(os=(256, 64, 128))):
        assert L.p8_kv_evict(c, c, evict_args(**bad), None) == ARG, bad
    for other in (dict(type=1), dict(width=128), dict(heads=1), dict(batch=1), dict(layers=2), dict(k=PTR + 4096), dict(k=2 * PTR), dict(slots=4)):
        assert L.p8_kv_evict(c, kv(**other), evict_args(), None) == ARG, other
    for bad in (dict(tokens=0), dict(target=0), dict(parents=0), dict(lens=0), dict(path=0), dict(accepted=0), dict(new=0), dict(next=0), dict(new=PTR),
                dict(n=0), dict(n=65)):
        assert L.p8_tree_accept(c, accept_args(**bad), None) == ARG, bad
    two = kv(layers=2)
    assert L.p8_kv_append(two, append_args(), None) == ARG and L.p8_tree_attn(two, attn_args(), None, 0, None) == ARG
    assert L.p8_attn_mass(two, mass_args(), None) == ARG
