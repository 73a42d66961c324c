"""Paged cache and beam search operators without a GPU: the rotation's tables, and what the entry points refuse before they touch a
device (the C entries get addresses that nothing may read: a call that is not refused ends at its launch, with another status)."""
import math
import struct

import pytest
import torch

import pingala8_llm_b200 as p8
from pingala8_llm_b200 import decode, paged

MB = 1 << 20
ARG, WORKSPACE, UNSUPPORTED = -1, -11, -13


def pages(**o):
    """16 pages of 2 heads x 8 slots x 64, 16 bits: 32 KB each of keys and values; tables of 4 rows x 5 columns: 80 bytes"""
    d = dict(k=16 * MB, v=32 * MB, type=1, layers=1, pages=16, heads=2, page=8, width=64, tables=48 * MB, rows=4, columns=5, ts=5) | o
    st = d.get("ks") or (d["pages"] * d["heads"] * d["page"] * d["width"], d["heads"] * d["page"] * d["width"], d["page"] * d["width"], d["width"])
    return struct.pack("=20q", d["k"], d["v"], d["type"], d["layers"], d["pages"], d["heads"], d["page"], d["width"], *st, *(d.get("vs") or st), d["tables"], d["rows"], d["columns"], d["ts"])


def append(c=None, **o):
    d = dict(q=50 * MB, k=51 * MB, v=52 * MB, qs=(512, 256, 64), ks=(256, 128, 64), vs=(256, 128, 64), tokens=2, heads=4, lens=53 * MB, counts=54 * MB, pos=55 * MB, cos=56 * MB, sin=57 * MB, positions=10,
             rotary=64, pairs=0, qn=58 * MB, kn=59 * MB, eps=1e-6, out=60 * MB, os=(512, 256, 64)) | o
    return p8.lib().p8_paged_append(c or pages(), struct.pack("=3q9q2q3q2q3q2qdq3q", d["q"], d["k"], d["v"], *d["qs"], *d["ks"], *d["vs"], d["tokens"], d["heads"], d["lens"], d["counts"], d["pos"], d["cos"], d["sin"],
                                                              d["positions"], d["rotary"], d["pairs"], d["qn"], d["kn"], d["eps"], d["out"], *d["os"]), None)


def attend(c=None, ws=70 * MB, bytes=64 * MB, **o):
    d = dict(q=50 * MB, qs=(256, 64), heads=4, lens=53 * MB, counts=54 * MB, scale=0.1, out=60 * MB, os=(256, 64), lse=61 * MB) | o
    return p8.lib().p8_paged_attn(c or pages(columns=100, ts=100), struct.pack("=6qd4q", d["q"], *d["qs"], d["heads"], d["lens"], d["counts"], d["scale"], d["out"], *d["os"], d["lse"]), ws, bytes, None)


def select(ws=70 * MB, bytes=64 * MB, **o):
    """2 groups of 3 beams, 1,000 tokens of 16 bits; 5 candidates"""
    d = dict(logits=16 * MB, type=1, batch=2, beams=3, vocab=1000, st=(3000, 1000), scores=50 * MB, done=51 * MB, end=7, n=5, out=52 * MB, parents=53 * MB, tokens=54 * MB, out_done=55 * MB) | o
    return p8.lib().p8_beam_select(struct.pack("=15q", d["logits"], d["type"], d["batch"], d["beams"], d["vocab"], *d["st"], d["scores"], d["done"], d["end"], d["n"], d["out"], d["parents"], d["tokens"], d["out_done"]),
                                   ws, bytes, None)


def reorder(c=None, parents=50 * MB, lens=51 * MB, batch=2, beams=2):
    return p8.lib().p8_beam_reorder(c or pages(), parents, lens, batch, beams, None)


no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that nothing may read: not where a launch would reach a GPU")

BAD = [dict(k=0), dict(v=0), dict(k=16 * MB + 8), dict(v=32 * MB + 4), dict(type=3), dict(type=-1), dict(layers=0), dict(pages=0), dict(pages=1 << 31), dict(heads=0), dict(page=0), dict(page=(1 << 20) + 1),
       dict(width=96), dict(width=256), dict(tables=0), dict(tables=48 * MB + 2), dict(rows=0), dict(columns=0), dict(columns=(1 << 27) + 1, ts=1 << 28), dict(ts=-5), dict(ts=4), dict(ks=(0, 1024, 512, 60)),
       dict(vs=(0, 1024, 516, 64)), dict(ks=(0, -1024, 512, 64)), dict(layers=40000)]


@no_gpu
@pytest.mark.parametrize("bad", BAD, ids=str)
def test_bad_pages_are_refused_by_every_entry(bad):
    c = pages(**bad)
    assert append(c) == ARG and attend(c) == ARG and reorder(c) == ARG and p8.lib().p8_paged_attn_workspace(c, 4) == 0


@no_gpu
def test_good_calls_are_not_refused():
    assert append() not in (0, ARG, UNSUPPORTED) and attend() not in (0, ARG, WORKSPACE, UNSUPPORTED) and select() not in (0, ARG, WORKSPACE) and reorder() not in (0, ARG, UNSUPPORTED)
    assert append(counts=0, qn=0, kn=0, pairs=1, rotary=8) != ARG and attend(counts=0, lse=0) != ARG and select(done=0, end=-1, out_done=0) not in (ARG, WORKSPACE)
    assert append(pages(k=1 << 40, v=1 << 42, page=1 << 20, columns=1 << 10, ts=1 << 10)) != ARG and attend(pages(ts=0)) != ARG and append(pages(ts=0)) != ARG
    assert reorder(pages(layers=7, ks=(1 << 20, 1024, 512, 64), vs=(1 << 20, 1024, 512, 64), v=1 << 40)) != ARG


@no_gpu
def test_append_refuses():
    for bad in (dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(lens=0), dict(pos=0), dict(cos=0), dict(sin=0), dict(q=50 * MB + 4), dict(sin=57 * MB + 8), dict(out=60 * MB + 8), dict(tokens=-1), dict(tokens=41),
                dict(heads=3), dict(heads=0), dict(positions=0), dict(eps=-1.0), dict(eps=math.nan), dict(qs=(512, 254, 64)), dict(ks=(256, 128, 66)), dict(os=(512, 252, 64)), dict(rotary=0), dict(rotary=4),
                dict(rotary=60), dict(rotary=72), dict(rotary=-8)):
        assert append(**bad) == ARG, bad
    # over what it reads: q is 8,192 bytes and its 16-bit result 4,096, k and v are 4,096 each, tables 10 x 128
    for bad in (dict(out=51 * MB), dict(out=50 * MB), dict(out=53 * MB), dict(out=55 * MB), dict(out=56 * MB + 1264), dict(out=48 * MB + 64), dict(out=16 * MB), dict(out=32 * MB + 32752), dict(k=16 * MB), dict(q=32 * MB),
                dict(lens=16 * MB + 4), dict(kn=60 * MB)):
        assert append(**bad) == ARG, bad
    assert append(pages(tables=16 * MB + 512)) == ARG and append(pages(v=16 * MB + 512)) == ARG
    assert append(pages(ks=(0, 512, 512, 64))) == ARG and append(os=(512, 64, 64)) == ARG  # rows that share memory
    assert append(pages(type=0), out=50 * MB) not in (0, ARG)  # in place
    assert append(out=50 * MB) == ARG and append(pages(type=0), out=50 * MB, os=(512, 256, 128)) == ARG
    assert append(pages(layers=2)) == ARG and append(pages(rows=4097)) == ARG
    nothing = dict(tokens=0, q=0, k=0, v=0, out=0, pos=0, lens=0, cos=0, sin=0)
    assert append(**nothing) == 0 and append(pages(width=96), **nothing) == ARG and append(**nothing, heads=3) == ARG


@no_gpu
def test_attention_refuses():
    for bad in (dict(q=0), dict(out=0), dict(lens=0), dict(heads=5), dict(heads=0), dict(scale=math.inf), dict(scale=math.nan), dict(scale=3e38), dict(q=50 * MB + 8), dict(out=60 * MB + 8), dict(qs=(256, 68)),
                dict(os=(260, 64)), dict(os=(128, 64))):
        assert attend(**bad) == ARG, bad
    # q and out are 2,048 bytes, lse 64
    for bad in (dict(out=50 * MB), dict(out=50 * MB + 2032), dict(out=53 * MB), dict(out=54 * MB - 2032), dict(out=48 * MB + 1584), dict(out=16 * MB), dict(lse=60 * MB + 2044), dict(lse=32 * MB), dict(lse=48 * MB),
                dict(ws=50 * MB), dict(ws=60 * MB), dict(ws=61 * MB), dict(ws=16 * MB), dict(ws=48 * MB), dict(ws=53 * MB)):
        assert attend(**bad) == ARG, bad
    assert attend(out=50 * MB + 2048) != ARG and attend(out=50 * MB + 128, qs=(512, 128), os=(512, 128)) != ARG  # side by side
    need = p8.lib().p8_paged_attn_workspace(pages(columns=100, ts=100), 4)
    assert need > 0 and attend(bytes=need - 1) == WORKSPACE and attend(ws=0) == WORKSPACE and attend(ws=70 * MB + 128) == WORKSPACE and attend(bytes=need) not in (ARG, WORKSPACE)
    assert p8.lib().p8_paged_attn_workspace(pages(), 4) == 0 and attend(pages(), ws=0, bytes=0) not in (ARG, WORKSPACE)  # sequences too short to be cut
    assert attend(pages(layers=2, columns=100, ts=100)) == ARG and attend(pages(rows=4097, columns=100, ts=100)) == ARG


@no_gpu
def test_select_refuses():
    for bad in (dict(logits=0), dict(scores=0), dict(out=0), dict(parents=0), dict(tokens=0), dict(type=3), dict(type=-1), dict(batch=0), dict(batch=4097), dict(beams=0), dict(beams=65), dict(vocab=0), dict(vocab=1 << 31),
                dict(n=0), dict(n=65), dict(end=1000), dict(end=-1), dict(logits=16 * MB + 1), dict(type=0, logits=16 * MB + 2), dict(st=(-3000, 1000)), dict(st=(3000, -1))):
        assert select(**bad) == ARG, bad
    assert select(end=999) != ARG and select(logits=16 * MB + 2) not in (ARG, WORKSPACE) and select(st=(0, 0)) not in (ARG, WORKSPACE)
    # logits are 12,000 bytes, scores 24, done 6; results 40, 40, 80 and 10
    for bad in (dict(out=16 * MB + 11999 // 4 * 4), dict(out=50 * MB + 20), dict(parents=52 * MB + 36), dict(tokens=53 * MB + 32), dict(out_done=54 * MB + 79), dict(out_done=51 * MB + 5), dict(out_done=50 * MB), dict(tokens=51 * MB),
                dict(ws=16 * MB), dict(ws=50 * MB), dict(ws=55 * MB)):
        assert select(**bad) == ARG, bad
    assert select(out=50 * MB + 24, parents=52 * MB + 40, out_done=51 * MB + 6) not in (ARG, WORKSPACE)
    L = p8.lib()
    need = L.p8_beam_select_workspace(2, 3, 1000, 5)
    assert need > 0 and select(bytes=need - 1) == WORKSPACE and select(ws=0) == WORKSPACE and select(ws=70 * MB + 8) == WORKSPACE and select(bytes=need) not in (ARG, WORKSPACE)
    for bad in ((0, 3, 1000, 5), (2, 65, 1000, 5), (2, 3, 0, 5), (2, 3, 1000, 0), (2, 3, 1000, 65), (4097, 3, 1000, 5), (2, 3, 1 << 31, 5)):
        assert L.p8_beam_select_workspace(*bad) == 0


@no_gpu
def test_reorder_refuses():
    assert reorder(parents=0) == ARG and reorder(lens=0) == ARG and reorder(batch=0) == ARG and reorder(batch=3) == ARG and reorder(batch=4, beams=1) != ARG
    assert reorder(pages(rows=65, columns=1, ts=1), batch=1, beams=65) == ARG and reorder(pages(ts=0)) == ARG and reorder(pages(ts=4)) == ARG
    # tables are 80 bytes, parents and lengths 16
    for bad in (dict(parents=48 * MB + 76), dict(lens=48 * MB), dict(lens=48 * MB - 12), dict(parents=16 * MB), dict(lens=32 * MB + 32764)):
        assert reorder(**bad) == ARG, bad
    assert reorder(parents=48 * MB + 80, lens=48 * MB - 16) != ARG
    assert reorder(pages(tables=16 * MB + 1024)) == ARG and reorder(pages(v=16 * MB)) == ARG and reorder(pages(ks=(0, 512, 512, 64))) == ARG and reorder(pages(layers=2, ks=(0, 1024, 512, 64))) == ARG


def test_tensors_on_the_cpu_are_refused():
    k, i, t = torch.zeros(2, 1, 8, 64), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32)
    q = torch.zeros(1, 1, 1, 64)
    for call in (lambda: paged.paged_append(q, q, q, k, k, t, i, i[None], k[0, 0], k[0, 0]), lambda: paged.paged_attention(q[0], k, k, t, i), lambda: paged.beam_select(q[0], q[0, :, :, 0]),
                 lambda: paged.beam_reorder(i[None], k, k, t, i), lambda: paged.attention_workspace_size(k, k, t, 1), lambda: paged.select_workspace_size(q[0], 1)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for n in (0, 65, True, 2.0):
        with pytest.raises(ValueError, match="candidates"):
            paged.beam_select(q[0], q[0, :, :, 0], candidates=n)


# ------------------------------------------------------------------------------------------------------------- tables
def angles(positions, width, theta, change=lambda i, inv: inv):
    return [[p * change(i, theta ** (-2 * i / width)) for i in range(width // 2)] for p in range(positions)]


def same(tables, want, gain=1.0):
    """angles off by a few roundings of 64 bits: positions up to 10^5 x 2^-51 are nothing beside the 2^-24 of a result"""
    for t, f in zip(tables, (math.cos, math.sin)):
        w = torch.tensor([[gain * f(x) for x in row] for row in want], dtype=torch.float64)
        assert t.dtype == torch.float32 and t.shape == w.shape and float((t.double() - w).abs().max()) <= gain * 2.0 ** -24 + 1e-9


def test_rotary_tables():
    same(paged.rotary_tables(50, 24, 1e6), angles(50, 24, 1e6))
    same(paged.rotary_tables(50, 24, 1e6, kind="linear", factor=4), angles(50, 24, 1e6, lambda i, v: v / 4))
    same(paged.rotary_tables(50, 24, 1e4, kind="theta", factor=8.0), angles(50, 24, 1e4 * 8 ** (24 / 22)))
    far = paged.rotary_tables(100_001, 8, 1e4)
    same([x[-1:] for x in far], [[100_000 * 1e4 ** (-2 * i / 8) for i in range(4)]])
    c = decode.QWEN3_4B
    assert all(torch.equal(a, b) for a, b in zip(paged.rotary_tables(300, c.head_dim, c.rope_theta), decode.rope_tables(c, 300, "cpu")))


def test_rotary_tables_for_longer_contexts():
    original, factor, low, high = 8192, 8.0, 1.0, 4.0

    def bands(i, v):
        wave = 2 * math.pi / v
        if wave < original / high:
            return v
        if wave > original / low:
            return v / factor
        smooth = (original / wave - low) / (high - low)
        return (1 - smooth) * v / factor + smooth * v

    same(paged.rotary_tables(64, 128, 5e5, kind="bands", factor=factor, original=original, low=low, high=high), angles(64, 128, 5e5, bands))
    theta, width, original, factor = 1e6, 128, 32768, 4.0
    at = lambda turns: width * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    first, last = max(math.floor(at(32)), 0), min(math.ceil(at(1)), width - 1)

    def ramp(i, v):
        r = min(max((i - first) / (last - first), 0), 1)
        return v / factor * r + v * (1 - r)

    same(paged.rotary_tables(64, width, theta, kind="ramp", factor=factor, original=original, low=1.0, high=32.0), angles(64, width, theta, ramp), 0.1 * math.log(factor) + 1)


def test_rotary_tables_refuse():
    for bad in (dict(width=0), dict(width=7), dict(positions=0), dict(theta=0.0), dict(theta=math.nan), dict(kind="other"), dict(kind="linear", factor=0.5), dict(kind="linear", factor=math.nan), dict(kind="bands", factor=2),
                dict(kind="ramp", factor=2, original=0), dict(kind="bands", factor=2, original=100, low=4.0, high=1.0), dict(kind="theta", width=2, factor=2)):
        with pytest.raises(ValueError):
            paged.rotary_tables(**({"positions": 4, "width": 8} | bad))


def test_a_beam_decoder_refuses_what_it_cannot_do():
    from types import SimpleNamespace

    model = SimpleNamespace(c=decode.ModelConfig("small", 2, 64, 128, 2, 1, 64, 100, 1e4, False), device=torch.device("cpu"), nl=2)
    good = dict(batch=2, beams=3, max_prompt=20, max_new=5)
    for bad in (dict(batch=0), dict(beams=0), dict(beams=65), dict(max_prompt=0), dict(max_new=0), dict(page=0), dict(end=100), dict(end=-1)):
        with pytest.raises(ValueError):
            decode.BeamDecoder(model, **(good | bad))
    d = decode.BeamDecoder(model, **good, page=4)
    assert d.columns == 7 and d.k.shape == (2, 2 * 5 + 6 * 3, 1, 4, 64)
    for bad in ([torch.zeros(3, dtype=torch.int64)], [torch.zeros(3, dtype=torch.int64), torch.zeros(21, dtype=torch.int64)], [torch.zeros(0, dtype=torch.int64)] * 2):
        with pytest.raises(ValueError, match="prompts"):
            d.prefill(bad)
    for n in (0, 6):
        with pytest.raises(ValueError, match="new tokens"):
            d.generate([torch.zeros(3, dtype=torch.int64)] * 2, n)
