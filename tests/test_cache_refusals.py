"""What the key/value cache operators refuse before they touch a device, and what they do not. The C entries get addresses that
nothing may read: without a GPU a call that is not refused ends at its launch, with another status than P8_ERR_ARG."""
import os
import random
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

import pingala8_llm_b200 as p8  # noqa: E402
from test_cache_ops import ARG, PTR, UNSUPPORTED, accept_args, append_args, attn_args, evict_args, kv, mass_args  # noqa: E402

if torch.cuda.is_available():
    pytest.skip("addresses that nothing may read: not where a launch would reach a GPU", allow_module_level=True)

MB = 1 << 20


@pytest.mark.parametrize("ns", [-1, 1 << 32, -(1 << 62)])
def test_a_wait_limit_out_of_range(ns):
    assert p8.lib().p8_cache_wait_limit(ns) == ARG


def places(at, dims, strides, last):
    """the addresses of 4-byte values"""
    rows = [at]
    for d, s in zip(dims, strides):
        rows = [r + 4 * s * i for r in rows for i in range(d)]
    return {r + 4 * j for r in rows for j in range(last)}


def test_buffers_that_share_memory_are_refused_and_those_that_lie_between_one_another_are_not():
    """masses and their sums, small strided views of one buffer, against all their addresses"""
    rng = random.Random(1)
    refused = taken = between = 0
    for _ in range(3000):
        b, h, n = rng.randint(1, 4), rng.randint(1, 4), rng.randint(1, 6)
        inner = n + rng.choice([0, 0, 1, rng.randint(0, 12)])
        if rng.random() < 0.5:
            os_ = (inner * h + rng.randint(0, 9), inner)
        else:
            os_ = (inner, inner * b + rng.randint(0, 9))
        ms = os_ if rng.random() < 0.5 else (rng.randint(1, 60), rng.randint(1, 60))
        base = 50 * MB
        off = rng.randint(-80, 80)
        x, y = places(base, (b, h), os_, n), places(base + 4 * off, (b, h), ms, n)
        one = off == 0 and (b == 1 or ms[0] == os_[0]) and (h == 1 or ms[1] == os_[1])
        st = p8.lib().p8_attn_mass(kv(batch=b, heads=h, slots=n), mass_args(heads=2 * h, qs=(2 * h * 2 * 64, 2 * h * 64, 64), q=4 * MB, out=base, os=os_, mass=base + 4 * off, ms=ms,
                                                                         lens=100 * MB, lse=101 * MB), None)
        assert st != 0
        assert (st == ARG) == (bool(x & y) and not one), (b, h, n, os_, ms, off)
        refused += st == ARG
        taken += st != ARG
        between += st != ARG and not one and min(x) < max(y) and min(y) < max(x)
    assert min(refused, taken, between) > 200


def test_interleaved_buffers_are_taken():
    """queries and outputs side by side in one buffer; a cache's two halves in turn, layer by layer"""
    L, c = p8.lib(), kv()
    side = dict(qs=(1024, 512, 128), os=(1024, 512, 128))
    assert L.p8_tree_attn(c, attn_args(out=4 * PTR + 128, lens=100 * MB, **side), 200 * MB, 1 << 40, None) != ARG
    assert L.p8_tree_attn(c, attn_args(out=4 * PTR + 64, lens=100 * MB, **side), 200 * MB, 1 << 40, None) == ARG
    assert L.p8_tree_attn(c, attn_args(out=4 * PTR - 112, lens=100 * MB, **side), 200 * MB, 1 << 40, None) == ARG
    heads = 2 * 64 * 64  # 2 heads x 64 slots x 64, as many bytes as 2 sequences' 16-bit halves
    st = (4 * heads, 2 * heads, 64 * 64, 64)
    src, dst = kv(k=16 * MB, v=32 * MB, layers=2, ks=(8 * heads, *st[1:]), vs=(8 * heads, *st[1:])), kv(k=16 * MB + 4 * heads * 2, v=32 * MB + 4 * heads * 2, layers=2, ks=(8 * heads, *st[1:]), vs=(8 * heads, *st[1:]))
    args = dict(mass=48 * MB, ms=(512, 128, 64), out=48 * MB + 4 * 256, os=(512, 128, 64), lens=100 * MB, new=101 * MB, kept=102 * MB)
    assert L.p8_kv_evict(src, dst, evict_args(**args), None) != ARG
    assert L.p8_kv_evict(src, dst, evict_args(**{**args, "out": 48 * MB + 4 * 255}), None) == ARG
    assert L.p8_kv_evict(src, kv(k=16 * MB + 2 * (2 * heads + 64 * 64), v=32 * MB + 4 * heads * 2, layers=2, ks=(8 * heads, *st[1:]), vs=(8 * heads, *st[1:])), evict_args(**args), None) == ARG


def accept(cache=None, **o):
    at = dict(tokens=50 * MB, target=51 * MB, parents=52 * MB, lens=53 * MB, counts=54 * MB, path=55 * MB, accepted=56 * MB, new=57 * MB, next=58 * MB) | o
    return p8.lib().p8_tree_accept(cache or kv(), accept_args(**at), None)


def test_accept_refuses_results_over_its_inputs():
    """two sequences, four tokens: the tree is 64 bytes of tokens and of targets and 32 of parents, lengths are 8 bytes"""
    assert accept() != ARG and accept(counts=0) != ARG
    assert accept(accepted=54 * MB + 8, path=52 * MB + 32, new=53 * MB + 8, next=51 * MB + 64) != ARG  # right behind one another
    for bad in (dict(accepted=54 * MB), dict(accepted=54 * MB + 4), dict(accepted=53 * MB), dict(path=52 * MB), dict(path=52 * MB + 28), dict(path=50 * MB + 60), dict(new=53 * MB),
                dict(new=53 * MB + 4), dict(new=53 * MB - 4), dict(new=54 * MB), dict(next=51 * MB + 56), dict(next=50 * MB), dict(next=58 * MB, new=58 * MB + 12),
                dict(accepted=57 * MB), dict(path=56 * MB - 28), dict(path=PTR), dict(next=2 * PTR + 2 * 2 * 64 * 64 * 2 - 8), dict(lens=PTR + 4096)):
        assert accept(**bad) == ARG, bad
    assert accept(kv(k=PTR, v=PTR)) == ARG and accept(kv(k=PTR, v=PTR + 4096)) == ARG  # keys and values over one another
    turns = (2 * 2 * 64 * 64 * 2, 2 * 64 * 64 * 2, 64 * 64 * 2, 64 * 2)
    assert accept(kv(k=PTR, v=PTR + 128, ks=turns, vs=turns)) != ARG  # and side by side in every slot


def evict(src=None, dst=None, **o):
    at = dict(mass=48 * MB, out=48 * MB, lens=53 * MB, new=54 * MB, kept=55 * MB) | o
    src = src or kv(k=16 * MB, v=32 * MB)
    return p8.lib().p8_kv_evict(src, dst or src, evict_args(**at), None)


def test_evict_refuses_results_over_its_inputs():
    """two sequences of two heads, 64 slots cut to 8: lengths are 8 bytes, kept slots 128, masses 1,024 (in rows of 256)"""
    other = kv(k=64 * MB, v=80 * MB)
    assert evict() != ARG and evict(dst=other, out=49 * MB) != ARG
    assert evict(new=53 * MB + 8, kept=53 * MB - 128) != ARG
    for bad in (dict(new=53 * MB), dict(new=53 * MB + 4), dict(new=53 * MB - 4), dict(kept=53 * MB), dict(kept=53 * MB - 124), dict(kept=54 * MB + 4), dict(new=55 * MB + 124),
                dict(kept=48 * MB + 1020), dict(new=48 * MB), dict(kept=16 * MB), dict(new=32 * MB), dict(lens=48 * MB), dict(lens=16 * MB + 4)):
        assert evict(**bad) == ARG, bad
        if not {48 * MB, 16 * MB, 32 * MB} & {x // 4096 * 4096 for x in bad.values()}:
            assert evict(dst=other, out=49 * MB, **bad) == ARG, bad
    one = kv(k=16 * MB, v=16 * MB)
    assert evict(one) == ARG  # keys and values in one place, cut in place
    assert evict(one, other, out=49 * MB) != ARG  # read from one place
    assert evict(dst=kv(k=64 * MB, v=64 * MB), out=49 * MB) == ARG  # written to one place
    assert evict(dst=other, out=64 * MB) == ARG and evict(dst=other, out=16 * MB) == ARG
    assert evict(dst=kv(k=32 * MB, v=80 * MB), out=49 * MB) == ARG


def append(cache=None, **o):
    at = dict(q=50 * MB, k=51 * MB, v=52 * MB, lens=53 * MB, counts=54 * MB, pos=55 * MB, cos=56 * MB, sin=57 * MB, qn=58 * MB, kn=59 * MB, out=60 * MB) | o
    return p8.lib().p8_kv_append(cache or kv(), append_args(**at), None)


def test_append_refuses_results_over_its_inputs():
    """two sequences of two tokens: q is 4,096 bytes and its 16-bit result 2,048, k and v are 2,048 each, tables 10 x 128"""
    assert append() != ARG and append(qn=0, kn=0, counts=0) != ARG
    for bad in (dict(out=51 * MB), dict(out=51 * MB + 2032), dict(out=52 * MB), dict(out=50 * MB), dict(out=53 * MB), dict(out=54 * MB - 2032), dict(out=55 * MB), dict(out=56 * MB + 1264),
                dict(out=57 * MB), dict(out=58 * MB), dict(out=59 * MB + 240), dict(out=PTR), dict(out=2 * PTR + 32752), dict(k=PTR), dict(v=PTR + 128), dict(q=2 * PTR), dict(lens=PTR),
                dict(cos=2 * PTR), dict(qn=PTR + 256)):
        assert append(**bad) == ARG, bad
    assert append(out=51 * MB + 2048, qn=59 * MB + 256) != ARG
    assert append(kv(k=PTR, v=PTR)) == ARG and append(kv(k=PTR, v=PTR + 64)) == ARG
    wide = kv(type=0)
    assert append(wide, out=50 * MB) != ARG  # in place
    for bad in (dict(k=50 * MB), dict(v=50 * MB + 2048), dict(cos=50 * MB), dict(out=50 * MB + 16), dict(os=(512, 256, 128))):
        assert append(wide, **{"out": 50 * MB, **bad}) == ARG, bad
    # queries, keys and values as one product leaves them, the queries in place
    packed = dict(q=50 * MB, k=50 * MB + 1024, v=50 * MB + 1536, qs=(1024, 512, 64), ks=(1024, 512, 64), vs=(1024, 512, 64))
    assert append(wide, out=50 * MB, os=(1024, 512, 64), **packed) != ARG
    assert append(wide, out=50 * MB, os=(1024, 512, 64), **{**packed, "k": 50 * MB + 1008}) == ARG


def attend(cache=None, ws=70 * MB, **o):
    at = dict(q=50 * MB, lens=53 * MB, counts=54 * MB, mask=55 * MB, ms=2, out=60 * MB, lse=61 * MB) | o
    return p8.lib().p8_tree_attn(cache or kv(), attn_args(**at), ws, 8 * MB, None)


def test_attention_refuses_results_over_its_inputs():
    """two sequences of two tokens and four heads of 64: q and out are 2,048 bytes, lse 64, masks 32"""
    assert attend() != ARG and attend(mask=0, counts=0, lse=0) != ARG and attend(kv(k=PTR, v=PTR)) != ARG
    for bad in (dict(out=50 * MB), dict(out=50 * MB + 2032), dict(out=53 * MB), dict(out=54 * MB - 2032), dict(out=55 * MB + 16), dict(out=61 * MB + 48), dict(lse=60 * MB + 2044), dict(lse=50 * MB),
                dict(lse=PTR), dict(lse=2 * PTR + 4), dict(lse=53 * MB + 4), dict(lse=55 * MB - 60), dict(ws=50 * MB), dict(ws=60 * MB), dict(ws=61 * MB), dict(ws=PTR), dict(ws=53 * MB),
                dict(ws=54 * MB), dict(ws=55 * MB)):
        assert attend(**bad) == ARG, bad
    assert attend(out=50 * MB + 2048, lse=55 * MB + 32) != ARG and attend(ms=0, lse=55 * MB + 16) != ARG


def weigh(cache=None, **o):
    at = dict(q=50 * MB, lse=52 * MB, lens=53 * MB, counts=54 * MB, rows=55 * MB, mass=60 * MB, out=60 * MB) | o
    return p8.lib().p8_attn_mass(cache or kv(), mass_args(**at), None)


def test_mass_refuses_results_over_its_inputs():
    """masses are 1,024 bytes, the two tokens' rows of two sequences 16"""
    assert weigh() != ARG and weigh(out=61 * MB) != ARG and weigh(counts=0, rows=0) != ARG
    for bad in (dict(q=60 * MB), dict(lse=60 * MB + 1020), dict(lse=60 * MB - 60), dict(lens=60 * MB), dict(counts=60 * MB + 512), dict(rows=60 * MB - 12), dict(out=52 * MB + 60), dict(out=PTR),
                dict(out=PTR + 2 * 2 * 64 * 64 * 2 - 4), dict(out=55 * MB + 12)):
        assert weigh(**bad) == ARG, bad
    assert weigh(out=52 * MB + 64) != ARG and weigh(out=55 * MB + 16) != ARG


def test_outputs_whose_rows_share_memory_are_refused():
    """a stride of nothing (a tensor expanded over its sequences), or one that does not step over the rows between"""
    for st in ((0, 64), (128, 0), (0, 0), (64, 64), (32, 64), (100, 64), (64, 100)):
        assert weigh(os=st, out=61 * MB) == ARG and weigh(ms=st, os=st) == ARG, st
        assert weigh(ms=st, out=61 * MB) != ARG, st  # read alone
    assert weigh(os=(64, 128), out=61 * MB) != ARG and weigh(os=(67, 200), out=61 * MB) != ARG
    heads = 64 * 64
    for ks in ((0, 2 * heads, 64, 64), (0, heads, heads, 64), (0, 2 * heads, heads, 32), (0, 128, 64, 64)):
        c = kv(ks=ks)
        assert append(c) == ARG and accept(c) == ARG and evict(kv(k=16 * MB, v=32 * MB, ks=ks)) == ARG, ks
        assert evict(kv(k=16 * MB, v=32 * MB, ks=ks), kv(k=64 * MB, v=80 * MB), out=49 * MB) != ARG, ks  # read alone
        assert attend(c) != ARG, ks
    assert append(kv(ks=(0, 64, 128, 256))) != ARG  # slots before heads before sequences
    assert append(os=(512, 64, 64)) == ARG and attend(os=(256, 256, 64)) == ARG and attend(os=(64, 128, 256)) != ARG
    assert evict(ms=(256, 128, 0), os=(256, 128, 0)) == ARG and evict(ms=(256, 0, 64), os=(256, 0, 64)) == ARG and evict(ms=(0, 128, 64), os=(0, 128, 64)) != ARG


def test_scales_that_32_bits_do_not_hold_are_refused():
    for scale in (1e39, -1e300, 3e38, -2.4e38, float("inf"), float("nan")):
        assert attend(scale=scale) == ARG and weigh(scale=scale) == ARG, scale
    for scale in (2.3e38, -2.3e38, 0.0, 1e-300, -0.5):
        assert attend(scale=scale) != ARG and weigh(scale=scale) != ARG, scale


def test_append_of_no_tokens_is_a_call_that_does_nothing():
    nothing = dict(tokens=0, q=0, k=0, v=0, out=0, pos=0)
    assert append(**nothing) == 0 and append(**nothing, lens=0, cos=0, sin=0) == 0
    assert append(kv(width=96), **nothing) == ARG and append(**nothing, heads=3) == ARG and append(**{**nothing, "tokens": -1}) == ARG


def test_evict_takes_more_rows_than_a_grid_is_high():
    many = dict(layers=80, batch=128, heads=8, slots=8)
    st = tuple(64 * x for x in (128 * 8 * 8, 8 * 8, 8, 1))
    src, dst = kv(k=1 << 32, v=2 << 32, ks=st, vs=st, **many), kv(k=3 << 32, v=4 << 32, ks=st, vs=st, **many)
    far = dict(mass=5 << 32, ms=(128 * 64, 64, 8), os=(128 * 64, 64, 8), kept=6 << 32, sinks=1, recent=1, budget=4)
    assert evict(src, **far, out=5 << 32) not in (ARG, UNSUPPORTED) and evict(src, dst, **far, out=7 << 32) not in (ARG, UNSUPPORTED)
    # 2^30 rows of 64 blocks are more than a grid has at all
    huge = dict(layers=1024, batch=4096, heads=256, slots=2048)
    st = tuple(64 * x for x in (4096 * 256 * 2048, 256 * 2048, 2048, 1))
    src, dst = kv(k=1 << 48, v=1 << 52, ks=st, vs=st, **huge), kv(k=1 << 53, v=1 << 54, ks=st, vs=st, **huge)
    far = dict(mass=1 << 55, ms=(4096 * 256 * 2048, 256 * 2048, 2048), os=(4096 * 256 * 2048, 256 * 2048, 2048), kept=1 << 56, budget=2048)
    assert evict(src, dst, **far, out=1 << 57) == UNSUPPORTED


def test_a_decoder_refuses_a_budget_that_its_first_eviction_could_not_keep():
    from types import SimpleNamespace

    from pingala8_llm_b200 import decode

    model = SimpleNamespace(c=decode.ModelConfig("small", 2, 64, 128, 2, 1, 64, 100, 1e4, False), device=torch.device("cpu"), nl=2)
    for bad in (dict(budget=64), dict(budget=0, sinks=0, recent=0), dict(budget=-1, sinks=0, recent=0), dict(budget=100, sinks=-1), dict(budget=100, recent=-1), dict(budget=100, slack=-1),
                dict(budget=100, sinks=50, recent=51)):
        with pytest.raises(ValueError, match="budget"):
            decode.TreeDecoder(model, 500, **bad)
    assert decode.TreeDecoder(model, 500, budget=68, sinks=4, recent=64, slack=0).k.shape == (2, 1, 1, 132, 64)
    assert decode.TreeDecoder(model, 500).mass is None


def test_the_decoder_without_the_cache_operators_module():
    """decode and its Model import where _cache_calls was not built; TreeDecoder says what is missing"""
    import subprocess

    code = """
import sys
sys.modules["pingala8_llm_b200._cache_calls"] = None
from pingala8_llm_b200 import decode
assert decode.Model and decode.lookup_draft([1, 2, 3]) == ([3], [-1])
try:
    decode.TreeDecoder(None, 10)
except ImportError as e:
    assert "pingala8_llm_b200.build" in str(e)
    print("named")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    assert subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, check=True).stdout == "named\n"
