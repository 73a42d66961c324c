"""What a bounded decoder keeps, and what its drafts give: the masses that it adds up, the slots that an eviction leaves, the pass
after it, and the passes that right, wrong and no drafts take, against plain torch on the same layers."""
import os
import sys

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

from pingala8_llm_b200 import cache, decode, synth  # noqa: E402
from pingala8_llm_b200.ops import device_error  # noqa: E402

CFG = decode.ModelConfig("qwen3-4b-2l", 2, 2560, 9728, 32, 8, 128, 4096, 1e6, True)
G = CFG.heads // CFG.kv_heads
E = 2.0 ** -23


@pytest.fixture(scope="module")
def model():
    slots = [{n: synth.make_slot(r, k, seed=100 * L + i, nd=3) for i, (n, r, k) in enumerate(decode.proj_shapes(CFG))} for L in range(CFG.layers)]
    return decode.Model(CFG, seed=1, slots=slots)


def prompt_of(n, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randint(0, CFG.vocab, (n,), device="cuda", generator=g)


def bounded(model, slack=32, dtype=torch.float16):
    return decode.TreeDecoder(model, 600, dtype=dtype, budget=96, sinks=4, recent=16, slack=slack)


def masses(d, n):
    return d.mass[:, 0, :, :n].double()


def test_masses_are_the_tokens_weights(model):
    """before an eviction: every token and head gives one weight in all, over the slots up to its own. A score of 128 products is off by
    at most 144 e A (A = |q||k| scale, |q| and |k| as the norms leave them: at most sqrt(128) times the largest norm weight 1.1, so
    A <= 128 * 1.21 / sqrt(128) < 14), the sum of up to 128 of them by a step each"""
    d = bounded(model)
    prompt = prompt_of(100, 1)
    d.prefill(prompt)
    assert d.used == 100 and device_error() == 0
    got = masses(d, 100)
    assert float((got.sum(-1) - 100 * G).abs().max()) <= 100 * G * (2 * 144 * E * 14 + 128 * E)
    assert float(got.min()) > 0
    # slot by slot: later tokens alone add to it, one token's weights at a time
    assert float((got[..., -1] - got[..., -1].clamp(max=G)).abs().max()) == 0  # the last slot was seen by the last token's heads alone
    # through a tree: the tokens on the confirmed path count, the others do not
    last = int(torch.argmax(d.prefill(prompt_of(1, 2))))
    one = masses(d, 101).sum(-1)
    nxt = int(d.step(torch.tensor([last], device="cuda"), torch.tensor([-1], dtype=torch.int32, device="cuda"))[-1])
    two = masses(d, 102).sum(-1)
    wrong = (nxt + 1) % CFG.vocab
    got = d.step(torch.tensor([nxt, wrong, wrong, wrong], device="cuda"), torch.tensor([-1, 0, 0, 1], dtype=torch.int32, device="cuda"))
    assert device_error() == 0
    n = got.numel()
    tol = 110 * G * (2 * 144 * E * 14 + 128 * E)
    assert float((two - one - G).abs().max()) <= tol and d.used == 102 + n
    assert float((masses(d, 102 + n).sum(-1) - two - n * G).abs().max()) <= tol


def test_an_eviction_keeps_the_heaviest_and_the_next_pass_attends_to_them(model):
    """the kept slots are those of the masses before it, with their keys, values and masses; the pass after it gives what plain attention
    over the kept rows gives"""
    d, full = bounded(model, slack=0), bounded(model, slack=500)
    prompt = prompt_of(150, 3)  # passes of 64, 64 and 22 tokens: cut after the second and the third
    seen = []
    for x in (d, full):
        x.prefill(prompt[:64])
    assert d.used == full.used == 64
    for x in (d, full):
        x.prefill(prompt[64:128])
    assert (d.used, full.used) == (96, 128) and device_error() == 0
    for L in range(2):
        for h in range(CFG.kv_heads):
            m = full.mass[L, 0, h, :128].tolist()
            mid = sorted(range(4, 112), key=lambda j: (-m[j], j))[:76]
            keep = sorted(list(range(4)) + mid + list(range(112, 128)))
            seen.append(len(set(keep) - set(range(32, 128))))
            at = torch.tensor(keep, device="cuda")
            assert torch.equal(d.k[L, 0, h, :96], full.k[L, 0, h, at]) and torch.equal(d.v[L, 0, h, :96], full.v[L, 0, h, at])
            assert torch.equal(d.mass[L, 0, h, :96], full.mass[L, 0, h, at])
    assert max(seen) > 4  # (the choice is no plain window)
    # the next pass, layer by layer in torch on what the decoder's own projections give, over the kept rows
    k0, v0, part = d.k.clone(), d.v.clone(), prompt[128:]
    mask, depth = cache.tree_plan(torch.arange(-1, 21, device="cuda"))
    logits = d.forward(part, mask, depth)
    want = plain_pass(model, d, k0, v0, 96, part)
    assert device_error() == 0
    # the pass's keys, values and queries are those of the same products, rounded to fp16 alike but for the last step; weights are fp16:
    # a few parts in 2^11 of the attention's output, which reaches the logits through one more layer
    assert float((logits - want).norm() / want.norm()) < 5e-3
    wrong = plain_pass(model, d, full.k[..., :96, :], full.v[..., :96, :], 96, part)  # as if the first 96 had been kept
    assert float((logits - wrong).norm() / wrong.norm()) > 2e-2


def plain_pass(model, d, k, v, n, tokens):
    """logits of `tokens` behind n kept slots: the projections as the decoder calls them, attention in torch"""
    c, T = CFG, tokens.numel()
    x = model.embed.dequant(tokens)
    cos, sin = d.cos[128:128 + T], d.sin[128:128 + T]
    for L, layer in enumerate(model.layers):
        t = layer["t"]
        q, kk, vv = decode.mul_mat_group([t["q"], t["k"], t["v"]], x, norm_weight=layer["attn_norm"], eps=c.eps)
        q, kk = (decode.apply_rope(decode.rms(y.view(T, -1, c.head_dim).transpose(0, 1), w, c.eps), cos, sin).half().float() for y, w in ((q, layer["qk_norm"][0]), (kk, layer["qk_norm"][1])))
        keys = torch.cat([k[L, 0, :, :n].float(), kk], 1).repeat_interleave(G, 0)
        vals = torch.cat([v[L, 0, :, :n].float(), vv.view(T, -1, c.head_dim).transpose(0, 1).half().float()], 1).repeat_interleave(G, 0)
        s = (q @ keys.transpose(-1, -2)) / c.head_dim ** 0.5
        s = s.masked_fill(~torch.ones(T, n + T, dtype=torch.bool, device="cuda").tril(n), float("-inf"))
        a = (torch.softmax(s, -1) @ vals).transpose(0, 1).reshape(T, -1)
        h = x + t["o"].mul_mat(a.contiguous())
        g, u = decode.mul_mat_group([t["gate"], t["up"]], h, norm_weight=layer["ffn_norm"], eps=c.eps)
        x = h + t["down"].mul_mat(g, up=u)
    return (decode.rms(x, model.final_norm, c.eps).half() @ model.head_w.T).float()


def test_right_wrong_and_no_drafts(model):
    """with the known continuation drafted seven tokens a pass are taken; with wrong drafts or none, one. A tie within the rounding of another number
    of columns may part two runs, so the right drafts are made from the run that confirms them"""
    d = decode.TreeDecoder(model, 200, dtype=torch.float32)
    prompt = prompt_of(40, 4)
    plain, passes = d.generate(prompt, 25, draft=lambda h: ([h[-1]], [-1]))
    assert passes == 24 and plain.numel() == 25 and plain.dtype == torch.int64
    seq = prompt.tolist() + plain.tolist()

    def known(history):
        rest = seq[len(history) - 1:len(history) + 5] if history == seq[:len(history)] else history[-1:]
        return rest, list(range(-1, len(rest) - 1))

    toks, passes = d.generate(prompt, 25, draft=known)
    same = next((i for i, (a, b) in enumerate(zip(toks.tolist(), plain.tolist())) if a != b), 25)
    # each pass takes six drafted tokens or, where the two runs part, as many as they share; after that one
    assert same == 25 and passes == 4 or same >= 7 and passes <= 24 - 5 * ((same - 1) // 6)

    def bad(history):
        return [history[-1]] + [(x + 1) % CFG.vocab for x in seq[len(history):len(history) + 3]], [-1, 0, 1, 2][:1 + len(seq[len(history):len(history) + 3])]

    toks, passes = d.generate(prompt, 6, draft=bad)
    assert toks.tolist() == plain[:6].tolist() and passes == 5
    assert device_error() == 0


def test_generate_nothing(model):
    d = decode.TreeDecoder(model, 60, dtype=torch.float16)
    toks, passes = d.generate(prompt_of(20, 5), 0)
    assert toks.shape == (0,) and toks.dtype == torch.int64 and passes == 0
    for n in (-1, 41):
        with pytest.raises(ValueError, match="max_len"):
            d.generate(prompt_of(20, 5), n)
