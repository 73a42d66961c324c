"""The paged operators as a decoder uses them together: beam search for a batch of prompts. The beams' hidden states against a plain
fp32 torch forward of the same architecture over each beam's own tokens (the bars of the one-token decoder: the final normed
hidden state within 2e-3 relative L2, the logits within 5e-3); the choices against a search over the decoder's own logits in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

from pingala8_llm_b200 import decode, synth  # noqa: E402
from pingala8_llm_b200.ops import device_error  # noqa: E402
from oracle.oracle import Oracle  # noqa: E402

CFG = decode.ModelConfig("qwen3-4b-2l", 2, 2560, 9728, 32, 8, 128, 4096, 1e6, True)


def rel(a, b):
    a, b = a.double(), b.double()
    return float((a - b).norm() / b.norm())


@pytest.fixture(scope="module")
def model_and_ref():
    slots = [{n: synth.make_slot(r, k, seed=100 * L + i, nd=3) for i, (n, r, k) in enumerate(decode.proj_shapes(CFG))} for L in range(CFG.layers)]
    m = decode.Model(CFG, seed=1, slots=slots)
    W = [{n: torch.from_numpy(Oracle(slots[L][n], r, k).dequant()).cuda() for n, r, k in decode.proj_shapes(CFG)} for L in range(CFG.layers)]
    return m, W, [(ly["attn_norm"], ly["ffn_norm"], ly["qk_norm"]) for ly in m.layers]


def prompts_of(*lens, seed=5):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return [torch.randint(0, CFG.vocab, (n,), device="cuda", generator=g) for n in lens]


class Search:
    """the same search over given logits, its beams as (score, tokens, whether it has ended)"""

    def __init__(self, batch, beams, end):
        self.beams, self.end = beams, end
        self.groups = [[(0.0, (), False)] for _ in range(batch)]

    def choose(self, logits):
        for b, group in enumerate(self.groups):
            every = []
            for w, (score, said, ended) in enumerate(group):
                if ended:
                    every.append((-score, w, 0, said + (self.end,), True))
                    continue
                p = score + torch.log_softmax(logits[b, w].double(), -1)
                val, tok = torch.sort(p, descending=True, stable=True)
                every += [(-v, w, i, said + (t,), t == self.end) for i, (v, t) in enumerate(zip(val[:self.beams].tolist(), tok[:self.beams].tolist()))]
            every.sort(key=lambda c: c[:3])
            self.groups[b] = [(-c[0], c[3], c[4]) for c in every[:self.beams]]


@pytest.mark.parametrize("dtype,beams,page,end", [(torch.float16, 4, 16, None), (torch.float32, 3, 8, 7), (torch.bfloat16, 5, 24, None)])
def test_the_search_is_that_over_its_own_logits_and_every_beam_has_its_own_history(model_and_ref, dtype, beams, page, end):
    m, W, norms = model_and_ref
    prompts, n_new = prompts_of(45, 16, 33), 9
    d = decode.BeamDecoder(m, 3, beams, 48, 12, dtype=dtype, page=page, end=end)
    if end is not None:  # make the token that ends a sequence a likely one
        d.m.head_w[end] += 0.5 * d.m.head_w[11]
    search = Search(3, beams, end)
    try:
        d.prefill(prompts)
        search.choose(d.logits)
        for i in range(n_new - 1):
            tokens = d.history(i + 1)  # what the beams are before this step
            d.step()
            logits, hidden = d.logits.clone(), d.hidden.view(3, beams, -1).clone()
            search.choose(logits)
            if i in (0, n_new - 2):
                bar = 2e-3 if dtype != torch.bfloat16 else 1.6e-2  # keys and values of 8 bits: eight times fp16's
                for b in range(3):
                    for w in range(beams):
                        _, hid = decode.reference_forward(CFG, W, norms, m.embed, m.head, m.final_norm, torch.cat([prompts[b], tokens[b, w]]))
                        assert rel(hidden[b, w], hid[-1]) < bar, (i, b, w)
    finally:
        if end is not None:
            d.m.head_w[end] = d.m.head.dequant(torch.tensor([end], device="cuda"))[0].half()
    assert device_error() == 0
    got, scores = d.history(n_new).tolist(), d.scores.tolist()
    for b, group in enumerate(search.groups):
        assert [tuple(t) for t in got[b]] == [said for _, said, _ in group]
        assert all(abs(x - s) <= 1e-5 * (1 + abs(s)) * n_new for x, (s, _, _) in zip(scores[b], group))
        if end is not None:
            assert d.done[b].tolist() == [e for _, _, e in group]


def test_generate_captured_is_generate_not_captured(model_and_ref):
    m = model_and_ref[0]
    d = decode.BeamDecoder(m, 2, 4, 40, 20)
    a = d.generate(prompts_of(40, 3), 20, graph=False)
    b = d.generate(prompts_of(40, 3), 20)
    c = d.generate(prompts_of(40, 3), 20)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(b[0], c[0]) and torch.equal(b[1], c[1])
    assert (a[1][:, :-1] >= a[1][:, 1:]).all() and device_error() == 0
    other = d.generate(prompts_of(12, 31, seed=6), 7)  # other lengths through the same graph
    again = decode.BeamDecoder(m, 2, 4, 40, 7).generate(prompts_of(12, 31, seed=6), 7, graph=False)
    assert torch.equal(other[0], again[0]) and torch.equal(other[1], again[1]) and device_error() == 0


def test_one_beam_is_greedy_decoding(model_and_ref):
    """where no two logits are nearer than the rounding of products of other widths"""
    m = model_and_ref[0]
    prompt = prompts_of(37, seed=8)[0]
    tokens, _ = decode.BeamDecoder(m, 1, 1, 37, 12, dtype=torch.float32).generate([prompt], 12)
    want, logits, _ = m.generate(prompt, 12)
    for i, lg in enumerate(logits):
        top = torch.topk(lg, 2).values
        if float(top[0] - top[1]) < 2e-2:
            break
        assert int(tokens[0, 0, i]) == int(want[i])


def test_stretched_positions(model_and_ref):
    m = model_and_ref[0]
    d = decode.BeamDecoder(m, 1, 3, 20, 4, rotary={"kind": "ramp", "factor": 4.0, "original": 4096, "low": 1.0, "high": 32.0})
    plain = decode.BeamDecoder(m, 1, 3, 20, 4)
    a, b = d.generate(prompts_of(20), 4), plain.generate(prompts_of(20), 4)
    assert not torch.equal(a[1], b[1])  # the angles are others
    assert math.isfinite(float(a[1].sum())) and device_error() == 0


@pytest.mark.parametrize("page", [4, 16])
def test_steps_beyond_the_longest_continuation_are_left_out_and_reported(model_and_ref, page):
    d = decode.BeamDecoder(model_and_ref[0], 2, 3, 40, 5, page=page)
    prompts = prompts_of(40, 3)
    d.generate(prompts, 5, graph=False)
    tokens, scores = d.generate(prompts, 5)
    assert device_error() == 0
    said = d.history(5)
    pages = d.k[:, :2 * d._shared].clone()  # the prompts'
    for _ in range(2 * page + 3):
        d.graph.replay()
    torch.cuda.synchronize()
    assert device_error() & 64
    assert torch.equal(d.k[:, :2 * d._shared], pages)
    for n in (0, 6):
        with pytest.raises(ValueError):
            d.history(n)
    again = d.generate(prompts, 5)
    assert torch.equal(said, tokens) and torch.equal(again[0], tokens) and torch.equal(again[1], scores) and device_error() == 0
