"""The cache operators as a decoder uses them together: drafted trees, their acceptance, and a bounded cache, against a plain
fp32 torch forward of the same architecture (the bars of the one-token decoder: the final normed hidden state within 2e-3
relative L2, the logits within 5e-3)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

from pingala8_llm_b200 import cache, decode, synth  # noqa: E402
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


def ref(model_and_ref, seq):
    m, W, norms = model_and_ref
    return decode.reference_forward(CFG, W, norms, m.embed, m.head, m.final_norm, seq)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_a_tree_gives_every_branch_its_own_logits(model_and_ref, dtype):
    """each token of a tree has the logits of the sequence that its branch is"""
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    d = decode.TreeDecoder(model_and_ref[0], 200, dtype=dtype)
    prompt = torch.randint(0, CFG.vocab, (70,), device="cuda", generator=g)
    lg = d.prefill(prompt)
    want, _ = ref(model_and_ref, prompt)
    assert rel(lg, want[-1]) < 5e-3
    tokens = torch.randint(0, CFG.vocab, (9,), device="cuda", generator=g)
    parents = [-1, 0, 0, 1, 1, 2, 5, 6, 3]
    mask, depth = cache.tree_plan(torch.tensor(parents, device="cuda"))
    logits = d.forward(tokens, mask, depth)
    assert device_error() == 0
    for t in range(9):
        branch, c = [], t
        while c >= 0:
            branch.append(c)
            c = parents[c]
        want, hid = ref(model_and_ref, torch.cat([prompt, tokens[branch[::-1]]]))
        assert rel(d.hidden[t], hid[-1]) < 2e-3 and rel(logits[t], want[-1]) < 5e-3


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_steps_confirm_what_the_model_says(model_and_ref, dtype):
    """with the right continuation among the drafted branches it is taken at once, and the cache is then the sequence's"""
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    d = decode.TreeDecoder(model_and_ref[0], 200, dtype=dtype)
    prompt = torch.randint(0, CFG.vocab, (20,), device="cuda", generator=g)
    plain = []  # one token at a time
    nxt = torch.argmax(d.prefill(prompt))
    for _ in range(6):
        plain.append(int(nxt))
        nxt = d.step(nxt.view(1), torch.tensor([-1], dtype=torch.int32, device="cuda"))[-1]
    plain.append(int(nxt))
    one = d.k[:, :, :, :26].clone()
    d.reset()
    d.k.zero_()
    assert int(torch.argmax(d.prefill(prompt))) == plain[0]
    # the true path goes through nodes 0, 2, 4, 5, 7, 8; the others are wrong
    wrong = [(x + 1) % CFG.vocab for x in plain]
    tokens = [plain[0], wrong[1], plain[1], wrong[2], plain[2], plain[3], wrong[4], plain[4], plain[5]]
    parents = [-1, 0, 0, 2, 2, 4, 5, 5, 7]
    got = d.step(torch.tensor(tokens, device="cuda"), torch.tensor(parents, dtype=torch.int32, device="cuda"))
    assert device_error() == 0
    assert got.tolist() == plain[1:] and d.path.tolist() == [0, 2, 4, 5, 7, 8] and d.lens.tolist() == [26] and d.position == 26
    # the keys of one layer, written by a pass over nine tokens, are those of six passes over one (other products: the GEMM's
    # fp16 operands against the GEMV's 14-bit ones, two bars of 1e-3)
    assert rel(d.k[0, :, :, :26].float(), one[0].float()) < 2e-3


def test_generate_with_and_without_drafts(model_and_ref):
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    m = model_and_ref[0]
    prompt = torch.randint(0, CFG.vocab, (30,), device="cuda", generator=g)
    prompt = torch.cat([prompt, prompt, prompt[:7]])
    d = decode.TreeDecoder(m, 160, dtype=torch.float32)
    toks, passes = d.generate(prompt, 24)
    assert device_error() == 0 and toks.numel() == 24 and 1 <= passes <= 23
    seq = torch.cat([prompt, toks])
    want, _ = ref(model_and_ref, seq[:-1])
    # every token is the reference's choice, or its logit is within the bar of that choice's (the logits are off by at most
    # 5e-3 of their norm in all, each of the two values by less than that)
    for i, t in enumerate(toks.tolist()):
        row = want[prompt.numel() - 1 + i]
        assert float(row.max() - row[t]) <= 2 * 5e-3 * float(row.norm())


def test_lookup_draft_shares_beginnings():
    tokens, parents = decode.lookup_draft([5, 6, 7, 1, 5, 6, 8, 2, 5])
    assert tokens == [5, 6, 8, 2, 5, 7, 1, 5, 6, 8, 2] and parents[:6] == [-1, 0, 1, 2, 3, 1]
    assert decode.lookup_draft([1, 2, 3]) == ([3], [-1])
    assert len(decode.lookup_draft([1] * 100)[0]) <= 64


def test_a_bounded_cache_keeps_its_budget_and_its_positions(model_and_ref):
    """the cache stays within its slots, sinks and recent tokens stay, and the weights that were added up are the tokens'"""
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    m = model_and_ref[0]
    d = decode.TreeDecoder(m, 600, dtype=torch.float16, budget=96, sinks=4, recent=16, slack=32)
    prompt = torch.randint(0, CFG.vocab, (300,), device="cuda", generator=g)
    full = decode.TreeDecoder(m, 600, dtype=torch.float16)
    full.prefill(prompt)
    d.prefill(prompt)
    assert device_error() == 0
    assert d.k.shape[3] == 96 + 32 + 64 and d.used == int(d.lens[0]) <= 128 and d.position == 300
    # layer 0 sees no attention: its keys do not depend on what was evicted
    n = d.used
    assert torch.equal(d.k[0, :, :, :4], full.k[0, :, :, :4])
    assert torch.equal(d.k[0, :, :, n - 16:n], full.k[0, :, :, 284:300])
    G = CFG.heads // CFG.kv_heads
    assert float(d.mass[:, :, :, :n].min()) >= 0 and float(d.mass[:, :, :, :n].sum(-1).max()) <= 300 * G * 1.001
    toks, _ = d.generate(prompt, 100)
    assert toks.numel() == 100 and d.position == 399 and d.used <= 128 and device_error() == 0
