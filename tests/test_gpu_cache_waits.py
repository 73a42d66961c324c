"""Waits of the attention and mass pipelines that run out: the call ends with bit 128 of the error word, what it had started has
ended with it, and the next calls are as if it had not been. (The limit is set to nothing, so that a wait gives up where its
barrier is not over at the first look; nothing is left out of the kernels.)"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

import pingala8_llm_b200 as p8  # noqa: E402
from pingala8_llm_b200 import cache  # noqa: E402

DEFAULT = 2_000_000_000


@pytest.fixture(autouse=True)
def limit_restored():
    yield
    assert p8.lib().p8_cache_wait_limit(DEFAULT) == 0


def limit(ns):
    assert p8.lib().p8_cache_wait_limit(ns) == 0


@pytest.mark.parametrize("B,T,H,hk,D,length", [
    (1, 1, 32, 8, 128, 129), (3, 7, 8, 2, 64, 3000), (1, 12, 32, 8, 128, 9000), (1, 33, 8, 2, 128, 5000), (2, 64, 8, 1, 64, 4000), (1, 64, 32, 8, 128, 20000),
    (1, 64, 9, 1, 128, 700)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_waits_that_run_out(dtype, B, T, H, hk, D, length):
    g = torch.Generator(device="cuda")
    g.manual_seed(T + length)
    k, v = (torch.randn(B, hk, length + T, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    q = torch.randn(B, T, H, D, device="cuda", generator=g).to(dtype)
    lens = torch.tensor([length - 11 * b for b in range(B)], dtype=torch.int32, device="cuda")
    before = torch.rand(B, hk, length + T, device="cuda", generator=g)

    def attend():
        return cache.tree_attention(q, k, v, lens)

    def weigh(lse):
        return cache.attention_mass(q, lse, k, lens, before, out=before.clone())

    # The 16-bit kernels wait for products in every call. The 32-bit ones wait for tiles alone, which may all have come while the
    # queries are loaded: only with more of them for a CTA (of 64 slots, in 148 or more equal shares) than its ring's 8 stages is a
    # wait certain to run out, that for a free stage.
    tiles = sum((int(n) + T + 63) // 64 for n in lens) * hk
    errors = (128,) if dtype != torch.float32 or tiles > 8 * 148 else (0, 128)
    out, lse = attend()
    mass = weigh(lse)
    assert p8.device_error() == 0
    for call in (attend, lambda: weigh(lse)):
        limit(0)
        for _ in range(3):
            call()
        torch.cuda.synchronize()
        assert p8.device_error() in errors
        call()  # the word was cleared; the next call reports for itself
        torch.cuda.synchronize()
        assert p8.device_error() in errors
        limit(1)  # the first look stays for microseconds: some waits run out in the middle of a call, or none
        for _ in range(3):
            call()
        torch.cuda.synchronize()
        assert p8.device_error() in (0, 128)
        limit(DEFAULT)
        again = attend()
        assert torch.equal(again[0], out) and torch.equal(again[1], lse) and torch.equal(weigh(lse), mass)
        torch.cuda.synchronize()
        assert p8.device_error() == 0
