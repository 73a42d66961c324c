"""Waits of the paged attention that run out: the call ends with bit 128 of the error word, what it had started has ended with it, and
the next calls are as if it had not been. (The limit is set to nothing, so that a wait gives up where its tile is not there at the
first look; nothing is left out of the kernel.)"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

import pingala8_llm_b200 as p8  # noqa: E402
from pingala8_llm_b200 import paged  # noqa: E402

DEFAULT = 2_000_000_000


@pytest.fixture(autouse=True)
def limit_restored():
    yield
    assert p8.lib().p8_cache_wait_limit(DEFAULT) == 0


def limit(ns):
    assert p8.lib().p8_cache_wait_limit(ns) == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,H,kv,D,page,length", [(1, 4, 1, 64, 16, 30), (3, 32, 8, 128, 16, 129), (70, 8, 2, 64, 24, 700), (2, 24, 2, 128, 64, 40000), (1, 32, 8, 128, 64, 60000)])
def test_waits_that_run_out(dtype, B, H, kv, D, page, length):
    g = torch.Generator(device="cuda")
    g.manual_seed(length)
    n = (length + page) // page
    k, v = (torch.randn(n * B, kv, page, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    tables = torch.randperm(n * B, device="cuda", generator=g).int().view(B, n)
    q = torch.randn(B, H, D, device="cuda", generator=g).to(dtype)
    lens = torch.tensor([length - 7 * b for b in range(B)], dtype=torch.int32, device="cuda")

    def attend():
        return paged.paged_attention(q, k, v, tables, lens)

    out, lse = attend()
    torch.cuda.synchronize()
    assert p8.device_error() == 0
    # In a short call all tiles may have come while the queries were loaded. With tens of them for every warp, each asked for when the one
    # two places before it is done with, some are not there at the first look.
    errors = (128,) if B * length * kv >= 480000 else (0, 128)
    limit(0)
    for _ in range(3):
        attend()
    torch.cuda.synchronize()
    assert p8.device_error() in errors
    limit(1)  # the first look stays for microseconds: some waits run out in the middle of a call, or none
    for _ in range(3):
        attend()
    torch.cuda.synchronize()
    assert p8.device_error() in (0, 128)
    limit(DEFAULT)
    again = attend()
    torch.cuda.synchronize()
    assert torch.equal(again[0], out) and torch.equal(again[1], lse) and p8.device_error() == 0
