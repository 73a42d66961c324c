"""Key/value cache operators at the edges of what they document: errors on other streams, buffers that lie between one another,
values next to a type's range, calls of nothing and of very many rows."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

import pingala8_llm_b200 as p8  # noqa: E402
from pingala8_llm_b200 import cache  # noqa: E402


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def ended(bits=0):
    assert p8.device_error() == bits


def test_an_error_on_another_stream_is_there_when_it_is_asked_for():
    """device_error waits for streams that do not block the default one"""
    g = gen(1)
    k, v, q = randn(g, 1, 2, 40, 64), randn(g, 1, 2, 40, 64), randn(g, 1, 3, 4, 64)
    lens, side = ints(39), torch.cuda.Stream()  # 39 + 3 tokens are more than 40 slots
    cache.tree_attention(q, k, v, ints(5))
    ended()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # 0.1 s
    cache.tree_attention(q, k, v, lens, stream=side)
    ended(64)
    ended()
