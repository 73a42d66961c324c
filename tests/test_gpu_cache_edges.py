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


def test_buffers_that_lie_between_one_another():
    """outputs in the gaps of inputs: what is documented is that they share no memory, not that they lie apart"""
    g = gen(2)
    B, T, H, hk, D, cap = 2, 5, 4, 2, 64, 90
    k, v, lens = randn(g, B, hk, cap, D, dtype=torch.float16), randn(g, B, hk, cap, D, dtype=torch.float16), ints(70, 31)
    both = randn(g, B, T, 2, H, D, dtype=torch.float16)  # a token's queries, then its outputs
    q = both[:, :, 0].clone()
    want, lse = cache.tree_attention(q, k, v, lens)
    got, _ = cache.tree_attention(both[:, :, 0], k, v, lens, out=both[:, :, 1])
    assert torch.equal(got, want) and torch.equal(both[:, :, 0], q)
    mass = torch.rand(B, 2, hk, cap, device="cuda", generator=g)
    plain = cache.attention_mass(q, lse, k, lens, mass[:, 0].contiguous(), out=mass[:, 1].contiguous())
    old = mass[:, 0].clone()
    assert torch.equal(cache.attention_mass(q, lse, k, lens, mass[:, 0], out=mass[:, 1]), plain) and torch.equal(mass[:, 0], old)
    kv = randn(g, 3, 2, B, hk, cap, D, dtype=torch.float16)  # of each layer the cache, then room for what is kept of it
    vv, m = randn(g, 3, 2, B, hk, cap, D, dtype=torch.float16), torch.rand(3, 2, B, hk, cap, device="cuda", generator=g)
    args = [x[:, 0].clone() for x in (kv, vv, m)]
    new, kept = cache.kv_evict(*args, lens, 40, 2, 8)
    new2, kept2 = cache.kv_evict(kv[:, 0], vv[:, 0], m[:, 0], lens, 40, 2, 8, k_out=kv[:, 1], v_out=vv[:, 1], mass_out=m[:, 1])
    assert torch.equal(new, new2) and torch.equal(kept, kept2)
    for b, n in enumerate(new.tolist()):
        for x, y in zip(args, (kv, vv, m)):
            assert torch.equal(y[:, 1, b, :, :n], x[:, b, :, :n])
    # one sequence, whose stride says nothing: in place all the same
    x = randn(g, 1, T, 3, D).as_strided((1, T, 3, D), (4 * D, 3 * D, D, 1))
    xk, c, pos = randn(g, 1, T, 1, D), torch.rand(9, D // 2, device="cuda", generator=g), ints(0, 1, 2, 3, 4)[None]
    kc, vc = randn(g, 1, 1, 20, D), randn(g, 1, 1, 20, D)
    want = cache.kv_append(x, xk, xk, kc, vc, ints(3), pos, c, c)
    y = x.clone()
    z = y.as_strided((1, T, 3, D), (8 * D, 3 * D, D, 1))
    assert torch.equal(cache.kv_append(y, xk, xk, kc, vc, ints(3), pos, c, c, q_out=z), want)
    ended()


def refused(call):
    with pytest.raises(p8.P8Error) as e:
        call()
    assert e.value.status == -1


def test_accept_in_place_of_its_inputs_is_refused():
    g = gen(3)
    k, v, lens, counts = randn(g, 2, 3, 2, 40, 64), randn(g, 2, 3, 2, 40, 64), ints(3, 0, 20), ints(4, 4, 2)
    tok, par = torch.zeros(3, 4, dtype=torch.int64, device="cuda"), ints(-1, 0, 1, 2).repeat(3, 1)
    for o in (dict(accepted=counts), dict(accepted=lens), dict(path=par), dict(new_lens=counts), dict(new_lens=lens)):
        refused(lambda: cache.tree_accept(tok, par, tok, k, v, lens, counts=counts, **o))
    refused(lambda: cache.tree_accept(tok, par, tok, k, k, lens))
    assert cache.tree_accept(tok, par, tok, k, v, lens, counts=counts).accepted.tolist() == [4, 4, 2]
    ended()


def test_evict_over_its_inputs_is_refused():
    g = gen(4)
    k, v, m = randn(g, 2, 2, 40, 64), randn(g, 2, 2, 40, 64), torch.rand(2, 2, 40, device="cuda", generator=g)
    lens = ints(30, 20, 10)
    refused(lambda: cache.kv_evict(k, v, m, lens[:2], 8, new_lens=lens[:2]))
    refused(lambda: cache.kv_evict(k, v, m, lens[:2], 8, new_lens=lens[1:]))
    refused(lambda: cache.kv_evict(k, k, m, lens[:2], 8))
    x = k.clone()
    refused(lambda: cache.kv_evict(k, v, m, lens[:2], 8, k_out=x, v_out=x, mass_out=m.clone()))
    refused(lambda: cache.kv_evict(k, v, m, lens[:2], 8, kept=m.view(torch.int32).view(-1)[:32].view(2, 2, 8)))
    assert cache.kv_evict(k, v, m, lens[:2], 8)[0].tolist() == [8, 8]
    ended()


def test_append_over_its_inputs_is_refused():
    g = gen(5)
    x = randn(g, 2, 5, 6, 64)
    q, xk, xv = x[:, :, :2], x[:, :, 2:4], x[:, :, 4:]
    k, v, c, pos = randn(g, 2, 2, 20, 64), randn(g, 2, 2, 20, 64), torch.rand(9, 32, device="cuda", generator=g), torch.arange(5, device="cuda").int().repeat(2, 1)
    lens = ints(3, 11)
    k0, v0 = k.clone(), v.clone()
    want = cache.kv_append(q, xk, xv, k0, v0, lens, pos, c, c)
    refused(lambda: cache.kv_append(q, xk, xv, k, v, lens, pos, c, c, q_out=xk))
    refused(lambda: cache.kv_append(q, xk, xv, k, v, lens, pos, c, c, q_out=k.transpose(1, 2)[:, :5]))
    refused(lambda: cache.kv_append(q, xk, xv, k, k, lens, pos, c, c))
    refused(lambda: cache.kv_append(q, k.transpose(1, 2)[:, 3:8], xv, k, v, lens, pos, c, c))
    assert torch.equal(cache.kv_append(q, xk, xv, k, v, lens, pos, c, c, q_out=q), want)  # in the product's own place
    assert torch.equal(k, k0) and torch.equal(v, v0)
    ended()


def test_masses_expanded_over_sequences_are_read_and_not_written():
    g = gen(6)
    k, q, lens = randn(g, 3, 2, 40, 64), randn(g, 3, 1, 4, 64), ints(30, 20, 10)
    lse = randn(g, 3, 1, 4) + 4
    one = torch.rand(1, 2, 40, device="cuda", generator=g)
    refused(lambda: cache.attention_mass(q, lse, k, lens, one.expand(3, 2, 40)))
    out = cache.attention_mass(q, lse, k, lens, one.expand(3, 2, 40), out=torch.zeros(3, 2, 40, device="cuda"))
    assert torch.equal(out, cache.attention_mass(q, lse, k, lens, one.repeat(3, 1, 1), out=torch.zeros(3, 2, 40, device="cuda")))
    refused(lambda: cache.tree_accept(torch.zeros(3, 1, dtype=torch.int64, device="cuda"), ints(-1, -1, -1)[:, None], torch.zeros(3, 1, dtype=torch.int64, device="cuda"),
                                      k[:1].expand(3, 2, 40, 64), k.clone(), lens))
    ended()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_values_next_to_the_end_of_the_type(dtype, D):
    """the largest finite numbers are numbers: in a drafted token that others do not see, in a key that draws no weight, in a value
    that is seen"""
    g = gen(7 + D)
    B, T, H, hk, n, big = 1, 5, 8, 2, 130, torch.finfo(dtype).max
    k, v = randn(g, B, hk, 150, D, dtype=dtype), randn(g, B, hk, 150, D, dtype=dtype)
    q, lens = randn(g, B, T, H, D, dtype=dtype), ints(n)
    q[..., 0] = q[..., 0].abs() + 0.5
    mask = torch.tensor([1, 3, 5, 1 | 8, 1 | 16], device="cuda")
    want, lse = cache.tree_attention(q, k, v, lens, mask=mask)
    k2, v2 = k.clone(), v.clone()
    for sign, col in ((1, 3), (-1, 9)):
        k2[:, :, n + 3, col], v2[:, :, n + 3, col] = sign * big, sign * big  # token 3, which 0, 1, 2 and 4 do not see
    got = cache.tree_attention(q, k2, v2, lens, mask=mask)
    others = [0, 1, 2, 4]
    assert torch.equal(got[0][:, others], want[:, others]) and torch.equal(got[1][:, others], lse[:, others])
    # slot 17's key is the lowest number in one column: its score is far below all others, and the rest as without the slot
    k2, rest = k.clone(), [x for x in range(n + T) if x != 17]
    k2[:, :, 17] = 0
    k2[:, :, 17, 0] = -big
    out, l2 = cache.tree_attention(q, k2, v, lens, mask=mask)
    less, l3 = cache.tree_attention(q, k[:, :, rest].contiguous(), v[:, :, rest].contiguous(), ints(n - 1), mask=mask)
    # two orders of the same sums: twice the bound that one has against 64 bits, (2 ds + (68 + 8 sqrt(n)) e) sum p |v| + the weights' and the result's roundings
    e, u = 2.0 ** -23, torch.finfo(dtype).eps / 2
    ds = (D + 16) * e * float((q.float().abs().amax(dim=(1, 2)) * k.float().abs().amax(dim=(0, 1, 2))).sum()) / D ** 0.5
    most = float(v.float().abs().max())
    tol = 2 * (2 * ds + (68 + 8 * 12) * e + (u if dtype != torch.float32 else 0)) * most + 2 * u * most
    assert float((out.float() - less.float()).abs().max()) <= tol and float((l2 - l3).abs().max()) <= 2 * (ds + (68 + 8 * 12) * e) + 2 * e * float(l3.abs().max())
    mass = cache.attention_mass(q, lse, k2, lens, torch.zeros(B, hk, 150, device="cuda"))
    assert bool((mass[..., 17] == 0).all()) and bool(mass.isfinite().all())
    # a value that is seen: weight times value, in 64 bits
    v2 = v.clone()
    v2[:, :, 40, 5] = big
    out, _ = cache.tree_attention(q, k, v2, lens, mask=mask)
    see = torch.cat([torch.ones(T, n, dtype=torch.bool, device="cuda"), (mask[:, None] >> torch.arange(T, device="cuda") & 1).bool()], dim=1)
    z = torch.einsum("thd,hsd->ths", q[0].double(), k[0, :, : n + T].double().repeat_interleave(H // hk, 0)) / D ** 0.5
    p = torch.softmax(z.masked_fill(~see[:, None], -float("inf")), -1)
    y = v2[0, :, : n + T, 5].double().repeat_interleave(H // hk, 0)
    exact, size = torch.einsum("ths,hs->th", p, y), torch.einsum("ths,hs->th", p, y.abs())
    assert bool(out[0, :, :, 5].isfinite().all())
    over = (out[0, :, :, 5].double() - exact).abs() - ((2 * ds + (68 + 8 * 12) * e + (u if dtype != torch.float32 else 0)) * size + u * exact.abs())
    assert float(over.max()) <= 0
    ended()


def test_append_of_no_tokens():
    k, v = torch.ones(2, 2, 20, 64, device="cuda"), torch.ones(2, 2, 20, 64, device="cuda")
    c = torch.rand(9, 32, device="cuda")
    x = torch.empty(2, 0, 4, 64, device="cuda")
    out = cache.kv_append(x, x[:, :, :2], x[:, :, 2:], k, v, ints(3, 11), torch.empty(2, 0, dtype=torch.int32, device="cuda"), c, c)
    ended()
    assert out.shape == (2, 0, 4, 64) and bool((k == 1).all()) and bool((v == 1).all())


@pytest.mark.parametrize("place", ["in place", "other buffers"])
def test_evict_of_very_many_rows(place):
    """80 layers x 128 sequences x 8 heads: the heaviest of the middle slots beside the first and the last"""
    g = gen(8)
    N, B, hk, cap, D, budget = 80, 128, 8, 6, 64, 3
    k, v = randn(g, N, B, hk, cap, D, dtype=torch.bfloat16), randn(g, N, B, hk, cap, D, dtype=torch.bfloat16)
    m = torch.rand(N, B, hk, cap, device="cuda", generator=g)
    lens = torch.randint(0, cap + 1, (B,), device="cuda", generator=g).int()
    at = torch.arange(cap, device="cuda")
    mid = (at >= 1) & (at < lens[:, None] - 1)
    best = torch.where(mid[None, :, None], m, -1.0).argmax(-1)
    n = lens[None, :, None].expand(N, B, hk)
    kept = torch.stack([torch.zeros_like(best), torch.where(n > budget, best, 1), torch.where(n > budget, n - 1, 2)], -1)
    kept = torch.where(torch.arange(budget, device="cuda") < n.clamp(max=budget)[..., None], kept, -1)
    x = [k.clone(), v.clone(), m.clone()]
    out = {} if place == "in place" else dict(k_out=torch.full_like(k[..., :budget, :], 3.0).contiguous(), v_out=torch.full_like(v[..., :budget, :], 3.0).contiguous(),
                                              mass_out=torch.full_like(m[..., :budget], 3.0).contiguous())
    new, got = cache.kv_evict(*x, lens, budget, 1, 1, **out)
    ended()
    assert torch.equal(new, lens.clamp(max=budget)) and torch.equal(got.long(), kept)
    y = list(out.values()) or x
    live, take = kept >= 0, kept.clamp(min=0)
    for a, b in ((k, y[0]), (v, y[1])):
        want = a.gather(3, take[..., None].expand(*take.shape, D))
        rest = torch.full_like(want, 3.0) if out else a[..., :budget, :]
        assert torch.equal(b[..., :budget, :], torch.where(live[..., None], want, rest))
        assert out or torch.equal(b[..., budget:, :], a[..., budget:, :])
    assert torch.equal(y[2][..., :budget], torch.where(live, m.gather(3, take), torch.full_like(m[..., :budget], 3.0) if out else m[..., :budget]))


@pytest.mark.parametrize("D,B", [(128, 37), (128, 38), (64, 55), (64, 56)])
def test_split_sequences_on_either_side_of_the_joins_row_counts(D, B):
    """64 rows a sequence: 2,368 rows are the last that 148 SMs add up at once with 128 columns, 3,520 of 3,552 with 64"""
    g = gen(B)
    T, H, hk, n = 16, 4, 1, 900
    k, v = randn(g, B, hk, n + T, D, dtype=torch.float16), randn(g, B, hk, n + T, D, dtype=torch.float16)
    q = randn(g, B, T, H, D, dtype=torch.float16)
    lens = (n - 7 * torch.arange(B, device="cuda")).int()
    out, lse = cache.tree_attention(q, k, v, lens)
    ended()
    z = torch.einsum("bthd,bsd->bths", q.double(), k[:, 0].double()) / D ** 0.5
    at = torch.arange(n + T, device="cuda") - lens[:, None, None]
    z = z.masked_fill((at > torch.arange(T, device="cuda")[None, :, None])[:, :, None], -float("inf"))
    p, want = torch.softmax(z, -1), torch.logsumexp(z, -1)
    exact, size = p @ v[:, :1].double(), p @ v[:, :1].double().abs()
    # per value: the weights' rounding to fp16, two errors of a score, the sum's; then the result's rounding
    e, u = 2.0 ** -23, 2.0 ** -11
    ds = (D + 16) * e * float((q.float().norm(dim=-1).max() * k.float().norm(dim=-1).max())) / D ** 0.5
    acc = (68 + 8 * 31) * e
    assert float(((out.double() - exact).abs() - ((u + 2 * ds + acc) * size + u * exact.abs())).max()) <= 0
    assert float((lse.double() - want).abs().max()) <= ds + acc + e * float(want.abs().max())


@pytest.mark.parametrize("dtype,T,H,hk,D,cap", [(torch.bfloat16, 3, 4, 2, 64, 60), (torch.float32, 2, 8, 1, 64, 90), (torch.float16, 40, 4, 1, 64, 75)])
def test_as_many_sequences_as_there_may_be(dtype, T, H, hk, D, cap):
    """4,096 sequences, padded: attention and masses of all against 64 bits"""
    g = gen(T)
    B, G = 4096, H // hk
    k, v = randn(g, B, hk, cap, D, dtype=dtype), randn(g, B, hk, cap, D, dtype=dtype)
    q = randn(g, B, T, H, D, dtype=dtype)
    lens = torch.randint(0, cap - T + 1, (B,), device="cuda", generator=g).int()
    counts = torch.randint(0, T + 1, (B,), device="cuda", generator=g).int()
    out, lse = cache.tree_attention(q, k, v, lens, counts=counts)
    mass = cache.attention_mass(q, lse, k, lens, torch.zeros(B, hk, cap, device="cuda"), counts=counts)
    ended()
    e, u = 2.0 ** -23, torch.finfo(dtype).eps / 2
    acc = (68 + 8 * cap ** 0.5) * e
    for b in torch.arange(B, device="cuda").split(512):
        n, c = lens[b], counts[b]
        z = torch.einsum("bthd,bhsd->bths", q[b].double(), k[b].double().repeat_interleave(G, 1)) / D ** 0.5
        ds = (D + 16) * e * float(q[b].float().norm(dim=-1).max() * k[b].float().norm(dim=-1).max()) / D ** 0.5
        at = torch.arange(cap, device="cuda") - n[:, None, None]
        t = torch.arange(T, device="cuda")[None, :, None]
        z = z.masked_fill(((at > t) | (at >= c[:, None, None]))[:, :, None], -float("inf"))
        real = torch.arange(T, device="cuda") < c[:, None]
        want = torch.logsumexp(z, -1)[real]
        p = torch.softmax(z, -1)
        vv = v[b].double().repeat_interleave(G, 1)
        exact, size = torch.einsum("bths,bhsd->bthd", p, vv)[real], torch.einsum("bths,bhsd->bthd", p, vv.abs())[real]
        assert float(((out[b][real].double() - exact).abs() - (((u if dtype != torch.float32 else 0) + 2 * ds + acc) * size + u * exact.abs())).max()) <= 0
        assert float(((lse[b][real].double() - want).abs() - (ds + acc + e * want.abs())).max()) <= 0
        assert bool((out[b][~real] == 0).all()) and bool((lse[b][~real] == 0).all())
        # a weight is off by its score's and lse's errors and a few steps, a sum of T * G of them by a step each
        w = torch.exp(z - lse[b].double()[..., None]).masked_fill(~real[:, :, None, None], 0).sum(1).unflatten(1, (hk, G)).sum(2)
        assert float(((mass[b].double() - w).abs() - (2 * ds + 8 * e + (T * G + 2) * e) * w).max()) <= 1e-30
