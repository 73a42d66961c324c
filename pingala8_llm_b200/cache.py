"""Key/value cache operators: what a decoder runs between its Pingala-8 projections.

A cache is a pair of tensors [batch, kv heads, slots, width] (float32, float16 or bfloat16; width 64 or 128), or with a
leading layer dimension for the two operators that serve all layers at once (kv_evict, tree_accept). Any strides whose
rows start on 16 bytes and have unit stride inside; the keys and the values may lie apart. Sequence b is as long as
the int32 device tensor lens[b] says and the device alone reads it, so calls can be captured in a CUDA graph and replayed
while sequences grow. A call's tokens have the slots behind the sequence's end; `counts` (int32 [batch]) says how many
of them are real where a batch is padded, and what belongs to the others has no effect and is not written.

One step of speculative decoding with a bounded cache:

    mask, depth = tree_plan(parents)                                    # once per tree
    q = kv_append(q, k, v, k_cache, v_cache, lens, lens[:, None] + depth, cos, sin)      # per layer
    out, lse = tree_attention(q, k_cache, v_cache, lens, mask=mask)                      # per layer
    acc = tree_accept(tokens, parents, target, all_k, all_v, lens)
    attention_mass(q, lse, k_cache, lens, mass, rows=acc.path, counts=acc.accepted)      # per layer
    lens, kept = kv_evict(all_k, all_v, all_mass, acc.new_lens, budget, sinks, recent)

Every call goes through the C ABI of libpingala8_b200.so on the tensors' device, on its current stream or the one
given; there is no CPU path and no gradient. Lengths, counts, positions and rows that are out of range leave their
sequence or token out and set bit 64 of device_error(). Outputs overlap neither one another nor what a call reads, but where
"in place" is said; a tensor expanded over a dimension (stride 0) is no output. Buffers may lie between one another's rows.
"""
import ctypes as C
from collections import namedtuple

import torch

from ._lib import check, lib

try:
    from . import _cache_calls as _c
except ImportError as e:
    raise ImportError(f"{e}: build it with `python -m pingala8_llm_b200.build` (no fallback)") from e

_c.bind(*(C.cast(getattr(lib(), n), C.c_void_p).value
          for n in ("p8_kv_append", "p8_tree_attn_workspace", "p8_tree_attn", "p8_attn_mass", "p8_kv_evict", "p8_tree_accept")))

TREE_MAX = 64

Accepted = namedtuple("Accepted", "path accepted next_token new_lens")


def _refuse(what):
    raise ValueError(what)


def _on(stream, k, call, *args, **kw):
    """the call with the caller's stream current, for the launch and for what it allocates"""
    if stream.device != k.device:
        _refuse("the stream must belong to the cache's device")
    with torch.cuda.stream(stream):
        return call(*args, **kw)


def tree_plan(parents):
    """Ancestor bits and depths of drafted trees: parents int [tokens] or [batch, tokens] (parents[t] < t is the token
    that t hangs on, -1 for a root) -> (mask int64, depth int32) of the same shape. Bit j of mask[t]: t is j or hangs on
    it. Torch operations on the tensor's own device; for a fixed tree it is done once."""
    if parents.dtype not in (torch.int32, torch.int64) or parents.dim() not in (1, 2):
        _refuse("parents must be int32 or int64 [tokens] or [batch, tokens]")
    n = parents.shape[-1]
    if not 1 <= n <= TREE_MAX:
        _refuse(f"a tree has 1 to {TREE_MAX} tokens")
    t = torch.arange(n, device=parents.device)
    root = parents < 0
    mask = (torch.ones_like(t) << t).expand(parents.shape).clone()
    up = torch.where(root, t, torch.minimum(parents.long(), t))
    depth = (up != t).int()
    step = 1
    while step < n:  # pointer doubling
        mask |= mask.gather(-1, up)
        depth = depth + depth.gather(-1, up)
        up = up.gather(-1, up)
        step *= 2
    return mask, depth


def kv_append(q, k, v, k_cache, v_cache, lens, pos, cos, sin, q_norm=None, k_norm=None, eps=1e-6, counts=None, q_out=None, stream=None):
    """New tokens into the cache: q float32 [batch, tokens, heads, width], k and v float32 [batch, tokens, kv heads,
    width] (views of the projections' outputs) -> rotated queries in the cache's type; rotated keys and plain values in
    the tokens' slots.

    pos int32 [batch, tokens]: each token's row of cos / sin float32 [positions, width / 2] (rotate-half form). q_norm,
    k_norm float32 [width]: RMSNorm per head before the rotation. Any number of tokens up to the cache's slots, none too.
    q_out may be q (in place) where the cache is float32."""
    if stream is not None:
        return _on(stream, k_cache, kv_append, q, k, v, k_cache, v_cache, lens, pos, cos, sin, q_norm, k_norm, eps, counts, q_out)
    if q_out is None:
        q_out = (torch.empty if counts is None else torch.zeros)(q.shape, dtype=k_cache.dtype, device=k_cache.device)
    st = _c.kv_append(q, k, v, k_cache, v_cache, lens, pos, cos, sin, q_norm, k_norm, eps, counts, q_out)
    if st:
        check(st, "p8_kv_append")
    return q_out


def tree_attention(q, k_cache, v_cache, lens, mask=None, counts=None, scale=None, out=None, lse=None, workspace=None, stream=None):
    """Attention of 1 to 64 tokens per sequence over the cache, their own keys and values already in it (kv_append).

    q [batch, tokens, heads, width] in the cache's type. Token t sees the whole sequence before the call's tokens and the
    tokens whose bits mask[t] has (int64 [tokens] or [batch, tokens], as tree_plan makes it; None: a chain). Returns
    (out like q, lse float32 [batch, tokens, heads]): the softmax average of the values and the natural log of the sum
    of exponentials; 0 and -inf for a token that sees nothing. scale: 1 / sqrt(width) unless given. With a 16-bit cache the
    weights are rounded to its type: out is off by up to 1.4 times as much as one of 32-bit weights, rounded once."""
    if stream is not None:
        return _on(stream, k_cache, tree_attention, q, k_cache, v_cache, lens, mask, counts, scale, out, lse, workspace)
    if out is None:
        out = (torch.empty if counts is None else torch.zeros)(q.shape, dtype=q.dtype, device=q.device)
    if lse is None:
        lse = (torch.empty if counts is None else torch.zeros)(q.shape[:3], dtype=torch.float32, device=q.device)
    st = _c.tree_attention(q, k_cache, v_cache, lens, mask, counts, scale, out, lse, workspace)
    if st:
        check(st, "p8_tree_attn")
    return out, lse


def attention_workspace_size(k_cache, tokens, heads):
    """workspace bytes of tree_attention on this cache, for callers that keep their own"""
    return _c.attention_workspace(k_cache, tokens, heads)


def attention_mass(q, lse, k_cache, lens, mass, rows=None, counts=None, scale=None, out=None, stream=None):
    """Adds to mass float32 [batch, kv heads, slots] the attention weight that each slot drew from a chain of tokens
    behind the sequence, summed over them and over the query heads of the slot's cache head.

    q, lse: as in the tree_attention call. rows int32 [batch, tokens]: the tokens' rows in q and lse (the accepted path,
    once tree_accept has moved its keys into place); None: 0, 1, 2, ... counts: how many tokens. The tokens' own slots
    start at 0. In place unless out is given."""
    if stream is not None:
        return _on(stream, k_cache, attention_mass, q, lse, k_cache, lens, mass, rows, counts, scale, out)
    if out is None:
        out = mass
    st = _c.attention_mass(q, lse, k_cache, lens, mass, rows, counts, scale, out)
    if st:
        check(st, "p8_attn_mass")
    return out


def kv_evict(k_cache, v_cache, mass, lens, budget, sinks=0, recent=0, k_out=None, v_out=None, mass_out=None, new_lens=None, kept=None, stream=None):
    """Shortens every sequence with more than `budget` slots to `budget`, per layer and cache head: the first `sinks`
    slots, the last `recent`, and of the others those with the largest mass (ties: the lowest slot), in order.

    Cache [layers, batch, kv heads, slots, width] or without layers, mass float32 of its first dimensions. The kept
    slots go to the front of k_out, v_out and mass_out (other buffers, budget slots or more; give all three), or of the
    cache itself. Returns (new_lens int32 [batch], kept int32 [..., kv heads, budget]: the kept slots, -1 behind them)."""
    if stream is not None:
        return _on(stream, k_cache, kv_evict, k_cache, v_cache, mass, lens, budget, sinks, recent, k_out, v_out, mass_out, new_lens, kept)
    if (v_out is None) != (k_out is None) or (mass_out is None) != (k_out is None):
        _refuse("give k_out, v_out and mass_out together")
    if k_out is None:
        k_out, v_out, mass_out = k_cache, v_cache, mass
    if new_lens is None:
        new_lens = torch.empty_like(lens)
    if kept is None:
        kept = torch.empty(*k_cache.shape[:-2], max(int(budget), 0), dtype=torch.int32, device=k_cache.device)
    st = _c.kv_evict(k_cache, v_cache, mass, lens, budget, sinks, recent, k_out, v_out, mass_out, new_lens, kept)
    if st:
        check(st, "p8_kv_evict")
    return new_lens, kept


def tree_accept(tokens, parents, target, k_cache, v_cache, lens, counts=None, path=None, accepted=None, next_token=None, new_lens=None, stream=None):
    """Greedy verification of drafted trees: tokens int64 [batch, tokens] (token 0 the last known one), parents int32,
    target int64 (the model's choice after each token). From token 0 the path goes on to the lowest child that is what
    the target chose; its keys and values move, in all layers of the cache [layers, batch, kv heads, slots, width] (or
    without layers), to the slots right behind the sequence.

    Returns Accepted(path int32 [batch, tokens] (-1 behind it), accepted int32 [batch] its length, next_token int64
    [batch] the target at its end, new_lens int32 [batch])."""
    if stream is not None:
        return _on(stream, k_cache, tree_accept, tokens, parents, target, k_cache, v_cache, lens, counts, path, accepted, next_token, new_lens)
    if path is None:
        path = torch.empty(tokens.shape, dtype=torch.int32, device=tokens.device)
    if accepted is None:
        accepted = torch.empty_like(lens)
    if next_token is None:
        next_token = torch.empty(lens.shape, dtype=torch.int64, device=lens.device)
    if new_lens is None:
        new_lens = torch.empty_like(lens)
    st = _c.tree_accept(tokens, parents, target, k_cache, v_cache, lens, counts, path, accepted, next_token, new_lens)
    if st:
        check(st, "p8_tree_accept")
    return Accepted(path, accepted, next_token, new_lens)
