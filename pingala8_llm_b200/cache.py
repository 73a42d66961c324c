"""Key/value cache operators: what a decoder runs between its Pingala-8 projections.

A cache is a pair of tensors [batch, kv heads, slots, width] (float32, float16 or bfloat16; width 64 or 128), or with a
leading layer dimension for the two operators that serve all layers at once (kv_evict, tree_accept). Any strides whose
rows start on 16 bytes and have unit stride inside; the keys and the values may lie apart. Sequence b is as long as
the int32 device tensor lens[b] says and the device alone reads it, so calls can be captured in a CUDA graph and replayed
while sequences grow. A call's tokens have the slots behind the sequence's end; `counts` (int32 [batch]) says how many
of them are real where a batch is padded, and what belongs to the others is neither read nor written.

One step of speculative decoding with a bounded cache:

    mask, depth = tree_plan(parents)                                    # once per tree
    q = kv_append(q, k, v, k_cache, v_cache, lens, lens[:, None] + depth, cos, sin)      # per layer
    out, lse = tree_attention(q, k_cache, v_cache, lens, mask=mask)                      # per layer
    acc = tree_accept(tokens, parents, target, all_k, all_v, lens)
    attention_mass(q, lse, k_cache, lens, mass, rows=acc.path, counts=acc.accepted)      # per layer
    lens, kept = kv_evict(all_k, all_v, all_mass, acc.new_lens, budget, sinks, recent)

Every call goes through the C ABI of libpingala8_b200.so on the tensors' device, on its current stream or the one
given; there is no CPU path and no gradient. Lengths, counts, positions and rows that are out of range leave their
sequence or token out and set bit 64 of device_error().
"""
import struct
from collections import namedtuple

import torch

from ._lib import check, lib

TREE_MAX = 64

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_KV = struct.Struct("=16q")
_APPEND = struct.Struct("=3q9q2q3q2qq2qd4q")
_ATTN = struct.Struct("=4q2q4qd5q")
_MASS = struct.Struct("=4q2q4qd6q")
_EVICT = struct.Struct("=8q3q3q")
_ACCEPT = struct.Struct("=10q")

Accepted = namedtuple("Accepted", "path accepted next_token new_lens")


def _refuse(what):
    raise ValueError(what)


# A decode step makes several of these calls per layer, and their checks are most of a small call's time on the host:
# each is one comparison of what torch hands out cheapest, and words are put together only for an error.
def _kv(k, v):
    """(packed p8_kv, shape) of one layer's cache"""
    if not k.is_cuda or k.dtype not in _TYPES:
        _refuse("the cache must be float32, float16 or bfloat16 CUDA tensors")
    shape = k.shape
    if len(shape) != 4:
        _refuse(f"the cache must be [batch, kv heads, slots, width], not {list(shape)}")
    a, b, c, d = vs = k.stride()
    vp = 0
    if v is not None:
        if v.shape != shape or v.dtype is not k.dtype or v.get_device() != k.get_device():
            _refuse("keys and values must have one shape, type and device")
        vs = v.stride()
        vp = v.data_ptr()
    if d != 1 or vs[3] != 1:
        _refuse("the cache's last dimension must have unit stride")
    return _KV.pack(k.data_ptr(), vp, _TYPES[k.dtype], 1, *shape, 0, a, b, c, 0, vs[0], vs[1], vs[2]), shape


def _kv_layers(k, v):
    """(packed p8_kv, shape with layers) of a cache with or without a layer dimension"""
    if k.dim() == 4:
        kv, shape = _kv(k, v)
        return kv, (1, *shape)
    if not k.is_cuda or k.dtype not in _TYPES:
        _refuse("the cache must be float32, float16 or bfloat16 CUDA tensors")
    shape = k.shape
    if len(shape) != 5:
        _refuse(f"the cache must be [batch, kv heads, slots, width] or [layers, batch, kv heads, slots, width], not {list(shape)}")
    if v.shape != shape or v.dtype is not k.dtype or v.get_device() != k.get_device():
        _refuse("keys and values must have one shape, type and device")
    ks, vs = k.stride(), v.stride()
    if ks[4] != 1 or vs[4] != 1:
        _refuse("the cache's last dimension must have unit stride")
    return _KV.pack(k.data_ptr(), v.data_ptr(), _TYPES[k.dtype], *shape, *ks[:4], *vs[:4]), shape


def _flat(t, shape, dtype, dev, name):
    if t.dtype is dtype and t.shape == shape and t.get_device() == dev and t.is_contiguous():
        return t.data_ptr()
    _refuse(f"{name} must be contiguous {dtype} {list(shape)} on the cache's device")


def _rows(t, shape, dtype, dev, name):
    """pointer and the three outer strides of [batch, tokens, heads, width]"""
    if t.dtype is dtype and t.shape == shape and t.get_device() == dev:
        a, b, c, d = t.stride()
        if d == 1:
            return t.data_ptr(), a, b, c
    _refuse(f"{name} must be {dtype} {list(shape)} with unit stride in its last dimension, on the cache's device")


def _query(q, k, shape):
    """pointer and strides of q [batch, tokens, heads, width] beside a cache of this shape, tokens, heads"""
    if q.dim() != 4:
        _refuse("q must be [batch, tokens, heads, width]")
    _, T, H, _ = q.shape
    if not 1 <= T <= TREE_MAX or H % shape[1] or not H:
        _refuse(f"1 to {TREE_MAX} tokens, and query heads in whole groups")
    return _rows(q, (shape[0], T, H, shape[3]), k.dtype, k.get_device(), "q"), T, H


_here = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream


def _on(dev, stream, call, *args):
    """call(*args) with the tensors' device, and the stream where the caller gave one, current: for the launch, and for
    what the call allocates"""
    if stream is not None:
        if stream.device.index != dev:
            _refuse("the stream must belong to the cache's device")
        with torch.cuda.stream(stream):
            return call(*args)
    if _here() != dev:
        with torch.cuda.device(dev):
            return call(*args)
    return call(*args)


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
    k_norm float32 [width]: RMSNorm per head before the rotation. Any number of tokens up to the cache's slots."""
    kv, (B, hk, _, D) = _kv(k_cache, v_cache)
    dev = k_cache.get_device()
    if q.dim() != 4 or cos.dim() != 2:
        _refuse("q must be [batch, tokens, heads, width], cos [positions, width / 2]")
    _, T, H, _ = q.shape
    P = cos.shape[0]
    f32, i32 = torch.float32, torch.int32
    qp, q0, q1, q2 = _rows(q, (B, T, H, D), f32, dev, "q")
    kp, k0, k1, k2 = _rows(k, (B, T, hk, D), f32, dev, "k")
    vp, v0, v1, v2 = _rows(v, (B, T, hk, D), f32, dev, "v")
    tail = (_flat(lens, (B,), i32, dev, "lens"), 0 if counts is None else _flat(counts, (B,), i32, dev, "counts"), _flat(pos, (B, T), i32, dev, "pos"),
            _flat(cos, (P, D // 2), f32, dev, "cos"), _flat(sin, (P, D // 2), f32, dev, "sin"), P,
            0 if q_norm is None else _flat(q_norm, (D,), f32, dev, "q_norm"), 0 if k_norm is None else _flat(k_norm, (D,), f32, dev, "k_norm"), eps)

    def call(q_out):
        if q_out is None:
            q_out = (torch.empty if counts is None else torch.zeros)(B, T, H, D, dtype=k_cache.dtype, device=k_cache.device)
        a = _APPEND.pack(qp, kp, vp, q0, q1, q2, k0, k1, k2, v0, v1, v2, T, H, *tail, *_rows(q_out, (B, T, H, D), k_cache.dtype, dev, "q_out"))
        check(lib().p8_kv_append(kv, a, _raw_stream(dev)), "p8_kv_append")
        return q_out

    return _on(dev, stream, call, q_out)


def tree_attention(q, k_cache, v_cache, lens, mask=None, counts=None, scale=None, out=None, lse=None, workspace=None, stream=None):
    """Attention of 1 to 64 tokens per sequence over the cache, their own keys and values already in it (kv_append).

    q [batch, tokens, heads, width] in the cache's type. Token t sees the whole sequence before the call's tokens and the
    tokens whose bits mask[t] has (int64 [tokens] or [batch, tokens], as tree_plan makes it; None: a chain). Returns
    (out like q, lse float32 [batch, tokens, heads]): the softmax average of the values and the natural log of the sum
    of exponentials; 0 and -inf for a token that sees nothing. scale: 1 / sqrt(width) unless given."""
    kv, shape = _kv(k_cache, v_cache)
    B = shape[0]
    dev = k_cache.get_device()
    (qp, q0, q1, q2), T, H = _query(q, k_cache, shape)
    lp = _flat(lens, (B,), torch.int32, dev, "lens")
    np_ = 0 if counts is None else _flat(counts, (B,), torch.int32, dev, "counts")
    mp = ms = 0
    if mask is not None:
        ms = T if mask.dim() == 2 else 0
        mp = _flat(mask, (B, T) if ms else (T,), torch.int64, dev, "mask")

    def call(out, lse, workspace):
        new = torch.empty if counts is None else torch.zeros
        if out is None:
            out = new(q.shape, dtype=q.dtype, device=q.device)
        if lse is None:
            lse = new((B, T, H), dtype=torch.float32, device=q.device)
        if workspace is None:
            workspace = torch.empty(lib().p8_tree_attn_workspace(kv, T, H), dtype=torch.uint8, device=q.device)
        elif workspace.get_device() != dev or not workspace.is_contiguous():
            _refuse("workspace must be contiguous on the cache's device")
        a = _ATTN.pack(qp, q0, q1, q2, T, H, lp, np_, mp, ms, shape[3] ** -0.5 if scale is None else scale,
                       *_rows(out, q.shape, q.dtype, dev, "out"), _flat(lse, (B, T, H), torch.float32, dev, "lse"))
        check(lib().p8_tree_attn(kv, a, workspace.data_ptr(), workspace.nbytes, _raw_stream(dev)), "p8_tree_attn")
        return out, lse

    return _on(dev, stream, call, out, lse, workspace)


def attention_workspace_size(k_cache, tokens, heads):
    """workspace bytes of tree_attention on this cache, for callers that keep their own"""
    return int(lib().p8_tree_attn_workspace(_kv(k_cache, k_cache)[0], tokens, heads))


def attention_mass(q, lse, k_cache, lens, mass, rows=None, counts=None, scale=None, out=None, stream=None):
    """Adds to mass float32 [batch, kv heads, slots] the attention weight that each slot drew from a chain of tokens
    behind the sequence, summed over them and over the query heads of the slot's cache head.

    q, lse: as in the tree_attention call. rows int32 [batch, tokens]: the tokens' rows in q and lse (the accepted path,
    once tree_accept has moved its keys into place); None: 0, 1, 2, ... counts: how many tokens. The tokens' own slots
    start at 0. In place unless out is given."""
    kv, shape = _kv(k_cache, None)
    B = shape[0]
    dev = k_cache.get_device()
    (qp, q0, q1, q2), T, H = _query(q, k_cache, shape)
    i32, f32 = torch.int32, torch.float32
    if out is None:
        out = mass
    ms = []
    for t in (mass, out):
        st = t.stride()
        if t.dtype is not f32 or t.shape != shape[:3] or st[2] != 1 or t.get_device() != dev:
            _refuse("mass and out must be float32 [batch, kv heads, slots] with unit slot stride on the cache's device")
        ms += (t.data_ptr(), st[0], st[1])
    a = _MASS.pack(qp, q0, q1, q2, T, H, _flat(lse, (B, T, H), f32, dev, "lse"), _flat(lens, (B,), i32, dev, "lens"),
                   0 if counts is None else _flat(counts, (B,), i32, dev, "counts"), 0 if rows is None else _flat(rows, (B, T), i32, dev, "rows"),
                   shape[3] ** -0.5 if scale is None else scale, *ms)

    def call():
        check(lib().p8_attn_mass(kv, a, _raw_stream(dev)), "p8_attn_mass")
        return out

    return _on(dev, stream, call)


def kv_evict(k_cache, v_cache, mass, lens, budget, sinks=0, recent=0, k_out=None, v_out=None, mass_out=None, new_lens=None, kept=None, stream=None):
    """Shortens every sequence with more than `budget` slots to `budget`, per layer and cache head: the first `sinks`
    slots, the last `recent`, and of the others those with the largest mass (ties: the lowest slot), in order.

    Cache [layers, batch, kv heads, slots, width] or without layers, mass float32 of its first dimensions. The kept
    slots go to the front of k_out, v_out and mass_out (other buffers, budget slots or more; give all three), or of the
    cache itself. Returns (new_lens int32 [batch], kept int32 [..., kv heads, budget]: the kept slots, -1 behind them)."""
    kv, (N, B, hk, S, D) = _kv_layers(k_cache, v_cache)
    dev = k_cache.get_device()
    place = k_out is None
    if (v_out is None) != place or (mass_out is None) != place:
        _refuse("give k_out, v_out and mass_out together")
    if place:
        kv2, S2, mass_out = kv, S, mass
    else:
        if k_out.dim() != k_cache.dim() or k_out.dtype is not k_cache.dtype:
            _refuse("k_out must have the cache's dimensions and type")
        kv2, shape = _kv_layers(k_out, v_out)
        S2 = shape[3]
        if tuple(shape) != (N, B, hk, S2, D) or k_out.get_device() != dev:
            _refuse("k_out must have the cache's shape but for its slots, on its device")
    budget = int(budget)
    lead = k_cache.shape[:-2]
    ms = []
    for t, s in ((mass, S), (mass_out, S2)):
        st = t.stride()
        if t.dtype is not torch.float32 or t.shape != (*lead, s) or st[-1] != 1 or t.get_device() != dev:
            _refuse("mass must be float32 [.., kv heads, slots] of the cache with unit slot stride, on its device")
        ms += (t.data_ptr(), *(st[:3] if len(lead) == 3 else (0, *st[:2])))
    lp = _flat(lens, (B,), torch.int32, dev, "lens")

    def call(new_lens, kept):
        if new_lens is None:
            new_lens = torch.empty_like(lens)
        if kept is None:
            kept = torch.empty(*lead, max(budget, 0), dtype=torch.int32, device=k_cache.device)
        a = _EVICT.pack(*ms, lp, _flat(new_lens, (B,), torch.int32, dev, "new_lens"), _flat(kept, (*lead, budget), torch.int32, dev, "kept"), budget, sinks, recent)
        check(lib().p8_kv_evict(kv, kv2, a, _raw_stream(dev)), "p8_kv_evict")
        return new_lens, kept

    return _on(dev, stream, call, new_lens, kept)


def tree_accept(tokens, parents, target, k_cache, v_cache, lens, counts=None, path=None, accepted=None, next_token=None, new_lens=None, stream=None):
    """Greedy verification of drafted trees: tokens int64 [batch, tokens] (token 0 the last known one), parents int32,
    target int64 (the model's choice after each token). From token 0 the path goes on to the lowest child that is what
    the target chose; its keys and values move, in all layers of the cache [layers, batch, kv heads, slots, width] (or
    without layers), to the slots right behind the sequence.

    Returns Accepted(path int32 [batch, tokens] (-1 behind it), accepted int32 [batch] its length, next_token int64
    [batch] the target at its end, new_lens int32 [batch])."""
    kv, (_, B, _, _, _) = _kv_layers(k_cache, v_cache)
    dev = k_cache.get_device()
    if tokens.dim() != 2 or not 1 <= tokens.shape[1] <= TREE_MAX:
        _refuse(f"tokens must be [batch, 1 to {TREE_MAX}]")
    T = tokens.shape[1]
    i32, i64 = torch.int32, torch.int64
    head = (_flat(tokens, (B, T), i64, dev, "tokens"), _flat(target, (B, T), i64, dev, "target"), _flat(parents, (B, T), i32, dev, "parents"), T,
            _flat(lens, (B,), i32, dev, "lens"), 0 if counts is None else _flat(counts, (B,), i32, dev, "counts"))

    def call(path, accepted, next_token, new_lens):
        if path is None:
            path = torch.empty((B, T), dtype=i32, device=k_cache.device)
        if accepted is None:
            accepted = torch.empty_like(lens)
        if next_token is None:
            next_token = torch.empty(B, dtype=i64, device=k_cache.device)
        if new_lens is None:
            new_lens = torch.empty_like(lens)
        a = _ACCEPT.pack(*head, _flat(path, (B, T), i32, dev, "path"), _flat(accepted, (B,), i32, dev, "accepted"),
                         _flat(new_lens, (B,), i32, dev, "new_lens"), _flat(next_token, (B,), i64, dev, "next_token"))
        check(lib().p8_tree_accept(kv, a, _raw_stream(dev)), "p8_tree_accept")
        return Accepted(path, accepted, next_token, new_lens)

    return _on(dev, stream, call, path, accepted, next_token, new_lens)
