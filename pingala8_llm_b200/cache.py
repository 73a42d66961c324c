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
import ctypes as C
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


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _kv(k, v, layers):
    """the packed p8_kv of a cache, and (layers, batch, heads, slots, width)"""
    _need(k.is_cuda and k.dtype in _TYPES, "the cache must be float32, float16 or bfloat16 CUDA tensors")
    nd = k.dim()
    _need(nd == 4 or (layers and nd == 5), "the cache must be [batch, kv heads, slots, width]" + (" or [layers, ...] of it" if layers else ""))
    ks = k.stride()
    _need(ks[-1] == 1, "the cache's last dimension must have unit stride")
    shape = tuple(k.shape) if nd == 5 else (1, *k.shape)
    if nd == 4:
        ks = (0, *ks)
    vp, vs = 0, ks
    if v is not None:
        _need(v.shape == k.shape and v.dtype == k.dtype and v.device == k.device, "keys and values must have one shape, type and device")
        vs = v.stride()
        _need(vs[-1] == 1, "the cache's last dimension must have unit stride")
        if nd == 4:
            vs = (0, *vs)
        vp = v.data_ptr()
    return _KV.pack(k.data_ptr(), vp, _TYPES[k.dtype], *shape, *ks[:4], *vs[:4]), shape


def _ints(t, shape, dtype, dev, name):
    _need(t.dtype == dtype and tuple(t.shape) == shape and t.is_contiguous() and t.device == dev, f"{name} must be contiguous {dtype} {list(shape)} on the cache's device")
    return t.data_ptr()


def _rows(t, shape, dtype, dev, name):
    """pointer and the three outer strides of [batch, tokens, heads, width]"""
    _need(t.dtype == dtype and tuple(t.shape) == shape and t.device == dev, f"{name} must be {dtype} {list(shape)} on the cache's device")
    st = t.stride()
    _need(st[3] == 1, f"{name}'s last dimension must have unit stride")
    return t.data_ptr(), st[0], st[1], st[2]


class _On:
    """Makes the tensors' device (and, where the caller gave one, the stream) current, for the launch and for what the
    call allocates."""

    def __init__(self, dev, stream):
        self.dev, self.stream, self.ctx = dev, stream, None

    def __enter__(self):
        if self.stream is not None:
            _need(self.stream.device == self.dev, "the stream must belong to the cache's device")
            self.ctx = torch.cuda.stream(self.stream)
        elif torch.cuda.current_device() != self.dev.index:
            self.ctx = torch.cuda.device(self.dev)
        if self.ctx is not None:
            self.ctx.__enter__()
        return C.c_void_p(torch._C._cuda_getCurrentRawStream(self.dev.index))

    def __exit__(self, *e):
        if self.ctx is not None:
            self.ctx.__exit__(*e)


def tree_plan(parents):
    """Ancestor bits and depths of drafted trees: parents int [tokens] or [batch, tokens] (parents[t] < t is the token
    that t hangs on, -1 for a root) -> (mask int64, depth int32) of the same shape. Bit j of mask[t]: t is j or hangs on
    it. Torch operations on the tensor's own device; for a fixed tree it is done once."""
    _need(parents.dtype in (torch.int32, torch.int64) and parents.dim() in (1, 2), "parents must be int32 or int64 [tokens] or [batch, tokens]")
    n = parents.shape[-1]
    _need(1 <= n <= TREE_MAX, f"a tree has 1 to {TREE_MAX} tokens")
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
    kv, (_, B, hk, _, D) = _kv(k_cache, v_cache, False)
    dev = k_cache.device
    _need(q.dim() == 4 and cos.dim() == 2, "q must be [batch, tokens, heads, width], cos [positions, width / 2]")
    T, H = q.shape[1], q.shape[2]
    f32 = torch.float32
    qp = _rows(q, (B, T, H, D), f32, dev, "q")
    kp = _rows(k, (B, T, hk, D), f32, dev, "k")
    vp = _rows(v, (B, T, hk, D), f32, dev, "v")
    P = cos.shape[0]
    i32 = torch.int32
    cp, sp = _ints(cos, (P, D // 2), f32, dev, "cos"), _ints(sin, (P, D // 2), f32, dev, "sin")
    lp, pp = _ints(lens, (B,), i32, dev, "lens"), _ints(pos, (B, T), i32, dev, "pos")
    np_ = _ints(counts, (B,), i32, dev, "counts") if counts is not None else 0
    qn = _ints(q_norm, (D,), f32, dev, "q_norm") if q_norm is not None else 0
    kn = _ints(k_norm, (D,), f32, dev, "k_norm") if k_norm is not None else 0
    with _On(dev, stream) as st:
        if q_out is None:
            q_out = (torch.empty if counts is None else torch.zeros)(B, T, H, D, dtype=k_cache.dtype, device=dev)
        op = _rows(q_out, (B, T, H, D), k_cache.dtype, dev, "q_out")
        a = _APPEND.pack(qp[0], kp[0], vp[0], *qp[1:], *kp[1:], *vp[1:], T, H, lp, np_, pp, cp, sp, P, qn, kn, float(eps), *op)
        check(lib().p8_kv_append(kv, a, st), "p8_kv_append")
    return q_out


def tree_attention(q, k_cache, v_cache, lens, mask=None, counts=None, scale=None, out=None, lse=None, workspace=None, stream=None):
    """Attention of 1 to 64 tokens per sequence over the cache, their own keys and values already in it (kv_append).

    q [batch, tokens, heads, width] in the cache's type. Token t sees the whole sequence before the call's tokens and the
    tokens whose bits mask[t] has (int64 [tokens] or [batch, tokens], as tree_plan makes it; None: a chain). Returns
    (out like q, lse float32 [batch, tokens, heads]): the softmax average of the values and the natural log of the sum
    of exponentials; 0 and -inf for a token that sees nothing. scale: 1 / sqrt(width) unless given."""
    kv, (_, B, hk, _, D) = _kv(k_cache, v_cache, False)
    dev = k_cache.device
    _need(q.dim() == 4, "q must be [batch, tokens, heads, width]")
    T, H = q.shape[1], q.shape[2]
    qp = _rows(q, (B, T, H, D), k_cache.dtype, dev, "q")
    _need(1 <= T <= TREE_MAX and H % hk == 0 and H > 0, f"1 to {TREE_MAX} tokens, and query heads in whole groups")
    i32 = torch.int32
    lp = _ints(lens, (B,), i32, dev, "lens")
    np_ = _ints(counts, (B,), i32, dev, "counts") if counts is not None else 0
    mp, ms = 0, 0
    if mask is not None:
        ms = T if mask.dim() == 2 else 0
        mp = _ints(mask, (B, T) if ms else (T,), torch.int64, dev, "mask")
    if scale is None:
        scale = D ** -0.5
    with _On(dev, stream) as st:
        new = torch.empty if counts is None else torch.zeros
        if out is None:
            out = new(B, T, H, D, dtype=q.dtype, device=dev)
        if lse is None:
            lse = new(B, T, H, dtype=torch.float32, device=dev)
        op = _rows(out, (B, T, H, D), q.dtype, dev, "out")
        ep = _ints(lse, (B, T, H), torch.float32, dev, "lse")
        if workspace is None:
            workspace = torch.empty(lib().p8_tree_attn_workspace(kv, T, H), dtype=torch.uint8, device=dev)
        _need(workspace.device == dev and workspace.is_contiguous(), "workspace must be contiguous on the cache's device")
        a = _ATTN.pack(*qp, T, H, lp, np_, mp, ms, float(scale), *op, ep)
        check(lib().p8_tree_attn(kv, a, C.c_void_p(workspace.data_ptr()), workspace.numel() * workspace.element_size(), st), "p8_tree_attn")
    return out, lse


def attention_workspace_size(k_cache, tokens, heads):
    """workspace bytes of tree_attention on this cache, for callers that keep their own"""
    kv, _ = _kv(k_cache, k_cache, False)
    return int(lib().p8_tree_attn_workspace(kv, tokens, heads))


def attention_mass(q, lse, k_cache, lens, mass, rows=None, counts=None, scale=None, out=None, stream=None):
    """Adds to mass float32 [batch, kv heads, slots] the attention weight that each slot drew from a chain of tokens
    behind the sequence, summed over them and over the query heads of the slot's cache head.

    q, lse: as in the tree_attention call. rows int32 [batch, tokens]: the tokens' rows in q and lse (the accepted path,
    once tree_accept has moved its keys into place); None: 0, 1, 2, ... counts: how many tokens. The tokens' own slots
    start at 0. In place unless out is given."""
    kv, (_, B, hk, S, D) = _kv(k_cache, None, False)
    dev = k_cache.device
    _need(q.dim() == 4, "q must be [batch, tokens, heads, width]")
    T, H = q.shape[1], q.shape[2]
    qp = _rows(q, (B, T, H, D), k_cache.dtype, dev, "q")
    _need(1 <= T <= TREE_MAX and H % hk == 0 and H > 0, f"1 to {TREE_MAX} tokens, and query heads in whole groups")
    i32, f32 = torch.int32, torch.float32
    lp = _ints(lens, (B,), i32, dev, "lens")
    ep = _ints(lse, (B, T, H), f32, dev, "lse")
    np_ = _ints(counts, (B,), i32, dev, "counts") if counts is not None else 0
    rp = _ints(rows, (B, T), i32, dev, "rows") if rows is not None else 0
    if out is None:
        out = mass
    for t in (mass, out):
        _need(t.dtype == f32 and tuple(t.shape) == (B, hk, S) and t.stride(2) == 1 and t.device == dev, "mass and out must be float32 [batch, kv heads, slots] with unit slot stride on the cache's device")
    if scale is None:
        scale = D ** -0.5
    with _On(dev, stream) as st:
        a = _MASS.pack(*qp, T, H, ep, lp, np_, rp, float(scale), mass.data_ptr(), mass.stride(0), mass.stride(1), out.data_ptr(), out.stride(0), out.stride(1))
        check(lib().p8_attn_mass(kv, a, st), "p8_attn_mass")
    return out


def kv_evict(k_cache, v_cache, mass, lens, budget, sinks=0, recent=0, k_out=None, v_out=None, mass_out=None, new_lens=None, kept=None, stream=None):
    """Shortens every sequence with more than `budget` slots to `budget`, per layer and cache head: the first `sinks`
    slots, the last `recent`, and of the others those with the largest mass (ties: the lowest slot), in order.

    Cache [layers, batch, kv heads, slots, width] or without layers, mass float32 of its first dimensions. The kept
    slots go to the front of k_out, v_out and mass_out (other buffers, budget slots or more; give all three), or of the
    cache itself. Returns (new_lens int32 [batch], kept int32 [..., kv heads, budget]: the kept slots, -1 behind them)."""
    kv, (N, B, hk, S, D) = _kv(k_cache, v_cache, True)
    dev = k_cache.device
    place = k_out is None
    _need((v_out is None) == place and (mass_out is None) == place, "give k_out, v_out and mass_out together")
    if place:
        kv2, S2, mass_out = kv, S, mass
    else:
        _need(k_out.dim() == k_cache.dim() and k_out.dtype == k_cache.dtype and k_out.device == dev, "k_out must have the cache's dimensions, type and device")
        kv2, shape = _kv(k_out, v_out, True)
        S2 = shape[3]
        _need(shape == (N, B, hk, S2, D), "k_out must have the cache's shape but for its slots")
    budget = int(budget)
    lead = k_cache.shape[:-2]
    ms = []
    for t, s in ((mass, S), (mass_out, S2)):
        _need(t.dtype == torch.float32 and tuple(t.shape) == (*lead, s) and t.stride(-1) == 1 and t.device == dev, "mass must be float32 [.., kv heads, slots] of the cache with unit slot stride")
        st = t.stride()
        ms.append((st[0], st[1], st[2]) if len(lead) == 3 else (0, st[0], st[1]))
    i32 = torch.int32
    lp = _ints(lens, (B,), i32, dev, "lens")
    with _On(dev, stream) as st:
        if new_lens is None:
            new_lens = torch.empty_like(lens)
        if kept is None:
            kept = torch.empty(*lead, max(budget, 0), dtype=i32, device=dev)
        a = _EVICT.pack(mass.data_ptr(), *ms[0], mass_out.data_ptr(), *ms[1], lp, _ints(new_lens, (B,), i32, dev, "new_lens"), _ints(kept, (*lead, budget), i32, dev, "kept"), budget, int(sinks), int(recent))
        check(lib().p8_kv_evict(kv, kv2, a, st), "p8_kv_evict")
    return new_lens, kept


def tree_accept(tokens, parents, target, k_cache, v_cache, lens, counts=None, path=None, accepted=None, next_token=None, new_lens=None, stream=None):
    """Greedy verification of drafted trees: tokens int64 [batch, tokens] (token 0 the last known one), parents int32,
    target int64 (the model's choice after each token). From token 0 the path goes on to the lowest child that is what
    the target chose; its keys and values move, in all layers of the cache [layers, batch, kv heads, slots, width] (or
    without layers), to the slots right behind the sequence.

    Returns Accepted(path int32 [batch, tokens] (-1 behind it), accepted int32 [batch] its length, next_token int64
    [batch] the target at its end, new_lens int32 [batch])."""
    kv, (_, B, _, _, _) = _kv(k_cache, v_cache, True)
    dev = k_cache.device
    _need(tokens.dim() == 2 and 1 <= tokens.shape[1] <= TREE_MAX, f"tokens must be [batch, 1 to {TREE_MAX}]")
    T = tokens.shape[1]
    i32, i64 = torch.int32, torch.int64
    tp, gp, pp = _ints(tokens, (B, T), i64, dev, "tokens"), _ints(target, (B, T), i64, dev, "target"), _ints(parents, (B, T), i32, dev, "parents")
    lp = _ints(lens, (B,), i32, dev, "lens")
    np_ = _ints(counts, (B,), i32, dev, "counts") if counts is not None else 0
    with _On(dev, stream) as st:
        if path is None:
            path = torch.empty(B, T, dtype=i32, device=dev)
        if accepted is None:
            accepted = torch.empty(B, dtype=i32, device=dev)
        if next_token is None:
            next_token = torch.empty(B, dtype=i64, device=dev)
        if new_lens is None:
            new_lens = torch.empty(B, dtype=i32, device=dev)
        a = _ACCEPT.pack(tp, gp, pp, T, lp, np_, _ints(path, (B, T), i32, dev, "path"), _ints(accepted, (B,), i32, dev, "accepted"),
                         _ints(new_lens, (B,), i32, dev, "new_lens"), _ints(next_token, (B,), i64, dev, "next_token"))
        check(lib().p8_tree_accept(kv, a, st), "p8_tree_accept")
    return Accepted(path, accepted, next_token, new_lens)
