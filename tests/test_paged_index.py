"""The index arithmetic of the paged operators on the host: division by page sizes, the attention's shares, and what its warps and
its joining launch make of them."""
import ctypes as C
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = """
#include "p8_paged_index.h"
extern "C" {
uint32_t page_of_(uint32_t page, uint32_t slot) { return p8::page_of(p8::page_div(page), slot); }
// the largest slot up to `slots` at which quotients of a page size are wrong, -1: none; every slot around multiples
int64_t wrong(uint32_t page, uint32_t slots) {
    const p8::PageDiv d = p8::page_div(page);
    for (uint64_t q = 0; q * page <= slots; q += 1 + q / 64)
        for (int64_t s = (int64_t)(q * page) - 2; s <= (int64_t)(q * page) + 2; ++s)
            if (s >= 0 && s <= slots && p8::page_of(d, (uint32_t)s) != s / page) return s;
    return -1;
}
int unit_places(int t, int least) { return p8::unit_places(t, least); }
int64_t cta_share(int64_t t, int64_t c, int64_t least) { return p8::cta_share(t, c, least); }
int warp_first(int s, int w, int n) { return p8::warp_first(s, w, n); }
int nth_bit(uint64_t m, int k) { return p8::nth_bit(m, k); }
uint32_t order_key(uint32_t b) { return p8::order_key(b); }
uint32_t order_bits(uint32_t k) { return p8::order_bits(k); }
int64_t select_splits(int64_t r, int64_t b, int64_t v, int64_t s, int64_t l, int64_t x) { return p8::select_splits(r, b, v, s, l, x); }
}
"""


@pytest.fixture(scope="module")
def ix(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged_index")
    (d / "x.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-I", os.path.join(ROOT, "pingala8_llm_b200", "csrc"), str(d / "x.cpp"), "-o", str(d / "x.so")], check=True)
    L = C.CDLL(str(d / "x.so"))
    i64, u32, u64 = C.c_int64, C.c_uint32, C.c_uint64
    for name, res, args in (("page_of_", u32, [u32, u32]), ("wrong", i64, [u32, u32]), ("unit_places", C.c_int, [C.c_int, C.c_int]), ("cta_share", i64, [i64, i64, i64]), ("warp_first", C.c_int, [C.c_int, C.c_int, C.c_int]),
                            ("nth_bit", C.c_int, [u64, C.c_int]), ("order_key", u32, [u32]), ("order_bits", u32, [u32]), ("select_splits", i64, [i64] * 6)):
        getattr(L, name).restype, getattr(L, name).argtypes = res, args
    return L


def test_slots_are_divided_by_any_page_size(ix):
    for page in (*range(1, 130), 255, 256, 257, 1000, 4096, 65535, 65536, 65537, 999983, (1 << 20) - 1, 1 << 20):
        assert ix.wrong(page, (1 << 30) + 5) == -1, page
        for slot in (0, 1, page - 1, page, (1 << 30) - 1, 1 << 30):
            assert ix.page_of_(page, slot) == slot // page


def test_bits_and_orders(ix):
    rng = random.Random(0)
    for _ in range(300):
        m = rng.getrandbits(64) | 1 << rng.randrange(64)
        bits = [i for i in range(64) if m >> i & 1]
        k = rng.randrange(len(bits))
        assert ix.nth_bit(m, k) == bits[k]
    import struct
    xs = sorted([rng.uniform(-1e3, 1e3) for _ in range(200)] + [0.0, 1e-45, -1e-45, float("inf"), -float("inf"), 3.4e38, -3.4e38])
    bits = [struct.unpack("<I", struct.pack("<f", x))[0] for x in xs]
    keys = [ix.order_key(b) for b in bits]
    assert keys == sorted(keys) and [ix.order_bits(k) for k in keys] == bits


def walk(ix, units, tiles, ctas, least, warps, pad):
    """What the kernel's CTAs leave for `tiles` [sequences]: {unit: its tiles in pieces}, {part of the workspace: unit}, {unit: who notes its cut}"""
    places = [ix.unit_places(t, pad) for t in tiles]
    total = units * sum(places)
    share = ix.cta_share(total, ctas, least)
    start, at = {}, 0
    for b, c in enumerate(places):
        for u in range(units):
            start[b, u] = at
            at += c
    order = sorted(((s, k) for k, s in start.items() if places[k[0]]), key=lambda x: x[0])
    covered, parts, cuts = {}, {}, {}
    for cta in range(ctas):
        pieces = []
        for w in range(warps):
            p = cta * share + ix.warp_first(share, w, warps)
            end = min(cta * share + ix.warp_first(share, w + 1, warps), total)
            slots = set()
            for s, (b, u) in order:
                lo, hi = max(p, s), min(end, s + places[b])
                if lo >= hi:
                    continue
                t0, t1 = lo - s, min(hi - s, tiles[b])
                if t0 >= t1:
                    continue
                covered.setdefault((b, u), []).append((t0, t1))
                if t0 == 0 and t1 == tiles[b]:
                    cuts.setdefault((b, u), []).append((0, 0))
                    continue
                slot = 1 if hi == end else 0  # at the warp's end in place of its tiles, before that in the workspace
                assert slot not in slots, "two pieces of a warp in one place"
                slots.add(slot)
                pieces.append((w, slot, (b, u), t0 == 0, t1 == tiles[b]))
        pieces.sort()
        i = 0
        while i < len(pieces):
            j = i
            while j < len(pieces) and pieces[j][2] == pieces[i][2]:
                j += 1
            left, right = pieces[i][3], pieces[j - 1][4]
            if left:
                b, u = pieces[i][2]
                further = (start[b, u] - cta * share + tiles[b] - 1) // share
                cuts.setdefault((b, u), []).append((cta, cta + further))
                assert right == (further == 0)
            if not (left and right):
                key = (cta, 1 if left else 0)
                assert key not in parts, "two parts of a CTA in one place"
                parts[key] = pieces[i][2]
            i = j
    return start, share, total, covered, parts, cuts


@pytest.mark.parametrize("seed", range(60))
def test_shares_cover_every_tile_once_and_the_join_finds_all_parts(ix, seed):
    rng = random.Random(seed)
    ctas, least, warps = rng.choice([3, 7, 20, 44]), rng.choice([1, 2, 8, 12, 24]), rng.choice([4, 8, 10, 12])
    units, B = rng.choice([1, 2, 8]), rng.choice([1, 2, 5, 40])
    tiles = [rng.choice([0, 1, 2, rng.randint(0, 30), rng.randint(0, 400)]) for _ in range(B)]
    start, share, total, covered, parts, cuts = walk(ix, units, tiles, ctas, least, warps, least if units * B <= ctas else 1)
    assert share * ctas >= total
    used = -(-total // share) if total else 0
    assert used <= units * sum(1 for _ in tiles) * max(1, -(-max(tiles) // least))  # the grid's bound
    left = dict(parts)
    for b, t in enumerate(tiles):
        for u in range(units):
            got = sorted(covered.get((b, u), []))
            assert [x for x, _ in got] == [0] * (t > 0) + [y for _, y in got[:-1]] and (not t or got[-1][1] == t)
            s = start[b, u]
            c0, c1 = s // share, (s + t - 1) // share if t else s // share
            if t:
                (cut,) = cuts[b, u]
                assert cut == ((c0, c1) if c1 > c0 else cut) and (c1 > c0) == (cut[1] > cut[0])
            for c in range(c0, c1 + 1) if c1 > c0 else ():
                assert left.pop((c, 1 if c == c0 else 0)) == (b, u)
    assert not left  # and nothing lies in the workspace that no one joins


def test_rows_of_logits_are_split_within_the_lists(ix):
    for rows, beams in ((1, 1), (4, 4), (12, 4), (256, 8), (64, 64), (4096 * 64, 64), (3, 3), (7, 1)):
        for vocab in (1, 15, 4096, 4097, 50001, 151936, 2 ** 31 - 65537):
            s = ix.select_splits(rows, beams, vocab, 444, 4096, 100000)
            chunk = (-(-vocab // s) + 127) // 128 * 128
            assert 1 <= s and s * beams <= 256 and chunk * s >= vocab and chunk * s < 2 ** 31
