"""Scales of a paged cache that nobody wrote, that nobody sees, or that are at the ends of fp32.

Unseen: bit for bit what comes out over clean pools.  Seen: against the formula, tolerances as in test_gpu_paged_attention.py, where they are derived."""
import math

import pytest
import torch

from test_gpu_paged_attention import DEV, Batch, queries
from VAR_Q import _cabi

pytestmark = pytest.mark.gpu
# subnormals (what small integers look like), zeros, negative numbers, the ends of the range, infinities, NaN
PATTERNS = [1, 5, 0x1fffff, 0x400000, 0x7fffff, 0x800000, 0, 0x80000000, 0x80000001, 0xbf800000, 0x7f7fffff, 0xff7fffff, 0x7f800000, 0xff800000, 0x7fc00000]


@pytest.fixture(params=["tc", "decode"], autouse=True)
def path(request):
    _cabi.force_attn_path(request.param)
    yield request.param
    _cabi.force_attn_path(None)


def bits_of(pattern):
    return pattern - (1 << 32) if pattern >= 1 << 31 else pattern


def put(cache, slots, pattern, names=("k_scale", "v_scale")):
    for name in names:
        flat = getattr(cache, name).view(torch.int32)
        flat[slots.to(DEV) // cache.page_size, :, slots.to(DEV) % cache.page_size] = bits_of(pattern)


def everything_but(cache, kept):
    rest = torch.ones(cache.num_pages * cache.page_size, dtype=torch.bool)
    rest[torch.cat(kept)] = False
    return rest.nonzero().flatten()


@pytest.mark.parametrize("D,kb,vb", [(64, 8, 8), (128, 4, 4), (64, 2, 2)])
@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [3, 40, 1, 130]])
def test_what_is_not_written_does_not_matter(D, kb, vb, counts):
    """lengths that end inside a tile, a page, or a copy of 16 rows"""
    b = Batch([3, 50, 333, 201], 2, D, kb, vb, page=32, seed=D)
    q = queries(sum(counts), 4, D)
    rest = everything_but(b.cache, b.slots)
    put(b.cache, rest, 0x3f800000)
    clean = b.check(q, counts)
    whole = b.check(q, counts, causal=False)
    for pattern in PATTERNS:
        put(b.cache, rest, pattern)
        for ref, kw in ((clean, {}), (whole, {"causal": False})):
            out, lse = b.attend(q, counts, 1.0 / math.sqrt(D), **kw)
            assert torch.equal(out, ref[0]) and torch.equal(lse, ref[1]), hex(pattern)


@pytest.mark.parametrize("window,sinks", [(50, 3), (7, 0), (130, 65)])
@pytest.mark.parametrize("c", [1, 5, 70])
def test_what_lies_in_front_of_the_window_does_not_matter(window, sinks, c):
    """tokens that every query has left behind: never written, or in pages that are zero or others' now"""
    n = 500
    b = Batch([n, n - 77], 2, 64, page=16, seed=window)
    q = queries(2 * c, 4, 64)
    hidden = torch.cat([s[sinks:max(sinks, len(s) - c - window + 1)] for s in b.slots])
    put(b.cache, hidden, 0x3f800000)
    clean = b.check(q, [c, c], window=window, sinks=sinks)
    for pattern in PATTERNS:
        put(b.cache, hidden, pattern)
        out, lse = b.attend(q, [c, c], 0.125, window=window, sinks=sinks)
        assert torch.equal(out, clean[0]) and torch.equal(lse, clean[1]), hex(pattern)


@pytest.mark.parametrize("pattern", [0, 1, 5, 0x1fffff, 0x400000, 0x7fffff, 0x800000])
@pytest.mark.parametrize("c", [1, 40])
@pytest.mark.parametrize("every", [1, 3, 1000])
def test_seen_values_that_are_zero_keep_their_weight(pattern, c, every):
    """V scales of 0 or next to it, in tiles with and without masks: the key's value is (as good as) zero, its weight counts"""
    b = Batch([300, 75], 2, 64, page=16, seed=every)
    put(b.cache, torch.cat([s[::every] for s in b.slots]), pattern, ("v_scale",))
    put(b.cache, b.slots[0][17:20], pattern, ("v_scale",))
    q = queries(2 * c, 4, 64)
    b.check(q, [c, c])
    b.check(q, [c, c], causal=False)
    b.check(q, [c, c], window=60, sinks=19)


def test_keys_that_are_zero_answer_nothing():
    """K scales of 0: a score of 0, in V's weight as any other"""
    b = Batch([300, 75], 2, 64, page=16, seed=1)
    put(b.cache, torch.cat([s[::3] for s in b.slots]), 0, ("k_scale",))
    for c in (1, 40):
        b.check(queries(2 * c, 4, 64), [c, c])


@pytest.mark.parametrize("pattern", [0x7f800000, 0x7fc00000, 0xbf800000])
@pytest.mark.parametrize("at", [0, 20, 290])
@pytest.mark.parametrize("c", [1, 40])
def test_scales_that_are_no_sizes_spoil_the_rows_that_see_them(pattern, at, c):
    b = Batch([300], 2, 64, page=16, seed=at)
    q = queries(c, 4, 64)
    clean = b.check(q, [c])
    put(b.cache, b.slots[0][at:at + 1], pattern, ("v_scale",))
    out, lse = b.attend(q, [c], 0.125)
    first = max(0, at - (300 - c))                                     # queries from here on see the key
    assert torch.isnan(out[first:]).all() and torch.isnan(lse[first:]).all()
    assert torch.equal(out[:first], clean[0][:first]) and torch.equal(lse[:first], clean[1][:first])


@pytest.mark.parametrize("c", [1, 40])
@pytest.mark.parametrize("vb,size", [(2, 1.2), (2, 1.9), (4, 1.9), (8, 1.9)])
def test_values_next_to_the_end_of_fp32(c, vb, size):
    """V up to size * 2^127: with 2 and 4 bits its scales are above 2^125, whose inverses are next to or below the smallest normal number.
    The other rows are 2^27 times smaller: weights times V scale of one row have to lie within 2^126 of one another."""
    n, D = 90, 64
    b = Batch([n], 1, D, 8, vb, page=16, seed=vb, v_gain=lambda j: torch.full_like(j, 2.0 ** 100, dtype=torch.float32))
    g = torch.Generator().manual_seed(7)
    slots = b.slots[0][1::3].to(DEV)
    v = (torch.rand((len(slots), 1, D), generator=g) * 2 - 1) * size * 2.0 ** 127
    v[:, 0, 5] = size * 2.0 ** 127
    b.cache.append(torch.randn((len(slots), 1, D), generator=g).to(DEV), v.to(DEV), slots)
    b.check(queries(c, 2, D, torch.bfloat16), [c])
    b.check(queries(c, 2, D, torch.bfloat16), [c], causal=False)
