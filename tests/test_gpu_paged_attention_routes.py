"""Both kernels of attention over a paged cache, pinned, on calls that the automatic choice would give to the other one.
Tolerances as in test_gpu_paged_attention.py, where they are derived."""
import math

import pytest
import torch

from test_gpu_paged_attention import BITS, DEV, Batch, queries
from VAR_Q import _cabi

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["tc", "decode"], autouse=True)
def path(request):
    _cabi.force_attn_path(request.param)
    yield request.param
    _cabi.force_attn_path(None)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kb,vb", BITS)
@pytest.mark.parametrize("counts,G", [([1, 1, 1], 1), ([1, 1, 1], 7), ([3, 2, 5], 4), ([33, 1, 100], 2), ([300, 257, 129], 1)])
def test_any_number_of_rows(D, kb, vb, counts, G):
    b = Batch([700, 260, 131], 2, D, kb, vb, page=32, seed=D + kb + G)
    q = queries(sum(counts), 2 * G, D, torch.bfloat16 if G == 4 else torch.float16)
    b.check(q, counts)
    b.check(q, counts, causal=False)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kb,vb", BITS)
@pytest.mark.parametrize("G,most,n", [(1, 24, 300), (5, 4, 90), (3, 7, 2000)])
def test_seventeen_to_twenty_four_rows(D, kb, vb, G, most, n):
    """many sequences with 17 to 24 rows of a head at most: one row tile holds them; some sequences have fewer, or none"""
    heads = 8
    kv = [n + 7 * i if i % 4 else i for i in range(8)]
    counts = [max(most - i, 0) if i != 3 else 0 for i in range(8)]
    b = Batch(kv, heads, D, kb, vb, page=16, seed=D + kb + most)
    q = queries(sum(counts), heads * G, D, torch.bfloat16 if G == 5 else torch.float16)
    b.check(q, counts)
    b.check(q, counts, causal=False)
    b.check(q, counts, window=33, sinks=5)


@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 1), (17, 5), (64, 64), (127, 0), (200, 130)])
@pytest.mark.parametrize("c", [1, 9, 150])
def test_windows(window, sinks, c):
    b = Batch([900, 150 + c], 2, 64, 4, 8, page=64, seed=window)
    b.check(queries(2 * c, 4, 64), [c, c], window=window, sinks=sinks)


@pytest.mark.parametrize("heads,G,c,n", [(1, 1, 1, 5000), (1, 2, 4, 9000), (2, 1, 40, 6000), (1, 1, 300, 7000), (1, 8, 1, 40000)])
def test_split_calls(heads, G, c, n):
    """few rows over long contexts: parts in clusters, parts in the workspace, both kinds of merge"""
    b = Batch([n], heads, 128, 8, 4, page=128, seed=n)
    q = queries(c, heads * G, 128, torch.bfloat16)
    b.check(q, [c])
    first = b.attend(q, [c], 0.1)
    again = b.attend(q, [c], 0.1)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_many_short_sequences():
    kv = [i % 40 for i in range(300)]
    b = Batch(kv, 1, 64, page=16, seed=1)
    b.check(queries(300, 3, 64), [1] * 300)
    b.check(queries(300, 3, 64), [1] * 300, causal=False)


@pytest.mark.parametrize("gain", [1e-5, 40.0])
@pytest.mark.parametrize("c", [1, 140])
def test_scaled_rows_next_to_usual_ones(gain, c):
    """bf16 queries outside fp16's comfortable range share a tile with others"""
    b = Batch([500], 1, 64, page=16, seed=2)
    q = queries(c, 4, 64, torch.bfloat16)
    q[:, 1] *= gain
    q[0, 2] *= 1e-30
    b.check(q, [c])


def test_values_and_keys_that_are_zero(path):
    b = Batch([200], 1, 64, page=16, seed=3)
    zeros = torch.zeros((100, 1, 64), device=DEV)
    b.cache.append(zeros, zeros, b.slots[0][50:150].to(DEV))
    for c in (1, 60):
        b.check(queries(c, 2, 64, gain=4.0), [c])


def test_both_kernels_agree(path):
    b = Batch([1000, 37], 2, 128, 4, 4, page=64, seed=4)
    q = queries(60, 4, 128)
    out = b.attend(q, [30, 30], 1 / math.sqrt(128))
    _cabi.force_attn_path("decode" if path == "tc" else "tc")
    other = b.attend(q, [30, 30], 1 / math.sqrt(128))
    assert (out[1] - other[1]).abs().max().item() <= 2.0 ** -15 * 2
    assert (out[0].double() - other[0].double()).abs().max().item() <= 2 * 2.0 ** -10 * 8.0      # each side's bound, |v| < 8
