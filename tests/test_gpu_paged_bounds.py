"""Attention over a paged cache where its numbers are large or its pages are gone: pages that no query sees any more, windows and first tokens up to the
largest int, lengths next to it.  Both kernels; tolerances as in test_gpu_paged_attention.py, where they are derived."""
import math

import pytest
import torch

from test_gpu_paged_attention import DEV, Batch, queries
from VAR_Q import _cabi

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["tc", "decode"], autouse=True)
def path(request):
    _cabi.force_attn_path(request.param)
    yield request.param
    _cabi.force_attn_path(None)


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("window,sinks", [(50, 3), (7, 0), (130, 40)])
@pytest.mark.parametrize("c", [1, 5, 70, 200])
def test_pages_that_no_query_sees_need_not_be_there(page, window, sinks, c):
    """a server gives the pages in front of the window back and leaves -1 in the table"""
    b = Batch([600, 523], 2, 64, page=page, seed=page)
    q = queries(2 * c, 4, 64)
    clean = b.check(q, [c, c], window=window, sinks=sinks)
    gone = 0
    for i, n in enumerate(b.kv):
        first = n - c - window + 1
        for p in range(-(-sinks // page), first // page):
            b.table[i, p], gone = -1, gone + 1
    assert gone > 0
    out, lse = b.attend(q, [c, c], 0.125, window=window, sinks=sinks)
    assert torch.equal(out, clean[0]) and torch.equal(lse, clean[1])
    assert _cabi.device_status() == 0


INT_MAX = 2 ** 31 - 1


@pytest.mark.parametrize("sinks", [1 << 30, INT_MAX - 1024, INT_MAX - 62, INT_MAX - 14, INT_MAX])
@pytest.mark.parametrize("c", [1, 100])
def test_all_tokens_as_first_tokens(sinks, c):
    b = Batch([500, 111], 2, 64, page=16, seed=3)
    q = queries(2 * c, 4, 64)
    out = b.check(q, [c, c], window=5, sinks=sinks)
    b.check(q, [c, c], out=out)                                        # nothing is hidden


@pytest.mark.parametrize("window", [1 << 30, INT_MAX - 600, INT_MAX - 1, INT_MAX])
@pytest.mark.parametrize("sinks", [0, 200, INT_MAX])
@pytest.mark.parametrize("counts", [[1, 1, 2], [5, 9, 700], [3, 90, 130]])
def test_windows_that_hold_everything(window, sinks, counts):
    """with more queries than tokens: the first ones stand in front of the sequence"""
    b = Batch([3, 60, 120], 2, 64, page=16, seed=4)
    q = queries(sum(counts), 4, 64)
    out = b.check(q, counts, window=window, sinks=sinks)
    b.check(q, counts, out=out)


def test_the_longest_sequences(path):
    """2^31 - 4096 tokens, all in one page; more are clamped and reported.  Sums of up to 2^18 fp32 terms, each addition off by 2^-22 of the sum at most (the tensor
    core's additions truncate): 2^-4 relative, 2^-4 absolute for the log of the sum"""
    D, page, most = 64, 1024, 2 ** 31 - 4096
    b = Batch([page], 1, D, 2, 2, page=page, seed=5)
    q = queries(1, 1, D)
    ref, ref_lse, bound, _ = b.reference(q, [1], 0.125)
    table = torch.full((1, 2 ** 31 // page), int(b.table[0, 0]), dtype=torch.int32, device=DEV)
    table[0, most // page:] = -1
    starts = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    for kv, status in ((most, 0), (most + 1, 65), (INT_MAX, 65)):
        lens = torch.tensor([kv], dtype=torch.int32, device=DEV)
        out, lse = b.cache.attend(q, table, lens, starts, 1, kv, 0.125, return_lse=True)
        assert _cabi.device_status() == status
        assert ((out.double() - ref).abs() <= 2.0 ** -4 * bound + 1e-3).all()
        assert (lse - (ref_lse + math.log(most // page))).abs().item() <= 2.0 ** -4
