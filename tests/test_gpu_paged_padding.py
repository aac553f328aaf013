"""Query rows that belong to no sequence (a batch padded to a fixed size, as a graph has it): zeros and -inf, like a query that sees nothing, on every route of both
kernels.  Tolerances of the other rows as in test_gpu_paged_attention.py, where they are derived."""
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


def leave_nan_behind():
    """blocks of the allocator that are handed out next hold NaN"""
    for size in (1 << 9, 1 << 12, 1 << 15, 1 << 18, 1 << 21, 1 << 24):
        held = [torch.full((size,), float("nan"), device=DEV) for _ in range(4)]
        del held


@pytest.mark.parametrize("front,behind", [(0, 1), (0, 500), (3, 0), (129, 70)])
@pytest.mark.parametrize("kv,counts,heads,G", [([300, 50], [1, 1], 2, 2), ([300, 50], [9, 40], 2, 1), ([20000], [1], 1, 2), ([20000], [150], 1, 2), ([700] * 70, [2] * 70, 3, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_of_no_sequence(front, behind, kv, counts, heads, G, D):
    """one part of the keys, parts in clusters, parts in the workspace; padding in front and behind"""
    b = Batch(kv, heads, D, page=64, seed=len(kv))
    n = sum(counts)
    q = queries(front + n + behind, heads * G, D)
    starts = torch.tensor([front + sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device=DEV)
    leave_nan_behind()
    out, lse = b.cache.attend(q, b.table.to(DEV), b.kv_dev, starts, max(counts), max(kv), D ** -0.5, return_lse=True)
    b.check(q[front:front + n], counts, out=(out[front:front + n], lse[front:front + n]))
    for rows in (slice(0, front), slice(front + n, None)):
        assert (out[rows] == 0).all() and (lse[rows] == -float("inf")).all()


def test_no_sequences_and_no_queries():
    b = Batch([100], 2, 64, seed=1)
    q, table = queries(5, 4, 64), b.table.to(DEV)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    for args in ((table[:0], b.kv_dev[:0], ints(0), 5, 100), (table[:0], b.kv_dev[:0], ints(0), 0, 0), (table, b.kv_dev, ints(0, 0), 0, 100), (table, b.kv_dev, ints(2, 2), 0, 0),
                 (table, b.kv_dev, ints(5, 5), 3, 100)):
        leave_nan_behind()
        out, lse = b.cache.attend(q, *args, 0.125, return_lse=True)
        assert (out == 0).all() and (lse == -float("inf")).all()
        assert _cabi.device_status() == 0


def test_a_bound_of_no_queries_that_does_not_hold_is_reported():
    b = Batch([100], 2, 64, seed=1)
    starts = torch.tensor([0, 5], dtype=torch.int32, device=DEV)
    b.cache.attend(queries(5, 4, 64), b.table.to(DEV), b.kv_dev, starts, 0, 100, 0.125)
    assert _cabi.device_status() == 64
