"""Paged caches without a GPU: sizes whose products leave an int, and what is left behind when a call fails."""
import pytest

from test_paged_cpu import good
from VAR_Q import _cabi


@pytest.mark.parametrize("q_heads,n_queries,max_q,ok", [(1 << 16, 1 << 17, 1 << 17, False), (1 << 16, 1 << 17, 1 << 20, False), (2 << 20, 2047, 2047, True), (2 << 20, 2048, 2048, False),
                                                        (1 << 16, 1 << 17, 4, True)])
def test_rows_of_a_head_are_counted_in_an_int(q_heads, n_queries, max_q, ok):
    """query rows of a sequence and head of the cache: below 2^31 - 512 (two tiles of 256 behind them)"""
    lib = _cabi.lib()
    cache, batch, t = good()
    batch.q_heads, batch.n_queries, batch.max_q, batch.causal = q_heads, n_queries, max_q, 1
    batch.window, batch.sinks = 0, 0
    if ok:                                                               # a refusal that comes behind this one
        batch.q_starts = None
    rc = lib.varq_paged_attn(cache, batch, t, t, None, None, 0, None)
    assert (rc, b"query rows" in lib.varq_last_error()) == ((-1, False) if ok else (-2, True))


def test_a_step_that_finds_no_pages_leaves_no_sequence_behind():
    import torch

    from VAR_Q.harness import StandInDecoder
    model = StandInDecoder(depth=1, width=64, heads=2, kv_heads=1, head_dim=64, num_pages=2, page_size=16, device="cpu")
    model.table.add("old")
    with pytest.raises(RuntimeError, match="pages"):
        model.step(["old", "new"], [torch.zeros(1, 64), torch.zeros(33, 64)])
    assert "new" not in model.table and "old" in model.table and model.table.length("old") == 0 and model.table.free_pages == 2
    model.table.add("new")                                               # as if it had never been there
    with pytest.raises(ValueError):
        model.step(["new", "twice", "twice"], [torch.zeros(1, 64)] * 3)
    assert "twice" not in model.table and "new" in model.table
