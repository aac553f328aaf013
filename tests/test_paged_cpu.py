"""Paged caches without a GPU: the page table, what the constructor and the C entry points refuse."""
import pytest
import torch

from VAR_Q import _cabi
from VAR_Q.paged import PagedCache, PageTable


def test_page_table_hands_out_and_takes_back_pages():
    t = PageTable(5, 16)
    t.add(1); t.add(2)
    s = t.extend([1, 2], [17, 16], "cpu")
    assert len(set(s.tolist())) == 33 and t.free_pages == 2
    assert s.dtype == torch.int64 and torch.equal(t.slots(1, "cpu"), s[:17]) and torch.equal(t.slots(2, "cpu"), s[17:])
    more = t.extend([2], [1], "cpu")
    assert t.free_pages == 1 and more.item() % 16 == 0
    table, lens, starts, max_q, max_kv = t.batch([2, 1], [1, 2], "cpu")
    assert table.tolist()[0][0] == s[17].item() // 16 and lens.tolist() == [17, 17] and starts.tolist() == [0, 1, 3] and (max_q, max_kv) == (2, 17)
    assert table.dtype == lens.dtype == starts.dtype == torch.int32
    with pytest.raises(RuntimeError, match="3 pages needed, 1 are free"):
        t.extend([1, 2], [32, 16], "cpu")
    assert t.free_pages == 1 and t.length(1) == 17                       # nothing was taken
    t.remove(1)
    assert t.free_pages == 3
    with pytest.raises(KeyError):
        t.length(1)


def test_page_table_edges():
    t = PageTable(2, 16)
    t.add("x")
    assert t.slots("x", "cpu").shape == (0,) and t.extend(["x"], [0], "cpu").shape == (0,)
    table, lens, starts, max_q, max_kv = t.batch(["x"], [0], "cpu")
    assert table.shape == (1, 0) and lens.tolist() == [0] and (max_q, max_kv) == (0, 0)
    assert t.batch([], [], "cpu")[2].tolist() == [0]
    for args in ((["x", "x"], [1, 1]), (["x"], [1, 2]), (["x"], [-1])):
        with pytest.raises(ValueError):
            t.extend(*args, "cpu")
    with pytest.raises(ValueError):
        t.add("x")
    t.extend(["x"], [16], "cpu")
    assert t.free_pages == 1                                             # a full page asks for no next one


@pytest.mark.parametrize("kw", [dict(head_dim=96), dict(page_size=8), dict(page_size=48), dict(page_size=2048), dict(k_bits=3), dict(v_bits=16), dict(num_pages=0),
                                dict(num_heads=0)])
def test_constructor_refuses(kw):
    args = dict(num_pages=2, page_size=16, num_heads=2, head_dim=64, device="cpu")
    args.update(kw)
    with pytest.raises(ValueError, match="VAR-Q"):
        PagedCache(**args)


def test_cpu_tensors_are_refused():
    cache = PagedCache(2, 16, 2, 64, 4, 2, device="cpu")
    assert cache.k_codes.shape == (2, 2, 16, 8) and cache.v_codes.shape == (2, 2, 16, 4) and (cache.k_bits, cache.v_bits) == (4, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        cache.read(torch.zeros(1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA"):
        cache.append(torch.zeros(1, 2, 64), torch.zeros(1, 2, 64), torch.zeros(1, dtype=torch.int64))


def good():
    """descriptors that pass every check in front of the pointers' first use; addresses are never touched on the host"""
    cache = _cabi.Paged(256, 256, 256, 256, 4, 16, 2, 64, 8, 8)
    batch = _cabi.PagedBatch(256, 256, 256, 4, 6, 4, 2, 4, 3, 64, 1, 0, 0, 0.125)
    t = _cabi.Tensor(256, _cabi.F16, 0, 0, 128, 64)
    return cache, batch, t


@pytest.mark.parametrize("field,value,rc,word", [
    ("n_pages", 0, -1, b"pages"), ("page_size", 24, -1, b"page"), ("page_size", 8, -1, b"page"), ("head_dim", 80, -2, b"head_dim"), ("k_bits", 3, -1, b"bits"),
    ("v_bits", 16, -1, b"bits"), ("n_heads", 0, -1, b"heads"), ("k_codes", None, -1, b"null"), ("v_scale", None, -1, b"null"), ("k_scale", 260, -1, b"16-byte")])
def test_c_entries_check_the_cache(field, value, rc, word):
    lib = _cabi.lib()
    cache, batch, t = good()
    setattr(cache, field, value)
    assert lib.varq_paged_append(cache, t, t, 256, 4, 1e-12, None) == rc and word in lib.varq_last_error()
    assert lib.varq_paged_read(cache, 256, 4, t, t, None) == rc and word in lib.varq_last_error()
    assert lib.varq_paged_attn(cache, batch, t, t, None, None, 0, None) == rc and word in lib.varq_last_error()


@pytest.mark.parametrize("field,value,rc,word", [
    ("n_seqs", -1, -1, b"negative"), ("n_queries", -1, -1, b"negative"), ("max_q", -1, -1, b"negative"), ("q_heads", 3, -1, b"heads"), ("q_heads", 0, -1, b"heads"),
    ("window", -1, -1, b"window"), ("sinks", 4, -1, b"window"), ("softmax_scale", 0.0, -1, b"softmax_scale"), ("softmax_scale", float("nan"), -1, b"softmax_scale"),
    ("n_seqs", 70000, -2, b"sequences"), ("n_queries", 1 << 31, -2, b"query tokens"), ("q_starts", None, -1, b"null"), ("kv_lens", 258, -1, b"misaligned"),
    ("block_table", None, -1, b"null")])
def test_attention_checks_the_batch(field, value, rc, word):
    lib = _cabi.lib()
    cache, batch, t = good()
    setattr(batch, field, value)
    assert lib.varq_paged_attn(cache, batch, t, t, None, None, 0, None) == rc and word in lib.varq_last_error()


def test_more_refusals_and_empty_calls():
    lib = _cabi.lib()
    cache, batch, t = good()
    assert lib.varq_paged_append(cache, t, t, 256, 0, 1e-12, None) == 0
    assert lib.varq_paged_read(cache, 256, 0, t, t, None) == 0
    assert lib.varq_paged_append(cache, t, t, 256, -1, 1e-12, None) == -1
    assert lib.varq_paged_append(cache, t, t, 256, 1 << 30, 1e-12, None) == -2
    assert lib.varq_paged_append(cache, t, t, 256, 1, 0.0, None) == -1 and b"eps" in lib.varq_last_error()
    assert lib.varq_paged_append(cache, t, _cabi.Tensor(256, _cabi.F32, 0, 0, 128, 64), 256, 1, 1e-12, None) == -1
    assert lib.varq_paged_append(cache, t, t, None, 1, 1e-12, None) == -1
    assert lib.varq_paged_append(cache, t, t, 260, 1, 1e-12, None) == -1 and b"misaligned" in lib.varq_last_error()
    assert lib.varq_paged_append(None, t, t, 256, 1, 1e-12, None) == -1
    f32 = _cabi.Tensor(256, _cabi.F32, 0, 0, 128, 64)
    assert lib.varq_paged_attn(cache, batch, f32, f32, None, None, 0, None) == -2 and b"fp16 or bf16" in lib.varq_last_error()
    batch.causal, batch.window = 0, 5
    assert lib.varq_paged_attn(cache, batch, t, t, None, None, 0, None) == -1 and b"causal" in lib.varq_last_error()
    for field in ("n_seqs", "n_queries", "max_q"):
        cache, batch, t = good()
        setattr(batch, field, 0)
        assert lib.varq_paged_attn(cache, batch, t, t, None, None, 0, None) == 0
