"""Attention over a paged cache against the formula in 64 bits, on the values that the cache stands for.

Tolerances, from the arithmetic that the operator promises (scores, sums and outputs in fp32, weights rounded to fp16 once, one rounding of the
output): with A = sum_j p_j |v_j| the weights' rounding moves an element by at most 2^-11 A, and as much again covers what scores in fp32 (at
most a few hundred in magnitude, each off by some 2^-22 of it) do to the weights; weights below fp16's normal range, relative to the largest
weight times V scale, carry 2^-25 of that instead, n of them 2^-25 n max|v|; the output's own rounding is 2^-11 (fp16) or 2^-8 (bf16) of it.
The log-sum-exp is fp32: 2^-16 absolute for scores of that size, and 2^-20 of its own."""
import math

import pytest
import torch

from VAR_Q import _cabi
from VAR_Q.paged import PagedCache

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Batch:
    """Sequences in pages in random order.  What is not written holds NaN scales, the table ends in -1, and one page more than needed is unused."""

    def __init__(self, kv, heads, D, kb=8, vb=8, page=16, seed=0, v_gain=None, dtype=torch.float32):
        g = torch.Generator().manual_seed(seed)
        self.kv, self.page = kv, page
        need = [-(-n // page) for n in kv]
        self.cache = PagedCache(sum(need) + 1, page, heads, D, kb, vb)
        self.cache.k_scale.fill_(math.nan)
        self.cache.v_scale.fill_(math.nan)
        self.cache.k_codes.random_()
        self.cache.v_codes.random_()
        order = torch.randperm(sum(need) + 1, generator=g).tolist()
        self.table = torch.full((len(kv), max(need + [0]) + 1), -1, dtype=torch.int32)
        self.slots = []
        for b, n in enumerate(kv):
            pages = [order.pop() for _ in range(need[b])]
            self.table[b, :need[b]] = torch.tensor(pages, dtype=torch.int32)
            self.slots.append(torch.tensor([pages[i // page] * page + i % page for i in range(n)], dtype=torch.int64))
            if n:
                k, v = (torch.randn((n, heads, D), generator=g) for _ in range(2))
                k[..., 3] *= 6.0
                if v_gain is not None:
                    v *= v_gain(torch.arange(n)).view(-1, 1, 1)
                self.cache.append(k.to(dtype).to(DEV), v.to(dtype).to(DEV), self.slots[b].to(DEV))
        self.kv_dev = torch.tensor(kv, dtype=torch.int32, device=DEV)

    def attend(self, q, counts, scale, **kw):
        starts = torch.tensor([sum(counts[:b]) for b in range(len(counts) + 1)], dtype=torch.int32, device=DEV)
        kw = {"max_q": max(counts), "max_kv": max(self.kv), **kw}
        return self.cache.attend(q, self.table.to(DEV), self.kv_dev, starts, kw.pop("max_q"), kw.pop("max_kv"), scale, return_lse=True, **kw)

    def reference(self, q, counts, scale, causal=True, window=None, sinks=0):
        """out, lse, A = sum p |v| and max |v| per element, in float64"""
        G = q.shape[1] // self.cache.num_heads
        D = q.shape[2]
        out, bound, top = (torch.zeros(q.shape, dtype=torch.float64, device=DEV) for _ in range(3))
        lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
        at = 0
        for b, (n, c) in enumerate(zip(self.kv, counts)):
            if n and c:
                k, v = (t.double() for t in self.cache.read(self.slots[b].to(DEV)))
                qd = q[at:at + c].double().view(c, -1, G, D)
                s = torch.einsum("ihgd,jhd->ihgj", qd, k) * scale
                i, j = torch.arange(n - c, n, device=DEV).view(-1, 1), torch.arange(n, device=DEV)
                see = torch.ones((c, n), dtype=torch.bool, device=DEV)
                if causal:
                    see = j <= i
                    if window:
                        see = see & ((i - j < window) | (j < sinks))
                s = s.masked_fill(~see.view(c, 1, 1, n), -math.inf)
                p = torch.nan_to_num(torch.softmax(s, -1))                # a row that sees nothing
                v = torch.where(see.any(0).view(-1, 1, 1), v, 0.0)
                out[at:at + c] = torch.einsum("ihgj,jhd->ihgd", p, v).reshape(c, -1, D)
                bound[at:at + c] = torch.einsum("ihgj,jhd->ihgd", p, v.abs()).reshape(c, -1, D)
                top[at:at + c] = v.abs().amax((0, 2)).repeat_interleave(G).view(1, -1, 1)
                lse[at:at + c] = torch.logsumexp(s, -1).reshape(c, -1)
            at += c
        return out, lse, bound, top

    def check(self, q, counts, scale=None, out=None, **kw):
        scale = scale or 1.0 / math.sqrt(q.shape[2])
        got, lse = out or self.attend(q, counts, scale, **kw)
        kw.pop("max_kv", None); kw.pop("max_q", None)
        ref, ref_lse, bound, top = self.reference(q, counts, scale, **kw)
        unit = 2.0 ** -11 if q.dtype == torch.float16 else 2.0 ** -8
        tol = 2.0 ** -10 * bound + 2.0 ** -25 * max(self.kv) * top + unit * ref.abs() * 1.01 + 1e-7
        # results beyond the type's range are infinite
        beyond = ref.abs() * (1 + 2.0 ** -9) >= torch.finfo(q.dtype).max
        assert (got[beyond].double().abs() >= 0.99 * torch.finfo(q.dtype).max).all() and (got[beyond].sign().double() == ref[beyond].sign()).all()
        worst = ((got.double() - ref).abs() / tol)[~beyond].max().item()
        assert got.shape == q.shape and got.dtype == q.dtype and worst <= 1.0, f"{worst:.3f} of the bound"
        seen = torch.isfinite(ref_lse)
        assert torch.equal(seen, torch.isfinite(lse)) and (lse[~seen] == -math.inf).all() and (got[~seen] == 0).all()
        if seen.any():
            assert ((lse - ref_lse).abs()[seen] <= 2.0 ** -16 + 2.0 ** -20 * ref_lse.abs()[seen]).all(), (lse - ref_lse).abs()[seen].max().item()
        assert _cabi.device_status() == 0
        return got, lse


def queries(tokens, heads, D, dtype=torch.float16, seed=1, gain=1.0):
    return (torch.randn((tokens, heads, D), generator=torch.Generator().manual_seed(seed)) * gain).to(dtype).to(DEV)


BITS = [(8, 8), (4, 4), (2, 2), (8, 4), (4, 2), (2, 8)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kb,vb", BITS)
@pytest.mark.parametrize("G", [1, 5])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_single_tokens(D, kb, vb, G, dtype):
    kv = [1, 2, 15, 16, 17, 300, 1025]
    b = Batch(kv, 3, D, kb, vb, page=16, seed=D + kb)
    b.check(queries(len(kv), 3 * G, D, dtype), [1] * len(kv))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kb,vb", BITS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_ragged_chunks(D, kb, vb, causal, dtype):
    """chunks of every kind in one batch: nothing, one token, whole prompts, more queries than a tile holds, behind a long context"""
    kv, counts = [5, 130, 257, 700, 33, 64, 128, 0], [0, 130, 1, 300, 33, 17, 127, 0]
    b = Batch(kv, 2, D, kb, vb, page=32, seed=D + vb)
    b.check(queries(sum(counts), 4, D, dtype), counts, causal=causal)


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257])
@pytest.mark.parametrize("G", [1, 3])
def test_lengths_around_the_tiles(n, G):
    """prompts without and with a little context in front"""
    for before in (0, 1, 63, 127, 130):
        b = Batch([before + n, n], 1, 64, page=16, seed=n)
        b.check(queries(2 * n, G, 64), [n, n])


@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [4, 2, 1, 3], [40, 7, 100, 129], [300, 200, 1, 150]])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 3), (16, 4), (100, 0), (129, 16), (130, 200), (5000, 7)])
def test_windows_and_first_tokens(counts, window, sinks):
    b = Batch([700, 203, 111, 1030], 2, 64, 8, 4, page=16, seed=window)
    b.check(queries(sum(counts), 6, 64), [min(c, n) for c, n in zip(counts, b.kv)] if counts[2] <= 111 else [300, 200, 1, 150], window=window, sinks=sinks)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("D", [64, 128])
def test_page_sizes(page, D):
    b = Batch([1500, 129, 1], 2, D, 4, 8, page=page, seed=page)
    b.check(queries(3, 8, D), [1, 1, 1])
    b.check(queries(205, 4, D), [140, 64, 1])
    b.check(queries(205, 4, D), [140, 64, 1], window=70, sinks=2)


@pytest.mark.parametrize("G", [1, 2, 4, 7, 8, 12, 16, 17, 64])
@pytest.mark.parametrize("c", [1, 2, 5])
def test_query_heads_per_head(G, c):
    b = Batch([333, 90], 2, 64, page=32, seed=G)
    b.check(queries(2 * c, 2 * G, 64, torch.bfloat16), [c, c])


def test_more_queries_than_cached_tokens():
    """the first queries stand in front of the sequence and see nothing"""
    b = Batch([3, 0, 100], 2, 64, seed=4)
    b.check(queries(170, 4, 64), [10, 20, 140])
    b.check(queries(15, 4, 64), [5, 4, 6])
    b.check(queries(170, 4, 64), [10, 20, 140], window=7, sinks=2)


def test_empty_batches():
    b = Batch([0, 0], 2, 64)
    b.check(queries(3, 2, 64), [1, 2])
    b.check(queries(3, 2, 64), [1, 2], causal=False)
    out, lse = b.attend(queries(0, 2, 64), [0, 0], 0.125)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)
    none = torch.empty((0, 3), dtype=torch.int32, device=DEV)
    out = b.cache.attend(queries(0, 2, 64), none, none[:, 0], torch.zeros(1, dtype=torch.int32, device=DEV), 0, 0, 0.125)
    assert out.shape == (0, 2, 64)


@pytest.mark.parametrize("c", [1, 3, 40, 200])
@pytest.mark.parametrize("D", [64, 128])
def test_long_contexts_are_split(c, D):
    """one sequence, one head: the keys are all there is to share out"""
    b = Batch([20011], 1, D, 8, 8, page=64, seed=c)
    b.check(queries(c, 2, D, torch.bfloat16), [c])
    b.check(queries(c, 2, D, torch.bfloat16), [c], window=4099, sinks=20)


@pytest.mark.parametrize("c", [1, 150])
@pytest.mark.parametrize("max_kv", [1, 100, 1 << 20])
def test_the_longest_length_is_a_hint(c, max_kv):
    b = Batch([3000, 555], 1, 64, page=64, seed=c)
    b.check(queries(2 * c, 2, 64), [c, c], max_kv=max_kv)


@pytest.mark.parametrize("c", [1, 2, 20, 100])
def test_no_nan_or_infinity_comes_out_of_what_is_not_seen(c):
    """masked keys that hold NaN: behind the diagonal, in front of the window"""
    n, page = 400, 16
    b = Batch([n], 2, 64, page=page, seed=9)
    q = queries(c, 4, 64)
    window, sinks = 50, 3
    clean = b.attend(q, [c], 0.125, window=window, sinks=sinks)
    first = n - c - window + 1                                         # first key that the first query's window holds
    hidden = b.slots[0][sinks:first].to(DEV)
    bad = torch.full((len(hidden), 2, 64), math.nan, device=DEV)
    bad[::2] = math.inf
    b.cache.append(bad, bad, hidden)
    after = b.attend(q, [c], 0.125, window=window, sinks=sinks)
    assert torch.equal(clean[0], after[0]) and torch.equal(clean[1], after[1])
    # the last token's row is NaN: only the last query sees it
    last = b.slots[0][-1:].to(DEV)
    b.cache.append(bad[:1], bad[:1], last)
    out, lse = b.attend(q, [c], 0.125, window=window, sinks=sinks)
    assert torch.equal(out[:-1], clean[0][:-1]) and torch.equal(lse[:-1], clean[1][:-1])
    assert torch.isnan(out[-1]).all()
    # a NaN in V alone
    fine, nan = torch.ones((1, 2, 64), device=DEV), bad[:1]
    b.cache.append(fine, nan, last)
    out, lse = b.attend(q, [c], 0.125, window=window, sinks=sinks)
    assert torch.equal(out[:-1], clean[0][:-1]) and torch.isnan(out[-1]).all()


@pytest.mark.parametrize("c", [1, 100])
def test_one_query_that_is_not_finite_spoils_its_own_row_only(c):
    b = Batch([200, 300], 2, 64, seed=2)
    q = queries(2 * c, 4, 64)
    clean = b.attend(q, [c, c], 0.125)[0]
    q[c - 1, 1, 5] = math.nan
    out = b.attend(q, [c, c], 0.125)[0]
    assert torch.isnan(out[c - 1, 1]).all()
    out[c - 1, 1] = clean[c - 1, 1]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("c", [1, 130])
@pytest.mark.parametrize("gain", [
    lambda j: torch.where(j % 7 == 0, 1000.0, 1e-3), lambda j: torch.where(j < 4, 1e-4, 1.0), lambda j: 2.0 ** (j % 40 - 20).float(),
    lambda j: torch.where(j == 100, 0.0, 1.0), lambda j: torch.zeros_like(j, dtype=torch.float32)])
def test_values_of_very_different_size(c, gain):
    """V scales that differ by many orders of magnitude, heavy keys with small values, values that are zero"""
    b = Batch([260, 131], 1, 64, page=32, seed=3, v_gain=gain)
    b.check(queries(2 * c, 2, 64, gain=3.0), [c, c])


@pytest.mark.parametrize("c", [1, 130])
@pytest.mark.parametrize("gain", [1e-6, 0.0, 30.0, 300.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_queries_of_very_different_size(c, gain, dtype):
    """scores from nothing to a few hundred: all weights alike, or one that is nearly everything"""
    b = Batch([300, 150], 1, 128, page=32, seed=5)
    q = queries(2 * c, 2, 128, dtype, gain=gain)
    b.check(q, [c, c], scale=(1.0 if gain < 300 else 0.1) / math.sqrt(128))


def test_growing_scores_move_the_reference():
    """keys that answer more and more loudly: the running maximum has to follow at every tile"""
    n, D = 1500, 64
    b = Batch([n], 1, D, page=64, seed=6)
    q = queries(140, 2, D)
    base = q[0, 0].float()
    k = torch.arange(n, device=DEV).view(-1, 1, 1) / n * 8.0 * base.view(1, 1, D)
    b.cache.append(k, torch.randn((n, 1, D), device=DEV), b.slots[0].to(DEV))
    same = base.half().expand(140, 2, D).contiguous()
    b.check(same, [140], scale=0.1)
    b.check(same[:1], [1], scale=0.1)
    b.check(same, [140], scale=0.1, causal=False)


@pytest.mark.parametrize("c", [1, 150])
def test_strides(c):
    """queries as views: of a fused activation, heads before tokens; a block table cut out of a wider one"""
    b = Batch([333, 222], 2, 64, page=16, seed=7)
    T, H, D = 2 * c, 4, 64
    fused = queries(T, 3 * H, D)
    starts = torch.tensor([0, c, 2 * c], dtype=torch.int32, device=DEV)
    wide = torch.full((2, b.table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    wide[:, 2:2 + b.table.shape[1]] = b.table.to(DEV)
    for q in (fused[:, H:2 * H], queries(H, T, D).transpose(0, 1), queries(T, H, 2 * D)[..., 1:1 + D], queries(T, 2 * H, D)[:, ::2]):
        out = b.cache.attend(q, wide[:, 2:2 + b.table.shape[1]], b.kv_dev, starts, c, 333, 0.125, return_lse=True)
        b.check(q, [c, c], scale=0.125, out=out)
        assert out[0].is_contiguous()


@pytest.mark.parametrize("c", [1, 6, 40, 260])
def test_the_same_call_gives_the_same_bits(c):
    b = Batch([5000, 700], 2, 128, page=64, seed=8)
    q = queries(2 * c, 6, 128, torch.bfloat16)
    first = b.attend(q, [c, c], 0.09)
    for _ in range(3):
        again = b.attend(q, [c, c], 0.09)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_parts_of_a_context_merge_by_their_log_sums():
    """attention over disjoint parts, each a sequence of its own, joined by the log-sum-exp"""
    b = Batch([500, 300], 2, 64, page=16, seed=10)
    q = queries(4, 4, 64, torch.float16)
    both = torch.cat([q, q])
    out, lse = b.check(both, [4, 4], causal=False)
    w = torch.softmax(torch.stack([lse[:4], lse[4:]]), 0).unsqueeze(-1)
    joined = w[0] * out[:4].float() + w[1] * out[4:].float()
    pages = torch.cat([b.table[0, :32][b.table[0, :32] >= 0], b.table[1, :20][b.table[1, :20] >= 0]])
    k, v = (torch.cat([b.cache.read(s.to(DEV))[i] for s in b.slots]).double() for i in (0, 1))
    s = torch.einsum("ihgd,jhd->ihgj", q.double().view(4, 2, 2, 64), k) * 0.125
    ref = torch.einsum("ihgj,jhd->ihgd", torch.softmax(s, -1), v).reshape(4, 4, 64)
    assert len(pages) == 32 + 19
    assert (joined.double() - ref).abs().max().item() <= 2.0 ** -9 * v.abs().max().item()


def test_chunk_by_chunk_is_the_whole_prompt():
    """a prompt in one call, and the same in chunks and single tokens as the cache grows: a row's own result does not hang on the split"""
    n, D = 300, 64
    b = Batch([n], 2, D, 8, 8, page=16, seed=11)
    q = queries(n, 4, D)
    whole = b.check(q, [n])[0]
    at = 0
    for c in (100, 1, 1, 17, 130, 1, 50):
        at += c
        lens = torch.tensor([at], dtype=torch.int32, device=DEV)
        starts = torch.tensor([0, c], dtype=torch.int32, device=DEV)
        out = b.cache.attend(q[at - c:at], b.table.to(DEV), lens, starts, c, at, 0.125)
        assert (out.double() - whole[at - c:at].double()).abs().max().item() <= 2.0 ** -8 * 4.0     # twice the bound of |v| < 4 for each side
    assert at == n


@pytest.mark.parametrize("c", [1, 100])
def test_another_stream_and_a_graph(c):
    b = Batch([900, 400], 2, 64, page=32, seed=12)
    q = queries(2 * c, 4, 64)
    ref = b.attend(q, [c, c], 0.125)
    side = torch.cuda.Stream()
    table, starts = b.table.to(DEV), torch.tensor([0, c, 2 * c], dtype=torch.int32, device=DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = b.cache.attend(q, table, b.kv_dev, starts, c, 900, 0.125, return_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b.cache.attend(q, table, b.kv_dev, starts, c, 900, 0.125, return_lse=True)
    # new lengths and queries under the same graph
    b.kv, b.slots = [850, 380], [b.slots[0][:850], b.slots[1][:380]]
    b.kv_dev.copy_(torch.tensor(b.kv, dtype=torch.int32))
    q.copy_(queries(2 * c, 4, 64, seed=77))
    graph.replay()
    torch.cuda.synchronize()
    b.check(q, [c, c], scale=0.125, out=(out[0], out[1]))


def test_pools_of_more_than_two_to_the_31_words():
    page, H, D, n = 64, 8, 128, 500
    pages = 2 ** 31 // (H * page * D // 4) + 8
    cache = PagedCache(pages, page, H, D, 8, 8)
    b = Batch([n], H, D, page=page, seed=13)
    table = torch.tensor([[pages - 1 - i for i in range(8)]], dtype=torch.int32, device=DEV)
    new = torch.cat([table[0].long() * page + i for i in range(1)]).view(-1, 1) + torch.arange(page, device=DEV)
    k, v = b.cache.read(b.slots[0].to(DEV))
    cache.append(k, v, new.flatten()[:n])
    for c in (1, 3, 200):
        q = queries(c, 16, D, torch.bfloat16)
        starts = torch.tensor([0, c], dtype=torch.int32, device=DEV)
        b.check(q, [c], out=cache.attend(q, table, b.kv_dev, starts, c, n, 1.0 / math.sqrt(D), return_lse=True))


@pytest.mark.parametrize("c", [1, 100])
def test_numbers_outside_their_bounds_are_clamped_and_reported(c):
    """What only the device sees: the access stays inside the tensors, and a code is left"""
    b = Batch([100, 200], 1, 64, page=16, seed=14)
    q, table = queries(2 * c, 2, 64), b.table.to(DEV)
    starts = torch.tensor([0, c, 2 * c], dtype=torch.int32, device=DEV)
    args = lambda **k: {"table": table, "lens": b.kv_dev, "starts": starts, **k}  # noqa: E731
    wrong = table.clone()
    wrong[0, 1] = 1 << 20
    for kind, code in ((args(table=wrong), 66), (args(lens=torch.tensor([100, 1 << 30], dtype=torch.int32, device=DEV)), 65),
                       (args(lens=torch.tensor([-5, 200], dtype=torch.int32, device=DEV)), 65),
                       (args(starts=torch.tensor([0, c, 1000 + c], dtype=torch.int32, device=DEV)), 64)):
        # pages behind the sequence are not there: for lengths that reach them the table holds pages that exist
        kind["table"] = torch.where(kind["table"] < 0, 0, kind["table"])
        b.cache.attend(q, kind["table"], kind["lens"], kind["starts"], c, 200, 0.125)
        assert _cabi.device_status() == code
    assert _cabi.device_status() == 0


def test_refusals():
    b = Batch([50], 2, 64, seed=15)
    q, table, starts = queries(1, 4, 64), b.table.to(DEV), torch.tensor([0, 1], dtype=torch.int32, device=DEV)

    def go(q=q, table=table, lens=b.kv_dev, starts=starts, max_q=1, max_kv=50, scale=0.125, **kw):
        return b.cache.attend(q, table, lens, starts, max_q, max_kv, scale, **kw)

    go()
    for bad, word in ((dict(q=q.float()), "float16"), (dict(q=q[..., :32]), "head_dim"), (dict(q=queries(1, 3, 64)), "heads"), (dict(q=q[0]), "tokens"),
                      (dict(q=queries(1, 4, 128)[..., ::2]), "contiguous"), (dict(table=table.long()), "block_table"), (dict(table=table[0]), "block_table"),
                      (dict(table=torch.zeros((1, 10), dtype=torch.int32, device=DEV)[:, ::2]), "block_table"), (dict(lens=b.kv_dev.long()), "kv_lens"), (dict(starts=starts[:1]), "q_starts"),
                      (dict(max_q=-1), "max_q"), (dict(max_kv=1 << 40), "max_kv"), (dict(scale=0.0), "softmax_scale"), (dict(scale=math.inf), "softmax_scale"),
                      (dict(window=0), "window"), (dict(window=-3), "window"), (dict(window=4, causal=False), "causal"), (dict(sinks=2), "sinks"),
                      (dict(sinks=-1, window=3), "sinks")):
        with pytest.raises(ValueError, match=word):
            go(**bad)
    with pytest.raises(RuntimeError, match="CUDA"):
        go(q=q.cpu())
    with pytest.raises(RuntimeError, match="CUDA"):
        go(lens=b.kv_dev.cpu())
    assert _cabi.device_status() == 0
