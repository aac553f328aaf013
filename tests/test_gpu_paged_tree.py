"""Trees of drafted tokens: masks and positions against a walk on the host, attention against the formula in 64 bits, on both kernels.
Tolerances as in test_gpu_paged_attention.py, where they are derived: a tree changes which keys are seen, not the arithmetic."""
import math
import random

import pytest
import torch

from test_gpu_paged_attention import BITS, DEV, Batch, queries
from VAR_Q import _cabi
from VAR_Q.paged import PagedCache, draft_tree

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[None, "tc", "decode"])
def path(request):
    _cabi.force_attn_path(request.param)
    yield request.param
    _cabi.force_attn_path(None)


def some_tree(n, seed, wide=6):
    rng = random.Random(seed)
    return [-1 if i == 0 or rng.random() < 0.1 else rng.randint(max(0, i - wide), i - 1) for i in range(n)]


def ancestors(parents):
    """[n, n] truth values: what each token sees of the others"""
    see = torch.zeros((len(parents), len(parents)), dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            see[i] = see[p]
        see[i, i] = True
    return see


def pack(see, words):
    """truth values [n, m] -> int32 [n, words]"""
    bits = torch.zeros((see.shape[0], words * 32), dtype=torch.int64)
    bits[:, :see.shape[1]] = see
    packed = (bits.view(see.shape[0], words, 32) << torch.arange(32)).sum(-1)
    return torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).to(torch.int32)


class Trees(Batch):
    def reference(self, q, counts, scale, tree=None, see=None, window=None, sinks=0, causal=True):
        G, D = q.shape[1] // self.cache.num_heads, q.shape[2]
        out, bound, top = (torch.zeros(q.shape, dtype=torch.float64, device=DEV) for _ in range(3))
        lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
        at = 0
        for b, (n, c) in enumerate(zip(self.kv, counts)):
            if n and c:
                k, v = (t.double() for t in self.cache.read(self.slots[b].to(DEV)))
                seen = torch.zeros((c, n), dtype=torch.bool)
                for i in range(c):
                    last = n - c + int(see[b][i].sum()) - 1
                    for j in range(n):
                        if j < n - c:
                            seen[i, j] = not window or last - j < window or j < sinks
                        else:
                            seen[i, j] = bool(see[b][i, j - (n - c)])
                seen = seen.to(DEV)
                qd = q[at:at + c].double().view(c, -1, G, D)
                s = (torch.einsum("ihgd,jhd->ihgj", qd, k) * scale).masked_fill(~seen.view(c, 1, 1, n), -math.inf)
                p = torch.nan_to_num(torch.softmax(s, -1))
                v = torch.where(seen.any(0).view(-1, 1, 1), v, 0.0)
                out[at:at + c] = torch.einsum("ihgj,jhd->ihgd", p, v).reshape(c, -1, D)
                bound[at:at + c] = torch.einsum("ihgj,jhd->ihgd", p, v.abs()).reshape(c, -1, D)
                top[at:at + c] = v.abs().amax((0, 2)).repeat_interleave(G).view(1, -1, 1)
                lse[at:at + c] = torch.logsumexp(s, -1).reshape(c, -1)
            at += c
        return out, lse, bound, top

    def attend(self, q, counts, scale, see=None, **kw):
        return super().attend(q, counts, scale, **kw)

    def run(self, counts, G, D, dtype=torch.float16, trees=None, see=None, words=None, **kw):
        see = see or [ancestors(t) for t in (trees or [some_tree(c, 7 * i + c) for i, c in enumerate(counts)])]
        words = words or max(1, -(-max(counts) // 32))
        tree = torch.cat([pack(s, words) for s in see]).to(DEV)
        q = queries(sum(counts), self.cache.num_heads * G, D, dtype)
        return self.check(q, counts, tree=tree, see=see, **kw)


# ------------------------------------------------------------------------------------------------ masks and positions
@pytest.mark.parametrize("counts", [[1], [5, 1, 0, 33], [32, 64, 31], [100, 3], [257]])
def test_masks_and_positions(counts):
    trees = [some_tree(c, c + i) for i, c in enumerate(counts)]
    trees[0] = list(range(-1, counts[0] - 1))                                # a chain
    lens = [c + 11 * i for i, c in enumerate(counts)]
    ints = dict(dtype=torch.int32, device=DEV)
    starts = torch.tensor([sum(counts[:b]) for b in range(len(counts) + 1)], **ints)
    for most in (max(counts), max(counts) + 40):                             # a loose bound
        masks, positions = draft_tree(torch.tensor(sum(trees, []), **ints), torch.tensor(lens, **ints), starts, most)
        words = -(-min(most, sum(counts)) // 32)
        assert masks.shape == (sum(counts), words) and masks.dtype == positions.dtype == torch.int32
        assert torch.equal(masks.cpu(), torch.cat([pack(ancestors(t), words) for t in trees]))
        assert positions.tolist() == [n - c + d for n, c, t in zip(lens, counts, trees) for d in (ancestors(t).sum(1) - 1).tolist()]
    assert _cabi.device_status() == 0


def test_masks_of_padded_and_bad_batches():
    ints = dict(dtype=torch.int32, device=DEV)
    parents = torch.tensor([9, 9, -1, 0, 1, -1, 9], **ints)
    held = torch.full((1 << 16,), 7, **ints)                                # what the allocator hands out next is no zeros
    del held
    masks, positions = draft_tree(parents, torch.tensor([13, 5], **ints), torch.tensor([2, 5, 6], **ints), 3)
    assert masks.flatten().tolist() == [0, 0, 1, 3, 7, 1, 0] and positions.tolist() == [0, 0, 10, 11, 12, 4, 0] and _cabi.device_status() == 0
    masks, _ = draft_tree(parents, torch.tensor([13], **ints), torch.tensor([0, 3], **ints), 3)      # parents that come later, or that are none
    assert masks.flatten().tolist()[:3] == [1, 2, 4] and _cabi.device_status() == 67
    masks, _ = draft_tree(torch.tensor([-5, 0], **ints), torch.tensor([13], **ints), torch.tensor([0, 2], **ints), 2)
    assert masks.flatten().tolist() == [1, 3] and _cabi.device_status() == 67
    draft_tree(torch.zeros(40, **ints) - 1, torch.tensor([50], **ints), torch.tensor([0, 40], **ints), 8)      # more tokens than the bound says
    assert _cabi.device_status() == 64
    masks, positions = draft_tree(parents[:0], torch.zeros(0, **ints), torch.zeros(1, **ints), 0)
    assert masks.shape == (0, 0) and positions.shape == (0,)
    masks, positions = draft_tree(parents, torch.zeros(0, **ints), torch.zeros(1, **ints), 5)       # rows, and no sequence
    assert (masks == 0).all() and (positions == 0).all() and _cabi.device_status() == 0


# ------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kb,vb", BITS)
@pytest.mark.parametrize("counts,G", [([1, 7, 16], 1), ([26, 3, 1], 5), ([64, 40, 5], 4)])
def test_types_and_rows(D, kb, vb, counts, G, path):
    b = Trees([300, 61, 17], 2, D, kb, vb, page=16, seed=D + kb + G)
    b.run(counts, G, D, torch.bfloat16 if G == 4 else torch.float16)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ctx", [0, 1, 15, 16, 17, 63, 64, 65, 127, 1000])
def test_contexts_and_tiles(D, ctx, path):
    """the first drafted token anywhere in a tile"""
    counts = [33, 1, 20]
    b = Trees([ctx + c for c in counts], 2, D, page=32, seed=ctx)
    b.run(counts, 2, D)


@pytest.mark.parametrize("n", [31, 32, 33, 63, 64, 65, 96, 130, 300])
def test_sizes_of_trees(n, path):
    b = Trees([n + 50, n], 1, 64, page=64, seed=n)
    b.run([n, n], 1, 64)
    b.run([n, n], 1, 64, words=-(-n // 32) + 2)                             # rows of more words than needed


@pytest.mark.parametrize("D", [64, 128])
def test_a_chain_is_causal(D, path):
    counts, G = [40, 7, 1], 3
    b = Trees([500, 90, 33], 2, D, page=16, seed=3)
    q = queries(sum(counts), 2 * G, D)
    tree = torch.cat([pack(ancestors(list(range(-1, c - 1))), 2) for c in counts]).to(DEV)
    for kw in ({}, {"window": 64, "sinks": 4}):
        one = Batch.attend(b, q, counts, D ** -0.5, tree=tree, **kw)
        two = Batch.attend(b, q, counts, D ** -0.5, **kw)
        assert ((one[0].double() - two[0].double()).norm() / two[0].double().norm()).item() <= 2.0 ** -9
        assert torch.allclose(one[1], two[1], atol=2.0 ** -15, rtol=0)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(40, 0), (64, 4), (200, 17), (2 ** 31 - 1, 0), (100, 2 ** 31 - 1)])
def test_windows(D, window, sinks, path):
    counts = [26, 1, 40, 9]
    b = Trees([700, 300, 45, 130], 2, D, 8, 4, page=16, seed=window % 1000)
    b.run(counts, 3, D, window=window, sinks=sinks)


def test_evicted_pages(path):
    """pages in front of all windows may be gone"""
    counts, page, window = [20, 5], 16, 48
    b = Trees([600, 400], 2, 128, page=page, seed=5)
    trees = [some_tree(c, c) for c in counts]
    ref = b.run(counts, 2, 128, trees=trees, window=window)
    for i, (n, c) in enumerate(zip(b.kv, counts)):
        b.table[i, :(n - c - window) // page] = -1
    assert all(torch.equal(x, y) for x, y in zip(ref, b.run(counts, 2, 128, trees=trees, window=window)))


def test_rows_that_see_nothing(path):
    """masks need not come from parents: rows of no bit, without a context"""
    b = Trees([12, 12 + 30], 2, 64, seed=1)
    see = [torch.rand((12, 12), generator=torch.Generator().manual_seed(s)) < 0.3 for s in (1, 2)]
    see[0][3] = see[0][11] = see[1][0] = False
    out, lse = b.run([12, 12], 2, 64, see=see)
    assert (out[[3, 11]] == 0).all() and (lse[[3, 11]] == -math.inf).all() and torch.isfinite(lse[12]).all()


def test_what_is_not_seen_may_hold_anything(path):
    """NaN in a drafted token reaches its descendants only"""
    parents = [-1, 0, 0, 1, 2, 2]
    b = Trees([206], 2, 128, page=16, seed=2)
    ref, _ = b.run([6], 1, 128, trees=[parents])
    for scale in (b.cache.k_scale, b.cache.v_scale):
        at = b.slots[0][200 + 2].item()
        kept = scale[at // 16, :, at % 16].clone()
        scale[at // 16, :, at % 16] = math.nan
        q = queries(6, 2, 128)
        out, lse = b.attend(q, [6], 128 ** -0.5, tree=pack(ancestors(parents), 1).to(DEV))
        assert torch.isnan(out[[2, 4, 5]]).all() and torch.equal(out[[0, 1, 3]], ref[[0, 1, 3]])
        scale[at // 16, :, at % 16] = kept


@pytest.mark.parametrize("kv,counts,heads,G", [([20000], [16], 1, 4), ([9000, 100], [64, 2], 2, 4), ([5000] * 20, [26] * 20, 2, 1), ([3000], [100], 1, 8)])
def test_parts_of_the_key_range(kv, counts, heads, G, path):
    b = Trees(kv, heads, 128, 4, 4, page=64, seed=len(kv))
    q = queries(sum(counts), heads * G, 128)
    trees = [some_tree(c, i) for i, c in enumerate(counts)]
    words = -(-max(counts) // 32)
    tree = torch.cat([pack(ancestors(t), words) for t in trees]).to(DEV)
    out, lse = b.attend(q, counts, 128 ** -0.5, tree=tree)
    # the same as the context and the tree on their own, merged: a reference of 20000 keys in a loop would take minutes
    at = 0
    for i, (n, c) in enumerate(zip(kv, counts)):
        k, v = (t.double() for t in b.cache.read(b.slots[i].to(DEV)))
        seen = torch.cat([torch.ones((c, n - c), dtype=torch.bool), ancestors(trees[i])], 1).to(DEV)
        s = torch.einsum("ihgd,jhd->ihgj", q[at:at + c].double().view(c, heads, G, 128), k) * 128 ** -0.5
        s = s.masked_fill(~seen.view(c, 1, 1, n), -math.inf)
        p = torch.softmax(s, -1)
        ref, bound = (torch.einsum("ihgj,jhd->ihgd", p, x).reshape(c, -1, 128) for x in (v, v.abs()))
        tol = 2.0 ** -10 * bound + 2.0 ** -25 * n * v.abs().max() + 2.0 ** -11 * ref.abs() * 1.01 + 1e-7
        assert ((out[at:at + c].double() - ref).abs() <= tol).all()
        ref_lse = torch.logsumexp(s, -1).reshape(c, -1)
        assert ((lse[at:at + c] - ref_lse).abs() <= 2.0 ** -16 + 2.0 ** -20 * ref_lse.abs()).all()
        at += c
    assert _cabi.device_status() == 0


@pytest.mark.parametrize("front,behind", [(0, 3), (5, 0), (70, 200)])
def test_padded_batches(front, behind, path):
    counts, G, D = [16, 3, 40], 2, 64
    b = Trees([316, 3, 90], 2, D, page=16, seed=1)
    n = sum(counts)
    see = [ancestors(some_tree(c, c)) for c in counts]
    tree = torch.cat([torch.full((front, 2), -1, dtype=torch.int32), torch.cat([pack(s, 2) for s in see]), torch.full((behind, 2), -1, dtype=torch.int32)]).to(DEV)
    q = queries(front + n + behind, 2 * G, D)
    starts = torch.tensor([front + sum(counts[:i]) for i in range(4)], dtype=torch.int32, device=DEV)
    held = torch.full((1 << 20,), math.nan, device=DEV)
    del held
    out, lse = b.cache.attend(q, b.table.to(DEV), b.kv_dev, starts, 40, 316, D ** -0.5, return_lse=True, tree=tree)
    b.check(q[front:front + n], counts, out=(out[front:front + n], lse[front:front + n]), see=see)
    for rows in (slice(0, front), slice(front + n, None)):
        assert (out[rows] == 0).all() and (lse[rows] == -math.inf).all()


def test_large_heads_of_a_group_and_strides(path):
    b = Trees([230, 40], 3, 128, 4, 8, page=32, seed=1)
    counts = [26, 4]
    see = [ancestors(some_tree(c, c)) for c in counts]
    tree = torch.cat([pack(s, 1) for s in see]).to(DEV)
    wide = queries(30, 24 + 6, 128, torch.bfloat16)
    q = wide[:, 3:27]                                                      # eight query heads to a head, a view
    b.check(q, counts, out=b.attend(q, counts, 128 ** -0.5, tree=tree), see=see)


def test_captured_and_replayed(path):
    counts, D = [16, 16], 128
    b = Trees([300, 200], 2, D, page=16, seed=1)
    parents = torch.tensor([-1, *range(15)] * 2, dtype=torch.int32, device=DEV)
    q, table = queries(32, 8, D), b.table.to(DEV)
    starts = torch.tensor([0, 16, 32], dtype=torch.int32, device=DEV)

    def call():
        masks, positions = draft_tree(parents, b.kv_dev, starts, 16)
        return masks, positions, b.cache.attend(q, table, b.kv_dev, starts, 16, 300, D ** -0.5, tree=masks)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for tree in ([-1, 0, 0, 1, 1, 2, 2, 3, 3, 4, 4, 5, 5, 6, 6, 7], [-1] * 16):
        parents.copy_(torch.tensor(tree * 2, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, call()))
    assert _cabi.device_status() == 0


@pytest.mark.parametrize("seqs,heads,counts,lens", [
    (24, 8, [0, 36, 1, 20], [0, 300, 300, 77, 1, 640]),                      # more blocks than multiprocessors, sequences ranked by length: equal ones, empty ones
    (32, 5, [5, 33], [64, 65, 400]), (33, 5, [5, 33], [64, 65, 400]),        # as many as are ranked, and more
])
def test_many_sequences_of_different_lengths(seqs, heads, counts, lens, path):
    """also as a padded batch, whose rows in front and behind are the first and the last sequence's"""
    D, counts = 64, [counts[i % len(counts)] for i in range(seqs)]
    kv = [lens[i % len(lens)] if counts[i] == 0 else lens[i % len(lens)] + counts[i] for i in range(seqs)]
    b = Trees(kv, heads, D, 4, 8, page=16, seed=seqs)
    see = [ancestors(some_tree(c, c + i)) for i, c in enumerate(counts)]
    n, front, behind = sum(counts), 3, 70
    tree = torch.cat([torch.full((front, 2), -1, dtype=torch.int32), *(pack(s, 2) for s in see), torch.full((behind, 2), -1, dtype=torch.int32)]).to(DEV)
    q = queries(front + n + behind, heads, D)
    got = b.check(q[front:front + n], counts, tree=tree[front:front + n], see=see)
    starts = torch.tensor([front + sum(counts[:i]) for i in range(seqs + 1)], dtype=torch.int32, device=DEV)
    out, lse = b.cache.attend(q, b.table.to(DEV), b.kv_dev, starts, max(counts), max(kv), D ** -0.5, return_lse=True, tree=tree)
    assert torch.equal(out[front:front + n], got[0]) and torch.equal(lse[front:front + n], got[1])
    for rows in (slice(0, front), slice(front + n, None)):
        assert (out[rows] == 0).all() and (lse[rows] == -math.inf).all()
    assert _cabi.device_status() == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kb", [8, 4, 2])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("pad,at", [(1, 1), (8, 0), (8, 3)])
def test_queries_at_any_address(D, kb, dtype, pad, at, path):
    counts = [26, 4]
    b = Trees([130, 40], 2, D, kb, 8, page=16, seed=kb)
    see = [ancestors(some_tree(c, c)) for c in counts]
    q = queries(30, 10, D + pad, dtype)[:, :, at:at + D]
    b.check(q, counts, out=b.attend(q, counts, D ** -0.5, tree=torch.cat([pack(s, 1) for s in see]).to(DEV)), see=see)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kb", [8, 4, 2])
@pytest.mark.parametrize("gain", [2.0 ** -40, 2.0 ** -8, 2.0 ** 9, 2.0 ** 30])
def test_queries_of_any_size(D, kb, gain, path):
    """bf16 queries beyond fp16's range, next to rows of zeros and ordinary ones, at scores of ordinary size"""
    counts = [40, 26]
    b = Trees([300, 90], 2, D, kb, 4, page=16, seed=kb)
    see = [ancestors(some_tree(c, c)) for c in counts]
    q = queries(66, 8, D, torch.bfloat16, gain=gain)
    q[3::7] = 0
    q[5::7] *= 2.0 ** (-3 if gain > 1 else 3)
    b.check(q, counts, D ** -0.5 / gain, tree=torch.cat([pack(s, 2) for s in see]).to(DEV), see=see)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_queries_that_are_no_numbers(dtype, value, path):
    """spoil their own row"""
    counts, D = [40, 26], 128
    b = Trees([300, 90], 2, D, page=16, seed=1)
    tree = torch.cat([pack(ancestors(some_tree(c, c)), 2) for c in counts]).to(DEV)
    q = queries(66, 8, D, dtype)
    ref, ref_lse = b.attend(q, counts, D ** -0.5, tree=tree)
    bad = torch.zeros((66, 8), dtype=torch.bool, device=DEV)
    bad[7, 3] = bad[41, 0] = bad[65, 7] = True
    q[7, 3, 5] = q[41, 0, 0] = q[65, 7, 127] = value
    out, lse = b.attend(q, counts, D ** -0.5, tree=tree)
    assert torch.equal(out[~bad], ref[~bad]) and torch.equal(lse[~bad], ref_lse[~bad])
    assert not torch.isfinite(lse[bad]).any() if math.isnan(value) else True
    assert torch.isnan(out[bad]).all() if math.isnan(value) else not (out[bad] == ref[bad]).all()
    assert _cabi.device_status() == 0


@pytest.mark.parametrize("kv,counts", [([4, 30, 0], [9, 30, 6]), ([70, 3], [90, 60])])
def test_fewer_tokens_than_queries(kv, counts, path):
    """the first drafted tokens are not in the cache"""
    b = Trees(kv, 2, 64, page=16, seed=1)
    b.run(counts, 2, 64)


def test_two_streams_and_two_graphs(path):
    """calls in parts, whose partial results lie in workspaces, next to each other"""
    D, counts = 128, [16, 64]
    b = Trees([6000, 3000], 1, D, 8, 4, page=64, seed=1)
    tree = torch.cat([pack(ancestors(some_tree(c, c)), 2) for c in counts]).to(DEV)
    qs = [queries(80, 4, D, seed=s) for s in (1, 2)]
    refs = [b.attend(q, counts, D ** -0.5, tree=tree) for q in qs]
    table, starts = b.table.to(DEV), torch.tensor([0, 16, 80], dtype=torch.int32, device=DEV)
    call = lambda q: b.cache.attend(q, table, b.kv_dev, starts, 64, 6000, D ** -0.5, return_lse=True, tree=tree)
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(qs[i]))
    graphs = []
    torch.cuda.synchronize()
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(q)
        graphs.append((graph, out))
    for _ in range(20):
        for s, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for ref, mine, (_, out) in zip(refs, got, graphs):
        assert all(torch.equal(x, y) for r in mine + [out] for x, y in zip(ref, r))
    assert _cabi.device_status() == 0


@pytest.mark.parametrize("D", [64, 128])
def test_pools_of_more_than_two_to_the_31_words(D, path):
    counts = [40, 3]
    b = Trees([300, 70], 8, D, page=64, seed=1)
    tree = torch.cat([pack(ancestors(some_tree(c, c)), 2) for c in counts]).to(DEV)
    q = queries(43, 16, D)
    ref = b.attend(q, counts, D ** -0.5, tree=tree)
    small, pages = b.cache, 2 ** 31 // (8 * 64 * D // 4) + 16
    b.cache = PagedCache(pages, 64, 8, D, 8, 8)
    assert b.cache.k_codes.numel() > 2 ** 31
    last = pages - small.k_codes.shape[0]
    for name in ("k_codes", "v_codes", "k_scale", "v_scale"):
        getattr(b.cache, name)[last:] = getattr(small, name)
    b.table = torch.where(b.table >= 0, b.table + last, b.table)
    assert all(torch.equal(x, y) for x, y in zip(ref, b.attend(q, counts, D ** -0.5, tree=tree)))
    assert _cabi.device_status() == 0


def test_refusals():
    b = Trees([40], 2, 64)
    q = queries(10, 2, 64)
    tree = torch.zeros((10, 1), dtype=torch.int32, device=DEV)
    for bad in (tree[:9], tree.long(), tree[:, :0], tree[:, 0], torch.zeros((10, 2), dtype=torch.int32, device=DEV)[:, ::2]):
        with pytest.raises(ValueError, match="tree"):
            b.attend(q, [10], 0.125, tree=bad)
    with pytest.raises(ValueError, match="tree"):
        b.attend(q, [10], 0.125, tree=tree, causal=False)
    with pytest.raises(ValueError, match="window"):
        b.attend(q, [10], 0.125, tree=tree, window=9)
    with pytest.raises(ValueError, match="bits"):
        Trees([80], 2, 64).attend(queries(40, 2, 64), [40], 0.125, tree=torch.zeros((40, 1), dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="CUDA"):
        b.attend(q, [10], 0.125, tree=tree.cpu())
    with pytest.raises(ValueError, match="int32"):
        draft_tree(torch.zeros(3, device=DEV), b.kv_dev, b.kv_dev, 3)
    with pytest.raises(ValueError, match="q_starts"):
        draft_tree(torch.zeros(3, dtype=torch.int32, device=DEV), b.kv_dev, b.kv_dev, 3)
