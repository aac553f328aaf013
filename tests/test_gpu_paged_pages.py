"""Copies of pages and moves of tokens, bit for bit against indexing on the host, in caches of different shapes side by side."""
import random

import pytest
import torch

from VAR_Q import _cabi
from VAR_Q.paged import PagedCache, PageTable, copy_pages, move_tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHAPES = [(3, 64, 8, 8), (1, 128, 4, 2), (8, 128, 8, 4), (5, 64, 2, 2), (2, 128, 2, 8)]


def caches(n, pages, page, seed=0):
    g = torch.Generator().manual_seed(seed)
    made = []
    for i in range(n):
        heads, D, kb, vb = SHAPES[i % len(SHAPES)]
        c = PagedCache(pages, page, heads, D, kb, vb)
        for pool in pools(c):
            pool.view(torch.int32).copy_(torch.randint(-2 ** 31, 2 ** 31 - 1, pool.shape, generator=g, dtype=torch.int32))
        made.append(c)
    return made


def pools(c):
    return [t.view(torch.int32) for t in (c.k_codes, c.v_codes, c.k_scale, c.v_scale)]


def snapshot(cs):
    return [[p.clone() for p in pools(c)] for c in cs]


def same(cs, expected):
    return all(torch.equal(a, b) for c, e in zip(cs, expected) for a, b in zip(pools(c), e))


def longs(x):
    return torch.tensor(x, dtype=torch.int64, device=DEV)


@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("layers", [1, 5, 64, 65, 130])
def test_pages(page, layers):
    pages = 6 if page == 1024 else 23
    cs = caches(layers, pages, page)
    order = random.Random(1).sample(range(pages), pages)
    half = pages // 2
    src, dst = order[:half], order[half:2 * half]
    expected = snapshot(cs)
    for e in expected:
        for p in e:
            p[dst] = p[src]
    before = _cabi.lib().varq_launch_count()
    copy_pages(cs, longs(src), longs(dst))
    assert _cabi.lib().varq_launch_count() - before == -(-layers // 64)
    assert same(cs, expected)


def test_one_page_to_many_and_pages_that_are_not_there():
    cs = caches(2, 9, 16) + caches(1, 4, 16)                                 # the last one has fewer pages
    expected = snapshot(cs)
    src, dst = [0, 0, 0, -1, 5, 2, 9, 2 ** 40], [1, 3, 6, 2, -1, 8, 4, 7]
    for e in expected:
        for p in e:
            for a, b in zip(src, dst):
                if 0 <= a < len(p) and 0 <= b < len(p):
                    p[b] = p[a]
    copy_pages(cs, longs(src), longs(dst))
    assert same(cs, expected)
    copy_pages(cs, longs([]), longs([]))
    copy_pages([], longs([1]), longs([2]))
    assert same(cs, expected) and _cabi.device_status() == 0


def moved(cs, moves, page):
    """one after another, on copies"""
    expected = snapshot(cs)
    for e in expected:
        for p in e:
            for a, b in moves:
                if 0 <= a < len(p) * page and 0 <= b < len(p) * page:
                    p[b // page, :, b % page] = p[a // page, :, a % page]
    return expected


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("layers", [1, 5, 66])
@pytest.mark.parametrize("draft", [1, 8, 64, 200, 700])
def test_accepted_drafts(page, layers, draft):
    """tokens move towards the front over one another's places, in groups of any length"""
    rng = random.Random(draft)
    groups = 4
    per = -(-(draft + 30) // page)
    cs = caches(layers if draft < 200 else min(layers, 5), groups * per, page, seed=draft)
    order = rng.sample(range(groups * per), groups * per)
    src, dst, starts = [], [], [0]
    for g in range(groups):
        at = lambda i: order[g * per + i // page] * page + i % page  # noqa: E731
        base = rng.randrange(30)
        kept = [i for i in range(draft) if g != 2 and rng.random() < (0.95 if g == 1 else 0.4)]      # many neighbours, few, none
        src += [at(base + i) for j, i in enumerate(kept) if g or i != j]      # (in the first group without those that stay)
        dst += [at(base + j) for j, i in enumerate(kept) if g or i != j]
        starts.append(len(src))
    expected = moved(cs, list(zip(src, dst)), page)
    move_tokens(cs, longs(src), longs(dst), torch.tensor(starts, dtype=torch.int32, device=DEV), draft)
    assert same(cs, expected) and _cabi.device_status() == 0


@pytest.mark.parametrize("layers,shape", [(40, (8, 128, 8, 8)), (70, (3, 64, 2, 4)), (9, (37, 128, 8, 4)), (2, (70, 64, 8, 8))])
@pytest.mark.parametrize("groups,most", [(70, 5), (64, 31), (1, 6), (1, 300)])
def test_caches_of_one_shape(layers, shape, groups, most):
    """a block may go through several caches and heads; one cache has fewer pages than the others"""
    page, span = 16, -(-2 * most // 16) * 16
    heads, D, kb, vb = shape
    rng = random.Random(groups + most)
    cs = [PagedCache(groups * span // page // (2 if i == layers - 1 and groups > 1 else 1), page, heads, D, kb, vb) for i in range(layers)]
    for c in cs:
        for pool in pools(c):
            pool.random_(-2 ** 31, 2 ** 31 - 1)
    src, dst, starts = [], [], [0]
    for g in range(groups):
        kept = sorted(rng.sample(range(2 * most), rng.randint(0 if groups > 1 else most, most)))
        src += [g * span + i for j, i in enumerate(kept) if i != j]
        dst += [g * span + j for j, i in enumerate(kept) if i != j]
        starts.append(len(src))
    src, dst = longs(src), longs(dst)
    expected = snapshot(cs)
    for e, c in zip(expected, cs):
        there = (src < c.num_pages * page) & (dst < c.num_pages * page)
        s, d = src[there], dst[there]
        for p in e:                                                        # no place is written before it is read
            p[d // page, :, d % page] = p[s // page, :, s % page]
    move_tokens(cs, src, dst, torch.tensor(starts, dtype=torch.int32, device=DEV), most)
    assert same(cs, expected) and _cabi.device_status() == 0


def test_long_moves_to_fresh_pages_with_any_hint():
    page, n = 32, 1500
    rng = random.Random(4)
    kept = sorted(rng.sample(range(3000), n))
    src, dst = kept, [3008 + i for i in range(n)]
    for hint in (0, 1, n, 2 ** 31 - 1):
        cs = caches(3, 142, page, seed=hint % 97)
        expected = moved(cs, list(zip(src, dst)), page)
        move_tokens(cs, longs(src), longs(dst), torch.tensor([0, n], dtype=torch.int32, device=DEV), hint)
        assert same(cs, expected)


def test_moves_that_are_none_and_starts_out_of_bounds():
    page = 16
    cs = caches(2, 5, page)
    ints = dict(dtype=torch.int32, device=DEV)
    src, dst = [3, -1, 9, 80, 7, 2 ** 45], [1, 2, -1, 5, 7, 4]
    expected = moved(cs, [(3, 1)], page)
    move_tokens(cs, longs(src), longs(dst), torch.tensor([0, 4, 6], **ints), 4)
    assert same(cs, expected) and _cabi.device_status() == 0
    expected = moved(cs, [(40, 41)], page)
    move_tokens(cs, longs([40]), longs([41]), torch.tensor([-3, 1, 99, 5], **ints), 4)      # clamped: one move, and no other
    assert _cabi.device_status() == 64 and same(cs, expected)
    move_tokens(cs, longs([]), longs([]), torch.tensor([0, 0], **ints), 0)
    move_tokens(cs, longs([1]), longs([2]), torch.tensor([0], **ints), 0)                     # no groups
    assert same(cs, expected)


def test_streams_and_graphs():
    cs = caches(3, 12, 16)
    src, dst, starts = longs([3, 20]), longs([2, 19]), torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    pages = longs([0, 1]), longs([10, 11])
    expected = moved(cs, [(3, 2), (20, 19)], 16)
    for e in expected:
        for p in e:
            p[[10, 11]] = p[[0, 1]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        move_tokens(cs, src, dst, starts, 1)
        copy_pages(cs, *pages)
    side.synchronize()
    assert same(cs, expected)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        move_tokens(cs, src, dst, starts, 1)
        copy_pages(cs, *pages)
    src.copy_(longs([50, 60]))
    expected = moved(cs, [(50, 2), (60, 19)], 16)
    for e in expected:
        for p in e:
            p[[10, 11]] = p[[0, 1]]
    graph.replay()
    torch.cuda.synchronize()
    assert same(cs, expected)


def test_pools_of_more_than_two_to_the_31_words():
    page, H, D = 64, 8, 128
    pages = 2 ** 31 // (H * page * D // 4) + 3
    cs = [PagedCache(pages, page, H, D, 8, 8)]
    for pool in pools(cs[0]):
        pool.zero_()
        pool[-2].random_()
        pool[1].random_()
    first, last = ([p[i].clone() for p in pools(cs[0])] for i in (1, -2))
    copy_pages(cs, longs([pages - 2, 1]), longs([0, pages - 1]))
    for p, a, z in zip(pools(cs[0]), first, last):
        assert torch.equal(p[0], z) and torch.equal(p[-1], a) and not p[2].any() and not p[-3].any()
    src, dst = [(pages - 2) * page + i for i in range(3, 64)], [2 * page + i for i in range(61)]
    for most in (61, 1):
        move_tokens(cs, longs(src + [page + 5]), longs(dst + [(pages - 3) * page + 63]), torch.tensor([0, 61, 62], dtype=torch.int32, device=DEV), most)
        for p, a, z in zip(pools(cs[0]), first, last):
            assert torch.equal(p[2, :, :61], z[:, 3:]) and not p[2, :, 61:].any() and torch.equal(p[-3, :, 63], a[:, 5]) and not p[-3, :, :63].any()
            p[2] = p[-3] = 0
    assert _cabi.device_status() == 0


def test_refusals():
    a, b = caches(1, 4, 16)[0], caches(1, 4, 32)[0]
    one = longs([1])
    with pytest.raises(ValueError, match="pages of 16 and 32"):
        copy_pages([a, b], one, one)
    with pytest.raises(ValueError, match="one length"):
        copy_pages([a], longs([1, 2]), one)
    with pytest.raises(ValueError, match="int64"):
        copy_pages([a], one.int(), one)
    with pytest.raises(RuntimeError, match="CUDA"):
        copy_pages([a], one.cpu(), one)
    starts = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="starts"):
        move_tokens([a], one, one, starts.long(), 1)
    with pytest.raises(ValueError, match="most"):
        move_tokens([a], one, one, starts, -1)
    with pytest.raises(ValueError, match="one length"):
        move_tokens([a], longs([1, 2]), one, starts, 1)


# ------------------------------------------------------------------------------------------------ with the table
def test_table_and_caches_together():
    """tokens of forked, cut and compacted sequences are where the table says"""
    page, D = 16, 64
    table, cache = PageTable(40, page), PagedCache(40, page, 1, D)
    rng, texts, count = random.Random(0), {}, 0
    mark = lambda i: (torch.arange(D) + 1.0) * (1 + i % 251)  # noqa: E731      # scale and codes tell the tokens apart

    def write(name, ids):
        x = torch.stack([mark(i) for i in ids]).view(-1, 1, D).to(DEV)
        cache.append(x, x, table.extend([name], [len(ids)]))
        texts[name] = texts[name] + ids

    for step in range(120):
        act = rng.choice(("add", "write", "write", "fork", "accept", "accept", "remove", "compact"))
        if act == "add" and len(texts) < 5:
            table.add(step)
            texts[step] = []
        elif act == "write" and texts:
            name, n = rng.choice(list(texts)), rng.randint(1, 40)
            if table.free_pages >= 4:
                write(name, list(range(count, count + n)))
                count += n
        elif act == "fork" and texts and len(texts) < 6 and table.free_pages > 2:
            names = [rng.choice(list(texts)) for _ in range(2)]
            children = [(step, 0), (step, 1)]
            copy_pages([cache], *table.fork(names, children))
            for a, b in zip(names, children):
                texts[b] = list(texts[a])
        elif act == "accept" and texts and table.free_pages >= 4:
            name, n = rng.choice(list(texts)), rng.randint(1, 40)
            write(name, list(range(count, count + n)))
            count += n
            kept = sorted(rng.sample(range(n), rng.randint(0, n)))
            move_tokens([cache], *table.accept([name], [n], [kept]))
            base = len(texts[name]) - n
            texts[name] = texts[name][:base] + [texts[name][base + i] for i in kept]
        elif act == "remove" and len(texts) > 2:
            name = rng.choice(list(texts))
            table.remove(name)
            del texts[name]
        elif act == "compact":
            copy_pages([cache], *table.compact())
            used = 40 - table.free_pages
            assert all(s < used * page for name in texts for s in table.slots(name, "cpu").tolist())
        for name, ids in texts.items():
            assert table.length(name) == len(ids)
            if ids:
                k, _ = cache.read(table.slots(name))
                top = k[:, 0].amax(-1).cpu()
                assert torch.allclose(top, torch.tensor([64.0 * (1 + i % 251) for i in ids]), rtol=1e-5)
    for name in list(texts):
        table.remove(name)
    assert table.free_pages == 40
