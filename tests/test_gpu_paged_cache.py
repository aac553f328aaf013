"""Writing to and reading from a paged cache, against torch on the CPU: packed words, scales and values bit for bit.

The definition is elementwise fp32 arithmetic with true division (scale = max(amax / (2^(bits-1) - 1), 1e-12), code = round half to even),
so nothing may differ: there is no tolerance in this file.  Values in 16 bits are one rounding of the fp32 product."""
import math

import pytest
import torch

from VAR_Q import _cabi
from VAR_Q.paged import PagedCache, PageTable

pytestmark = pytest.mark.gpu
DEV = "cuda"


def plain_rows(x, bits):
    """[T, H, D] -> words [T, H, D * bits / 32], scale [T, H], codes"""
    x = x.float().cpu()
    top = torch.tensor(float(2 ** (bits - 1) - 1))
    scale = (x.abs().amax(-1) / top).clamp_min(1e-12)
    codes = torch.round(x / scale.unsqueeze(-1)).clamp(-2 ** (bits - 1), 2 ** (bits - 1) - 1).to(torch.int64)
    per = 32 // bits
    fields = (codes & (2 ** bits - 1)).unflatten(-1, (-1, per)) << torch.arange(0, 32, bits)
    words = fields.sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32), scale, codes


def slots_of(pages, page_size, n, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pages * page_size, generator=g)[:n]


def pools_at(cache, slots):
    page, at = slots // cache.page_size, slots % cache.page_size
    return [t.cpu()[page, :, at] for t in (cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale)]


def check(cache, k, v, slots):
    kc, vc, ks, vs = pools_at(cache, slots)
    for got, got_scale, x, bits in ((kc, ks, k, cache.k_bits), (vc, vs, v, cache.v_bits)):
        words, scale, _ = plain_rows(x, bits)
        assert torch.equal(got, words)
        assert torch.equal(got_scale, scale)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        rk, rv = cache.read(slots.to(DEV), dtype)
        for got, x, bits in ((rk, k, cache.k_bits), (rv, v, cache.v_bits)):
            _, scale, codes = plain_rows(x, bits)
            assert torch.equal(got.cpu(), (codes.float() * scale.unsqueeze(-1)).to(dtype))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kb,vb", [(8, 8), (4, 4), (2, 2), (8, 4), (4, 2), (2, 8)])
@pytest.mark.parametrize("T,H,page", [(1, 1, 16), (3, 5, 32), (130, 8, 64), (999, 3, 1024)])
def test_round_trip(D, kb, vb, T, H, page):
    dtype = (torch.float32, torch.float16, torch.bfloat16)[(T + D + kb) % 3]
    pages = -(-T // page) + 2
    cache = PagedCache(pages, page, H, D, kb, vb)
    g = torch.Generator().manual_seed(T * D + kb * vb)
    k, v = (torch.randn((T, H, D), generator=g).mul_(s).to(dtype) for s in (3.0, 0.1))
    slots = slots_of(pages, page, T, T)
    cache.append(k.to(DEV), v.to(DEV), slots.to(DEV))
    check(cache, k, v, slots)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows(D, dtype):
    """enough rows for the form with several rows per thread, the last block of it ragged"""
    T, H, page = 12345 if D == 128 else 24683, 7, 64
    pages = -(-T // page) + 1
    cache = PagedCache(pages, page, H, D, 8, 4)
    g = torch.Generator().manual_seed(D)
    k, v = (torch.randn((T, H, D), generator=g).to(dtype) for _ in range(2))
    slots = slots_of(pages, page, T, 3)
    cache.append(k.to(DEV), v.to(DEV), slots.to(DEV))
    check(cache, k, v, slots)


@pytest.mark.parametrize("offset", [0, 1, 4, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_strided_and_unaligned_inputs(offset, dtype):
    """views of a fused activation; rows that do not start on 16 bytes take element loads"""
    T, H, D = 37, 3, 64
    g = torch.Generator().manual_seed(offset)
    fused = torch.randn((T, 3 * H * D + offset), generator=g).to(dtype).to(DEV)
    view = fused[:, offset:].unflatten(1, (3, H, D))
    k, v = view[:, 1], view[:, 2]
    cache = PagedCache(4, 16, H, D, 8, 2)
    slots = slots_of(4, 16, T, 1)
    cache.append(k, v, slots.to(DEV))
    check(cache, k, v, slots)
    heads_first = torch.randn((H, T, D), generator=g).to(dtype).to(DEV).transpose(0, 1)
    cache.append(heads_first, heads_first, slots.to(DEV))
    check(cache, heads_first, heads_first, slots)


@pytest.mark.parametrize("bits", [8, 4, 2])
def test_ties_and_their_neighbours(bits):
    """quotients on and next to k + 1/2, with scales that are and are not powers of two"""
    top = 2 ** (bits - 1) - 1
    rows = []
    for amax in (float(top), top * 0.75, 1.0, 3.1415927, 1e-20, 2.0 ** 100):
        base = torch.tensor([(c + 0.5) * amax / top for c in range(-top, top)][-62:] or [0.0])
        for nudge in (0.0, 1.0, -1.0):
            x = torch.zeros(64)
            y = base if nudge == 0 else torch.nextafter(base, torch.full_like(base, nudge * float("inf")))
            x[:len(y)] = y
            x[63] = amax
            rows.append(x.clamp(-amax, amax))
    k = torch.stack(rows).unsqueeze(1)
    cache = PagedCache(4, 16, 1, 64, bits, bits)
    slots = torch.arange(len(rows))
    cache.append(k.to(DEV), (-k).to(DEV), slots.to(DEV))
    check(cache, k, -k, slots)


@pytest.mark.parametrize("bits", [8, 4, 2])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_scales_of_every_magnitude(bits, dtype):
    """rows from the smallest to the largest numbers of the type, with every leading pattern of the largest value: the scale's division has to round as it should"""
    g = torch.Generator().manual_seed(bits)
    info = torch.finfo(dtype)
    lo, hi = math.log2(info.tiny), math.log2(info.max)
    T = 4096
    size = 2.0 ** (torch.rand((T, 1, 1), generator=g, dtype=torch.float64) * (hi - lo) + lo)
    k = (torch.rand((T, 1, 64), generator=g, dtype=torch.float64) * 2 - 1) * size
    k = k.clamp(-info.max, info.max).to(dtype)
    k[0, 0, 0], k[1, 0, 1], k[2] = info.max, -info.max, 0.0
    cache = PagedCache(T // 16, 16, 1, 64, bits, bits)
    slots = torch.arange(T)
    cache.append(k.to(DEV), (-k).to(DEV), slots.to(DEV))
    check(cache, k, -k, slots)


def test_tiny_rows_use_the_smallest_scale():
    k = torch.zeros((3, 1, 64))
    k[1, 0, 5] = 1e-13
    k[2, 0, 5] = 2e-10
    cache = PagedCache(1, 16, 1, 64, 8, 8)
    slots = torch.tensor([2, 0, 9])
    cache.append(k.to(DEV), k.to(DEV), slots.to(DEV))
    check(cache, k, k, slots)


def test_padding_slots_write_nothing_and_read_zeros():
    T, H, D = 20, 2, 128
    cache = PagedCache(2, 16, H, D, 4, 8)
    before = [t.random_(-1000, 1000).clone() for t in (cache.k_codes, cache.v_codes)] + [t.fill_(-7.0).clone() for t in (cache.k_scale, cache.v_scale)]
    k = torch.randn((T, H, D))
    k[::2] = float("nan")                                            # what a padding token holds does not matter
    slots = torch.full((T,), -1, dtype=torch.int64)
    slots[1::2] = torch.arange(3, 3 + T // 2)
    beyond = slots.clone()
    beyond[4] = 2 * 16                                               # behind the pool
    beyond[6] = 1 << 40
    for s in (slots, beyond):
        cache.append(k.to(DEV), k.to(DEV), s.to(DEV))
        kc, vc = cache.read(s.to(DEV))
        assert torch.equal(kc[0::2].cpu(), torch.zeros(T // 2, H, D)) and torch.equal(vc[0::2].cpu(), torch.zeros(T // 2, H, D))
        check(cache, k[1::2], k[1::2], slots[1::2])
    untouched = [i for i in range(32) if i not in slots.tolist()]
    for t, old in zip((cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale), before):
        flat = lambda x: x.transpose(1, 2).flatten(0, 1)[untouched].cpu()  # noqa: E731
        assert torch.equal(flat(t), flat(old))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_that_are_not_finite_read_as_nan(bad, dtype):
    k = torch.randn((4, 2, 64)).to(dtype)
    k[1, 0, 17] = bad
    k[3, 1, 63] = bad
    v = torch.randn((4, 2, 64)).to(dtype)
    cache = PagedCache(1, 16, 2, 64)
    slots = torch.tensor([5, 6, 7, 8])
    cache.append(k.to(DEV), v.to(DEV), slots.to(DEV))
    rk, rv = (t.cpu() for t in cache.read(slots.to(DEV)))
    whole = torch.ones((4, 2), dtype=torch.bool)
    whole[1, 0] = whole[3, 1] = False
    assert torch.isnan(rk[~whole]).all()
    _, scale, codes = plain_rows(k, 8)
    assert torch.equal(rk[whole], (codes.float() * scale.unsqueeze(-1))[whole])
    assert torch.isfinite(rv).all()


def test_nothing_to_do():
    cache = PagedCache(1, 16, 2, 64)
    none = torch.empty((0,), dtype=torch.int64, device=DEV)
    cache.append(torch.empty((0, 2, 64), device=DEV), torch.empty((0, 2, 64), device=DEV), none)
    k, v = cache.read(none, torch.float16)
    assert k.shape == v.shape == (0, 2, 64) and k.dtype == torch.float16


def test_pools_of_more_than_two_to_the_31_words():
    page, H, D = 64, 8, 128
    pages = 2 ** 31 // (H * page * D // 4) + 3                       # 8-bit codes, four in a word
    cache = PagedCache(pages, page, H, D, 8, 8)
    assert cache.k_codes.numel() > 2 ** 31
    k, v = torch.randn((5, H, D)), torch.randn((5, H, D))
    slots = torch.tensor([0, pages * page - 1, (pages - 1) * page, 17, (pages - 2) * page + 5])
    cache.append(k.to(DEV), v.to(DEV), slots.to(DEV))
    rk, rv = (t.cpu() for t in cache.read(slots.to(DEV)))
    for got, x in ((rk, k), (rv, v)):
        _, scale, codes = plain_rows(x, 8)
        assert torch.equal(got, codes.float() * scale.unsqueeze(-1))


def test_another_stream_and_a_graph():
    T, H, D = 50, 4, 64
    cache = PagedCache(8, 16, H, D, 8, 4)
    slots = slots_of(8, 16, T, 2)
    k, v, s = torch.randn((T, H, D), device=DEV), torch.randn((T, H, D), device=DEV), slots.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.append(k, v, s)
    torch.cuda.current_stream().wait_stream(side)
    check(cache, k, v, slots)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(k, v, s)
        out = cache.read(s)
    k.normal_(); v.normal_()
    graph.replay()
    torch.cuda.synchronize()
    check(cache, k, v, slots)
    assert torch.equal(out[0], cache.read(s)[0])


def test_refusals():
    T, H, D = 4, 2, 64
    cache = PagedCache(2, 16, H, D)
    k, s = torch.randn((T, H, D), device=DEV), torch.arange(T, device=DEV)
    with pytest.raises(ValueError, match="slot"):
        cache.append(k, k, s.int())
    with pytest.raises(ValueError, match="slot"):
        cache.append(k, k, torch.arange(2 * T, device=DEV)[::2])
    with pytest.raises(ValueError, match="heads"):
        cache.append(k[:, :1], k, s)
    with pytest.raises(ValueError, match="slot per token"):
        cache.append(k[:3], k, s)
    with pytest.raises(ValueError, match="type"):
        cache.append(k, k.half(), s)
    with pytest.raises(ValueError, match="type"):
        cache.append(k.double(), k.double(), s)
    with pytest.raises(ValueError, match="contiguous"):
        cache.append(k.transpose(1, 2).contiguous().transpose(1, 2), k, s)
    with pytest.raises(RuntimeError, match="CUDA"):
        cache.append(k.cpu(), k, s)
    with pytest.raises(TypeError):
        cache.append(None, k, s)
    with pytest.raises(ValueError, match="dtype"):
        cache.read(s, torch.float64)
    with pytest.raises(ValueError, match="head_dim"):
        PagedCache.over(cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale, 96).read(s)
    with pytest.raises(ValueError, match="pools"):
        PagedCache.over(cache.k_codes, cache.v_codes, cache.k_scale.half(), cache.v_scale, D).read(s)
    with pytest.raises(ValueError, match="pools differ"):
        PagedCache.over(cache.k_codes, cache.v_codes[:1], cache.k_scale, cache.v_scale, D).read(s)
    cache.eps = 0.0
    with pytest.raises(ValueError, match="eps"):
        cache.append(k, k, s)
    assert _cabi.device_status() == 0


def test_page_table_with_a_cache():
    """two sequences that grow in turn, one of which leaves and makes room"""
    table, cache = PageTable(6, 16), PagedCache(6, 16, 2, 64)
    kept = {"a": [], "b": []}
    table.add("a"); table.add("b")
    for na, nb in ((20, 3), (1, 1), (11, 30)):
        x = torch.randn((na + nb, 2, 64))
        cache.append(x.to(DEV), -x.to(DEV), table.extend(["a", "b"], [na, nb], DEV))
        kept["a"].append(x[:na]); kept["b"].append(x[na:])
    for name, parts in kept.items():
        x = torch.cat(parts)
        assert table.length(name) == len(x)
        check(cache, x, -x, table.slots(name, "cpu"))
    with pytest.raises(RuntimeError, match="pages"):
        table.extend(["a"], [60], DEV)
    table.remove("a")
    table.add("c")
    x = torch.randn((48, 2, 64))
    cache.append(x.to(DEV), x.to(DEV), table.extend(["c"], [48], DEV))
    check(cache, x, x, table.slots("c", "cpu"))
    check(cache, torch.cat(kept["b"]), -torch.cat(kept["b"]), table.slots("b", "cpu"))


@pytest.mark.parametrize("T", [1, 7, 300])
@pytest.mark.parametrize("kb,vb", [(8, 4), (2, 8)])
def test_nothing_is_written_outside(T, kb, vb):
    """pools, values, outputs and log-sums carved out of larger buffers whose rest has to stay as it is"""
    H, D, page, pages, G = 3, 64, 16, 24, 2
    lib = _cabi.lib()
    guard = 12345.0

    def carved(shape, dtype):
        n = int(torch.Size(shape).numel())
        big = torch.full((n + 256,), guard, dtype=torch.float32, device=DEV).to(dtype)
        return big, big[128:128 + n].view(shape)

    shape = (pages, H, page)
    bigs, pools = zip(carved((*shape, D * kb // 32), torch.int32), carved((*shape, D * vb // 32), torch.int32), carved(shape, torch.float32), carved(shape, torch.float32))
    cache = PagedCache.over(*pools, D)
    slots = torch.randperm(pages * page)[:T]
    slots[T // 2] = pages * page - 1 if pages * page - 1 not in slots else slots[T // 2]
    k, v = torch.randn((T, H, D)), torch.randn((T, H, D))
    cache.append(k.to(DEV), v.to(DEV), slots.to(DEV))
    check(cache, k, v, slots)
    read = [carved((T, H, D), torch.float16) for _ in range(2)]
    desc = [_cabi.Tensor(t.data_ptr(), _cabi.F16, 0, 0, H * D, D) for _, t in read]
    c = _cabi.Paged(*(p.data_ptr() for p in pools), pages, page, H, D, kb, vb)
    s = slots.to(DEV)
    _cabi.check(lib.varq_paged_read(c, s.data_ptr(), T, *desc, _cabi.stream_ptr(DEV)))
    assert torch.equal(read[0][1], cache.read(s, torch.float16)[0]) and torch.equal(read[1][1], cache.read(s, torch.float16)[1])
    # attention: a sequence over the first pages
    full = torch.arange(pages * page)
    x = torch.randn((pages * page, H, D), device=DEV)
    cache.append(x, x, full.to(DEV))
    n = min(T + 20, pages * page)
    q = torch.randn((T, H * G, D), device=DEV).half()
    table = torch.arange(pages, dtype=torch.int32, device=DEV).view(1, -1)
    lens, starts = (torch.tensor(z, dtype=torch.int32, device=DEV) for z in ([n], [0, T]))
    big_o, out = carved((T, H * G, D), torch.float16)
    big_l, lse = carved((T, H * G), torch.float32)
    od, qd = (_cabi.Tensor(t.data_ptr(), _cabi.F16, 0, 0, H * G * D, D) for t in (out, q))
    b = _cabi.PagedBatch(starts.data_ptr(), lens.data_ptr(), table.data_ptr(), pages, T, pages, 1, H * G, T, n, 1, 0, 0, 0.125)
    need = lib.varq_paged_attn_workspace_bytes(c, b)
    ws = torch.full((need + 512,), 77, dtype=torch.uint8, device=DEV)
    _cabi.check(lib.varq_paged_attn(c, b, qd, od, lse.data_ptr(), ws.data_ptr() + 256, need, _cabi.stream_ptr(DEV)))
    ref = cache.attend(q, table, lens, starts, T, n, 0.125, return_lse=True)
    assert torch.equal(out, ref[0]) and torch.equal(lse, ref[1])
    assert (ws[:256] == 77).all() and (ws[256 + need:] == 77).all()
    for big, t in list(zip(bigs, pools)) + read + [(big_o, out), (big_l, lse)]:
        edge = torch.cat([big[:128], big[128 + t.numel():]])
        assert torch.equal(edge, torch.full_like(edge, guard))
    assert lib.varq_paged_attn(c, b, qd, od, lse.data_ptr(), None, need - 1, _cabi.stream_ptr(DEV)) == (_cabi.ERR_WORKSPACE if need else 0)
