"""Norms and rotary positions of queries and keys against the formula in 64 bits, and the same in front of a paged cache.

Tolerances, from the arithmetic: a row's sum of squares is at most 20 roundings deep, halved by the root; root, division and two products add one or two each:
below 2^-20 of an element before the rotation.  The angle's turns are rounded to 2^-25 of half a turn at most (8 2^-26 radians), sine and cosine to 2^-23: below 2^-21.
So y = a cos t - b sin t is off by at most 2^-19 (|a| + |b|) before its own rounding, which is half a step of the output's type (2^-25 absolute where fp16 is subnormal)."""
import math
from fractions import Fraction

import pytest
import torch

from VAR_Q import _cabi
from VAR_Q.hooks import LayerKV
from VAR_Q.paged import PagedCache
from VAR_Q.rotary import NORMS, Rotary

pytestmark = pytest.mark.gpu
DEV = "cuda"
TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937510")


def reference(rot, x, positions, norm, weight, eps):
    """y and |a| + |b| of every element, in float64; x [..., tokens, heads, dim], positions [axes, ..., tokens] as integers on the host"""
    x = x.double().cpu()
    if norm == "l2":
        x = x / x.square().sum(-1, keepdim=True).sqrt().clamp(min=eps)
    if norm == "rms":
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        x = x * weight.double().cpu()
    y, both = x.clone(), x.abs()
    for i, (f, axis) in enumerate(zip(rot.frequencies, rot.axes)):
        turn = Fraction(f) / TWO_PI
        pos = positions[axis].flatten().tolist()
        t = torch.tensor([2 * math.pi * float((turn * p) % 1) for p in pos], dtype=torch.float64).view(positions[axis].shape).unsqueeze(-1)
        a, b = (2 * i, 2 * i + 1) if rot.interleaved else (i, i + rot.rotary_dim // 2)
        y[..., a] = x[..., a] * t.cos() - x[..., b] * t.sin()
        y[..., b] = x[..., b] * t.cos() + x[..., a] * t.sin()
        both[..., a] = both[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, both


def check(rot, x, got, positions, norm=None, weight=None, eps=None):
    ref, both = reference(rot, x, positions, norm, weight, NORMS[norm][1] if eps is None else eps)
    half = torch.finfo(got.dtype).eps / 2
    got = got.double().cpu()
    tol = 2.0 ** -19 * both + half * ref.abs() * 1.01 + (2.0 ** -25 if half == 2.0 ** -11 else 1e-38)
    assert got.shape == x.shape
    worst = ((got - ref).abs() / tol).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3f} of the bound"


def rows(*shape, dtype=torch.float32, seed=0, gain=1.0):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * gain
    x[..., 5] *= 8.0
    return x.to(dtype).to(DEV)


TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("norm", [None, "l2", "rms"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_types_norms_pairs(D, dtype, norm, interleaved):
    rot = Rotary(D, interleaved=interleaved)
    q, k = rows(37, 5, D, dtype=dtype), rows(37, 2, D, dtype=dtype, seed=1)
    pos = torch.randint(0, 100000, (37,), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    qo, ko = rot.rotate(q, k, pos.to(DEV), norm=norm)
    assert qo.dtype == ko.dtype == dtype and qo.is_contiguous() and ko.is_contiguous()
    check(rot, q, qo, pos.view(1, -1), norm)
    check(rot, k, ko, pos.view(1, -1), norm)


@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 1, 1), (1, 64, 8), (2, 3, 3), (17, 28, 4), (300, 7, 1), (5000, 9, 2), (3, 0, 2), (3, 2, 0), (0, 4, 4)])
@pytest.mark.parametrize("D", [64, 128])
def test_sizes(tokens, heads, kv_heads, D):
    rot = Rotary(D, base=500000.0)
    q, k = rows(tokens, heads, D, dtype=torch.bfloat16), rows(tokens, kv_heads, D, dtype=torch.bfloat16, seed=1)
    pos = torch.arange(tokens, dtype=torch.int64) * 7 + 3
    qo, ko = rot.rotate(q, k, pos.to(DEV), norm="rms")
    check(rot, q, qo, pos.view(1, -1), "rms")
    check(rot, k, ko, pos.view(1, -1), "rms")


@pytest.mark.parametrize("kw", [dict(sections=(16, 24, 24)), dict(sections=(32, 32), restart=True, interleaved=True), dict(sections=(1, 62, 1)),
                                dict(rotary_dim=64), dict(rotary_dim=64, interleaved=True), dict(rotary_dim=16, sections=(3, 5)), dict(rotary_dim=96), dict(rotary_dim=112, interleaved=True),
                                dict(axes=[0, 1, 2, 1] * 16), dict(frequencies=[(-1) ** i * 3.0 ** (i % 7 - 5) for i in range(64)])])
def test_axes_and_frequencies(kw):
    rot = Rotary(128, **kw)
    q, k = rows(3, 50, 4, 128), rows(3, 50, 2, 128, seed=1)
    gen = torch.Generator().manual_seed(3)
    for shape in ((rot.n_axes, 50), (rot.n_axes, 3, 50)):                   # shared by the batch, and not
        pos = torch.randint(-200, 4000, shape, generator=gen, dtype=torch.int32)
        qo, ko = rot.rotate(q, k, pos.to(DEV), norm="l2")
        on_host = pos.unsqueeze(1).expand(-1, 3, -1) if pos.dim() == 2 else pos
        check(rot, q, qo, on_host, "l2")
        check(rot, k, ko, on_host, "l2")


@pytest.mark.parametrize("positions", [[0, 1, -1, 2 ** 31 - 1, -2 ** 31, 123456789], [2 ** 40 + 12345, -2 ** 50, 2 ** 62, 0, 2 ** 63 - 1, -2 ** 63]])
def test_far_positions(positions):
    # (turns carry 2^-65 each: from 2^42 on the angle is off by more than the bound, so of the long ones only the first is compared)
    rot = Rotary(64)
    pos = torch.tensor(positions, dtype=torch.int32 if max(positions) < 2 ** 31 else torch.int64)
    q, k = rows(6, 2, 64), rows(6, 1, 64, seed=1)
    qo, ko = rot.rotate(q, k, pos.to(DEV))
    n = 6 if pos.dtype == torch.int32 else 1
    check(rot, q[:n], qo[:n], pos.view(1, -1)[:, :n])
    check(rot, k[:n], ko[:n], pos.view(1, -1)[:, :n])
    # lengths of pairs stay what they are, wherever
    assert torch.allclose(qo.view(6, 2, 2, 32).norm(dim=2), q.view(6, 2, 2, 32).norm(dim=2), rtol=1e-6)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_weights(dtype):
    rot = Rotary(128)
    q, k = rows(20, 6, 128, dtype=dtype), rows(20, 3, 128, dtype=dtype, seed=1)
    pos = torch.arange(20, dtype=torch.int32)
    g = torch.Generator().manual_seed(5)
    per_dim, per_head, both = torch.randn(128, generator=g), torch.randn((6, 1), generator=g), torch.randn((3, 128), generator=g)
    strided = torch.randn((3, 256), generator=g)[:, ::2]
    odd = torch.randn(129, generator=g)[1:]                                  # four bytes off
    for qw, kw in ((per_dim, None), (per_head, both), (None, per_dim.view(1, -1)), (odd, strided), (torch.full((1, 1), 0.5), None)):
        on = lambda w: None if w is None else w.to(DEV)  # noqa: E731
        qo, ko = rot.rotate(q, k, pos.to(DEV), norm="rms", q_weight=on(qw), k_weight=on(kw), eps=1e-5)
        check(rot, q, qo, pos.view(1, -1), "rms", qw, 1e-5)
        check(rot, k, ko, pos.view(1, -1), "rms", kw, 1e-5)
    w = torch.randn((6, 256), generator=g).to(DEV)[:, ::2]                   # a view whose elements are not neighbours
    qo, _ = rot.rotate(q, k, pos.to(DEV), q_weight=w)
    check(rot, q, qo, pos.view(1, -1), None, w)


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_views(dtype):
    rot = Rotary(64, interleaved=True)
    fused = rows(33, 11, 64, dtype=dtype)
    pos = torch.arange(33, dtype=torch.int32)
    q, k = fused[:, :5], fused[:, 5:8]
    for a, b in ((q, k), (q.transpose(0, 1).contiguous().transpose(0, 1), k)):
        qo, ko = rot.rotate(a, b, pos.to(DEV), norm="l2")
        check(rot, a, qo, pos.view(1, -1), "l2")
        check(rot, b, ko, pos.view(1, -1), "l2")
    odd = rows(33, 5, 67, dtype=dtype)[..., 1:65]                            # rows that start anywhere
    qo, ko = rot.rotate(odd, k, pos.to(DEV), norm="l2")
    check(rot, odd, qo, pos.view(1, -1), "l2")
    # other layouts by transposed views; positions with a stride
    x = rows(2, 3, 33, 64, dtype=dtype)
    y = x.transpose(1, 2)
    wide = torch.arange(66, dtype=torch.int64, device=DEV)[::2]
    qo, ko = rot.rotate(y, y, wide)
    check(rot, y, qo, (pos * 2).view(1, 1, -1).expand(-1, 2, -1))
    assert torch.equal(qo, ko)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_fp32_outputs(dtype):
    rot = Rotary(128)
    q, k = rows(9, 4, 128, dtype=dtype), rows(9, 4, 128, dtype=dtype, seed=1)
    pos = torch.arange(9, dtype=torch.int32)
    qo, ko = rot.rotate(q, k, pos.to(DEV), norm="rms", dtype=torch.float32)
    assert qo.dtype == torch.float32
    check(rot, q, qo, pos.view(1, -1), "rms")
    check(rot, k, ko, pos.view(1, -1), "rms")
    q16, k16 = rot.rotate(q, k, pos.to(DEV), norm="rms")
    assert torch.equal(qo.to(dtype), q16) and torch.equal(ko.to(dtype), k16)


@pytest.mark.parametrize("interleaved", [False, True])
def test_zeros_infinities_and_nan(interleaved):
    rot = Rotary(64, rotary_dim=32, interleaved=interleaved)
    q = rows(4, 2, 64)
    q[0] = 0.0
    q[1, 0, 40] = math.inf                                                  # where nothing turns
    q[2, 0, 3] = math.nan
    pos = torch.arange(4, dtype=torch.int32, device=DEV)
    out, _ = rot.rotate(q, q, pos)
    assert (out[0] == 0).all() and not torch.isnan(out[1]).any() and out[1, 0, 40] == math.inf
    touched = {2, 3} if interleaved else {3, 19}
    assert set(torch.isnan(out[2, 0]).nonzero().flatten().tolist()) == touched and not torch.isnan(out[2, 1]).any()
    for norm in ("l2", "rms"):
        out, _ = rot.rotate(q, q, pos, norm=norm)
        assert (out[0] == 0).all()                                          # 0 / eps
        assert torch.isnan(out[2, 0]).all() and not torch.isnan(out[2, 1]).any() and not torch.isnan(out[3]).any()


# ------------------------------------------------------------------------------------------------ in front of the cache
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kb,vb", [(8, 8), (4, 2), (2, 4)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("norm,kw", [(None, dict()), ("rms", dict(interleaved=True)), ("l2", dict(rotary_dim=48, sections=(10, 14)))])
def test_append_is_rotate_and_append(D, kb, vb, dtype, norm, kw):
    """one launch gives the bits of rotation to fp32 and a separate append"""
    rot, page, heads, kv_heads, tokens = Rotary(D, **kw), 16, 6, 3, 70
    fused = rows(tokens, heads + 2 * kv_heads, D, dtype=dtype)
    q, k, v = fused.split((heads, kv_heads, kv_heads), 1)
    g = torch.Generator().manual_seed(1)
    pos = torch.randint(0, 10 ** 6, (rot.n_axes, tokens), generator=g).to(DEV)
    slots = torch.randperm(7 * page, generator=g)[:tokens]
    slots[3] = -1
    slots = slots.to(DEV)
    w = torch.randn(D, generator=g).to(DEV)
    one, two = (PagedCache(7, page, kv_heads, D, kb, vb) for _ in range(2))
    for c in (one, two):
        for pool in (c.k_codes, c.v_codes, c.k_scale, c.v_scale):
            pool.fill_(7)
    out = one.append_rotated(q, k, v, slots, rot, pos, norm=norm, q_weight=w, k_weight=w)
    q2, k2 = rot.rotate(q, k, pos, norm=norm, q_weight=w, k_weight=w, dtype=torch.float32)
    two.append(k2, v.float(), slots)
    assert torch.equal(out, q2.to(dtype))
    for a, b in ((one.k_codes, two.k_codes), (one.v_codes, two.v_codes), (one.k_scale, two.k_scale), (one.v_scale, two.v_scale)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("tokens", [1, 33, 4000])
def test_append_sizes(tokens):
    rot, D, kv_heads = Rotary(128), 128, 2
    cache = PagedCache(-(-tokens // 64) + 1, 64, kv_heads, D, 8, 4)
    q, k, v = (rows(tokens, h, D, dtype=torch.bfloat16, seed=h) for h in (7, kv_heads, kv_heads))
    slots = torch.arange(tokens, device=DEV) + 3
    pos = torch.arange(tokens, dtype=torch.int32)
    out = cache.append_rotated(q, k, v, slots, rot, pos.to(DEV), norm="rms")
    check(rot, q, out, pos.view(1, -1), "rms")
    kr, vr = cache.read(slots)
    ref, _ = reference(rot, k, pos.view(1, -1), "rms", None, 1e-6)
    step = ref.abs().amax(-1, keepdim=True) / 127                           # half a step, and what the element was off by
    assert ((kr.double().cpu() - ref).abs() <= step * (0.5 + 1e-3)).all()
    other = PagedCache(cache.num_pages, 64, kv_heads, D, 8, 4)
    other.append(k, v, slots)
    assert torch.equal(vr, other.read(slots)[1])


def test_append_with_bad_rows_and_no_tokens():
    rot, cache = Rotary(64), PagedCache(2, 16, 1, 64)
    q = rows(3, 2, 64)
    k, v = rows(3, 1, 64, seed=1), rows(3, 1, 64, seed=2)
    k[1, 0, 7] = math.nan
    v[2, 0, 7] = math.inf
    slots, pos = torch.tensor([0, 1, 2], device=DEV), torch.arange(3, device=DEV)
    cache.append_rotated(q, k, v, slots, rot, pos, norm="rms")
    kr, vr = cache.read(slots)
    assert torch.isnan(kr[1]).all() and not torch.isnan(kr[[0, 2]]).any() and torch.isnan(vr[2]).all() and not torch.isnan(vr[:2]).any()
    before = cache.k_codes.clone()
    out = cache.append_rotated(q[:0], k[:0], v[:0], slots[:0], rot, pos[:0])
    assert out.shape == (0, 2, 64)
    out = cache.append_rotated(q, k, v, torch.tensor([-1, 32, 2 ** 40], device=DEV), rot, pos)      # nowhere to write; the queries turn all the same
    assert torch.equal(before, cache.k_codes) and torch.equal(out, rot.rotate(q, k, pos)[0])
    cache.append_rotated(q[:, :0], k, v, slots, rot, pos)                   # no query heads


def test_streams_and_graphs():
    rot = Rotary(128)
    q, k, v = (rows(50, h, 128, dtype=torch.bfloat16, seed=h) for h in (4, 2, 2))
    pos, slots = torch.arange(50, device=DEV), torch.arange(50, device=DEV)
    cache = PagedCache(1, 64, 2, 128)
    ref = rot.rotate(q, k, pos, norm="rms")
    cache.append_rotated(q, k, v, slots, rot, pos, norm="rms")
    codes = cache.k_codes.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rot.rotate(q, k, pos, norm="rms")
    side.synchronize()
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.append_rotated(q, k, v, slots, rot, pos, norm="rms")
    cache.k_codes.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ref[0]) and torch.equal(cache.k_codes[:, :, :50], codes[:, :, :50])
    pos.add_(5)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, rot.rotate(q, k, pos, norm="rms")[0])


def test_offsets_behind_two_to_the_31():
    rot, heads, few = Rotary(128, interleaved=True), 32, 50
    tokens = 2 ** 31 // (heads * 128) + few
    last = rows(few, heads + 2, 128, dtype=torch.bfloat16)
    q, pos = torch.zeros((tokens, heads + 2, 128), dtype=torch.bfloat16, device=DEV), torch.arange(tokens, device=DEV)
    q[-few:] = last
    ref = rot.rotate(last[:, :heads], last[:, heads:], pos[-few:], norm="l2")
    for got, x in zip(rot.rotate(q[:, :heads], q[:, heads:], pos, norm="l2"), ref):
        assert torch.equal(got[-few:], x) and not got[:few].any()
    del q, got
    page = 64
    pages = 2 ** 31 // (2 * page * 128 // 4) + 3                            # a pool of as many words
    far, near = PagedCache(pages, page, 2, 128), PagedCache(1, page, 2, 128)
    slots = torch.arange(few, device=DEV)
    q, k = last[:, :heads], last[:, heads:]
    out = [c.append_rotated(q, k, k, slots + at, rot, pos[-few:], norm="l2") for c, at in ((near, 0), (far, (pages - 1) * page))]
    assert torch.equal(*out) and torch.equal(out[0], ref[0])
    for a, b in ((near.k_codes, far.k_codes), (near.v_codes, far.v_codes), (near.k_scale, far.k_scale), (near.v_scale, far.v_scale)):
        assert torch.equal(a[0, :, :few], b[-1, :, :few])


@pytest.mark.parametrize("dtype", TYPES)
def test_shared_rows(dtype):
    """strides of zero: one row for all tokens, or for all heads"""
    rot = Rotary(64, rotary_dim=48)
    x, pos = rows(1, 1, 64, dtype=dtype), torch.arange(30, device=DEV) * 1000
    q, k = x.expand(30, 5, 64), x[0].expand(30, 2, 64)
    got, ref = rot.rotate(q, k, pos, norm="rms"), rot.rotate(q.contiguous(), k.contiguous(), pos, norm="rms")
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    at = pos[:1].expand(30)
    assert all(torch.equal(a, b) for a, b in zip(rot.rotate(q, k, at), rot.rotate(q, k, at.contiguous())))


# ------------------------------------------------------------------------------------------------ in front of an image schedule
@pytest.mark.parametrize("fmt", ["BLHc", "BHLc"])
def test_a_schedule_with_two_axes(fmt):
    """step_rotated is the norms, the rotation and the ordinary step"""
    rot, heads, B = Rotary(64, sections=(16, 16), restart=True, interleaved=True), 3, 2
    fused, plain = (LayerKV(8, 'G_TOKEN_HEAD', fmt) for _ in range(2))
    factor = torch.rand((heads, 1), generator=torch.Generator().manual_seed(9)).to(DEV) * 4 + 1
    for side in (1, 2, 3, 5):
        x = rows(B, side * side, 3 * heads, 64, dtype=torch.bfloat16, seed=side)
        q, k, v = x.split(heads, 2)
        pos = torch.stack([torch.arange(side * side) // side, torch.arange(side * side) % side]).to(torch.int32).to(DEV)
        qn, kn = (torch.nn.functional.normalize(t.float(), dim=-1) for t in (q, k))
        qr, kr = rot.rotate(qn * factor, kn, pos)
        turn = (lambda t: t.transpose(1, 2)) if fmt == "BHLc" else (lambda t: t)
        out = fused.step_rotated(turn(q), turn(k), turn(v), rot, pos, 1.0, torch.bfloat16, q_weight=factor)
        ref = plain.step(turn(qr), turn(kr), turn(v), 1.0, torch.bfloat16)
        assert out.shape == (B, side * side, heads, 64)
        # 8-bit codes of two K that differ by some 2^-22: a code on a rounding boundary moves one element of one key by 1 / 127 of its largest
        assert ((out.float() - ref.float()).norm() / ref.float().norm()).item() <= 2.0 ** -7
    assert fused.n_tokens == 1 + 4 + 9 + 25 and _cabi.device_status() == 0
