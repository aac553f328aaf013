"""Rows whose squares leave fp32 behind the norms: finite ones come out as the formula says, in front of a cache too.

Tolerances are those of test_gpu_rotary.py.  The rows are multiplied by 2^-68 before their squares are added up, which is exact but for elements that become subnormal:
those are off by 2^-150, next to a root of the sum (of the mean) of 2^-8 or more, so by 2^-142 of a result for which the tolerance holds 1e-38."""
import math

import pytest
import torch

from test_gpu_rotary import DEV, check, reference, rows
from VAR_Q import _cabi
from VAR_Q.paged import PagedCache
from VAR_Q.rotary import Rotary

pytestmark = pytest.mark.gpu
MOST = 3.3e38


def large(tokens, heads, D, dtype, gain, seed=0):
    """rows of `gain`; every third one is ordinary, next to them in the same warp"""
    x = torch.randn((tokens, heads, D), generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * gain
    x[..., 5] *= 8.0
    x[::3] /= gain
    return x.clamp(-MOST, MOST).to(dtype).to(DEV)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("norm", ["l2", "rms"])
@pytest.mark.parametrize("gain", [1e17, 1e18, 3e18, 1e19, 1e25, 1e33, 1e37, 1e39])
@pytest.mark.parametrize("interleaved", [False, True])
def test_norms(D, dtype, norm, gain, interleaved):
    rot = Rotary(D, interleaved=interleaved, rotary_dim=D - 16)
    q, k = large(20, 5, D, dtype, gain), large(20, 2, D, dtype, gain, seed=1)
    pos = torch.arange(20, dtype=torch.int32) * 17
    for out in (dtype, torch.float32):
        qo, ko = rot.rotate(q, k, pos.to(DEV), norm=norm, dtype=out)
        check(rot, q, qo, pos.view(1, -1), norm)
        check(rot, k, ko, pos.view(1, -1), norm)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("norm", ["l2", "rms"])
def test_weights_and_views(dtype, norm):
    rot = Rotary(128)
    q, k = large(30, 7, 128, dtype, 1e30)[..., 1:4, :], large(30, 9, 128, dtype, 1e22, seed=1)[:, ::3]
    odd = torch.empty(30 * 3 * 128 + 1, dtype=dtype, device=DEV)[1:].view(30, 3, 128).copy_(q)      # rows that do not begin on 16 bytes
    g = torch.Generator().manual_seed(3)
    per_head, per_dim, both = torch.rand((3, 1), generator=g) * 9 + 1, torch.randn(128, generator=g), torch.randn((3, 128), generator=g)
    pos = torch.arange(30, dtype=torch.int64)
    for x, qw, kw in ((q, per_head, None), (odd, per_dim, both), (q, both, per_dim), (q, None, per_head)):
        on = lambda w: None if w is None else w.to(DEV)  # noqa: E731
        qo, ko = rot.rotate(x, k, pos.to(DEV), norm=norm, q_weight=on(qw), k_weight=on(kw))
        check(rot, x, qo, pos.view(1, -1), norm, qw)
        check(rot, k, ko, pos.view(1, -1), norm, kw)


@pytest.mark.parametrize("norm", ["l2", "rms"])
@pytest.mark.parametrize("value", [MOST, 2.0 ** 64, 2.0 ** 61, 1.0])
def test_rows_of_one_value(norm, value):
    """the squares of all elements at their largest, and around the border"""
    rot = Rotary(128)
    q = torch.full((4, 2, 128), value, device=DEV)
    q[1, :, 1::2] *= -1.0
    q[2, :, 1:] = 0.0                                                       # one element alone
    q[3, :, 3] = 1e-20
    pos = torch.arange(4, dtype=torch.int32)
    out, _ = rot.rotate(q, q[:, :1], pos.to(DEV), norm=norm)
    check(rot, q, out, pos.view(1, -1), norm)


@pytest.mark.parametrize("norm", ["l2", "rms"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinities_next_to_large_elements(norm, dtype):
    """x / |x| where |x| is infinite: 0 for what is finite, no number for what is not; nothing of it reaches another row"""
    rot = Rotary(64, rotary_dim=32)
    q = large(9, 2, 64, dtype, 1e30)
    q[4, 0, 40] = math.inf                                                  # where nothing turns
    q[7, 1, 3] = math.nan
    pos = torch.arange(9, dtype=torch.int32)
    out, _ = rot.rotate(q, q, pos.to(DEV), norm=norm)
    assert out[4, 0, 40].isnan() and (out[4, 0, :40] == 0).all() and (out[4, 0, 41:] == 0).all() and out[7, 1].isnan().all()
    good = [0, 1, 2, 3, 5, 6, 8]
    check(rot, q[good], out[good], pos[good].view(1, -1), norm)
    assert torch.isfinite(out[[4, 7], [1, 0]]).all()


@pytest.mark.parametrize("D,kb,dtype", [(64, 4, torch.float32), (128, 8, torch.bfloat16), (128, 8, torch.float32)])
@pytest.mark.parametrize("norm", ["l2", "rms"])
def test_append(D, kb, dtype, norm):
    """keys of such rows are no zeros in the cache: the values of the formula to half a step of their codes, the bits of rotation and a separate append"""
    rot, tokens = Rotary(D), 40
    q, k = large(tokens, 4, D, dtype, 1e25), large(tokens, 2, D, dtype, 1e30, seed=1)
    v = rows(tokens, 2, D, dtype=dtype, seed=2)
    one, two = (PagedCache(4, 16, 2, D, kb, 8) for _ in range(2))
    slots, pos = torch.arange(tokens, device=DEV), torch.arange(tokens, dtype=torch.int32)
    out = one.append_rotated(q, k, v, slots, rot, pos.to(DEV), norm=norm)
    check(rot, q, out, pos.view(1, -1), norm)
    q2, k2 = rot.rotate(q, k, pos.to(DEV), norm=norm, dtype=torch.float32)
    two.append(k2, v.float(), slots)
    at = (slice(None), slice(None), slice(None))
    for a, b in zip(one.read(slots), two.read(slots)):
        assert torch.equal(a[at], b[at])
    assert torch.equal(out, q2.to(dtype))
    ref, _ = reference(rot, k, pos.view(1, -1), norm, None, {"l2": 1e-12, "rms": 1e-6}[norm])
    step = ref.abs().amax(-1, keepdim=True) / (2 ** (kb - 1) - 1)
    assert ((one.read(slots)[0].double().cpu() - ref).abs() <= step * (0.5 + 1e-3)).all()
    assert _cabi.device_status() == 0


@pytest.mark.parametrize("eps", [1e-18, 1e-9, 1e-3, 1.0, 1e6, 1e11, 1e13, 9e17])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("norm", ["l2", "rms"])
def test_any_eps(eps, dtype, norm):
    """norms around eps, wherever it lies, with a factor for the row and for its elements"""
    rot = Rotary(64)
    g = torch.Generator().manual_seed(4)
    sizes = torch.logspace(-3, 3, 25, dtype=torch.float64).view(-1, 1, 1) * (eps if norm == "l2" else eps ** 0.5) / 8
    sizes[7] = 0.0
    most = 6e4 if dtype == torch.float16 else MOST
    q = (torch.randn((25, 3, 64), generator=g, dtype=torch.float64) * sizes).clamp(-most, most).to(dtype).to(DEV)
    pos = torch.arange(25, dtype=torch.int32)
    per_head, per_dim = torch.rand((3, 1), generator=g) + 0.5, torch.rand(64, generator=g) + 0.5
    for weight in (None, per_head, per_dim):
        out, _ = rot.rotate(q, q, pos.to(DEV), norm=norm, eps=eps, q_weight=None if weight is None else weight.to(DEV), dtype=torch.float32)
        check(rot, q, out, pos.view(1, -1), norm, weight, eps)
