"""Keys that are louder than all others by many powers of two, next to keys that matter in the columns in which the loud one's codes are zero.

A weight is held in fp16, times its V scale and relative to the row's reference.  Tolerance of an element: with p_j the softmax weights, v_j = c_j s_j the values, A = sum p_j |v_j| and
M = max p_j s_j: 2^-10 A for the weights' rounding (2^-12 each, twice where a reference is raised inside a tile) and for scores in fp32, FLOOR M sum |c_j| for weights below fp16's normal range
(2^-25 each, relative to the largest, which is held as 2^6 or more: FLOOR = 2^-30 with as much again for a second rounding), and the rounding of the output."""
import pytest
import torch

from test_gpu_paged_attention import DEV, Batch, queries
from VAR_Q import _cabi

pytestmark = pytest.mark.gpu
FLOOR = 2.0 ** -30


@pytest.fixture(params=["tc", "decode"], autouse=True)
def path(request):
    _cabi.force_attn_path(request.param)
    yield request.param
    _cabi.force_attn_path(None)


def case(score, gain, D=64, vb=8, page=64, seed=0):
    """one head; K such that a query of ones has score[j] (natural log), V ~ gain[j] with column 0 its largest; the loudest key's V is nothing but column 0"""
    n = len(score)
    b = Batch([n], 1, D, 8, vb, page=page, seed=seed)
    g = torch.Generator().manual_seed(seed)
    k = score.view(n, 1, 1).expand(n, 1, D).contiguous()
    v = torch.rand((n, 1, D), generator=g) * 0.6 + 0.1               # of one sign: roundings do not cancel
    v[:, 0, 0] = 1.0
    v[int(gain.argmax()), 0, 1:] = 0.0
    b.cache.append(k.to(DEV), (v * gain.view(n, 1, 1)).to(DEV), b.slots[0].to(DEV))
    return b


def check(b, c, dtype, D=64, **kw):
    q = torch.ones((c, 1, D), dtype=dtype, device=DEV)
    out, lse = b.attend(q, [c], 1.0 / D, causal=False, **kw)
    k, v = (t[:, 0].double() for t in b.cache.read(b.slots[0].to(DEV)))
    slots = b.slots[0].to(DEV)
    s = b.cache.v_scale[slots // b.page, 0, slots % b.page].double().view(-1, 1)
    x = (k.sum(1) / D).view(-1, 1)
    p = torch.softmax(x, 0)
    ref, A = (p * v).sum(0), (p * v.abs()).sum(0)
    tol = 2.0 ** -10 * A + FLOOR * (p * s).max() * (v / s).abs().sum(0) + (2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8) * ref.abs()
    off = (out[:, 0].double() - ref).abs() / (tol + 1e-7)
    assert off[:, 1:].max().item() <= 1.0, f"{off[:, 1:].max().item():.2f} of the bound"
    if ref[0] < torch.finfo(dtype).max:
        assert off[:, 0].max().item() <= 1.0
    assert (lse.double() - torch.logsumexp(x, 0)).abs().max().item() <= 2.0 ** -14
    assert _cabi.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("up", [10.3, 18.0, 21.7, 23.4])
def test_a_reference_raised_inside_a_tile(up, dtype):
    """the first half of a tile's weights is there, up to 2^7.5 times the reference, when a key in the second half raises it by 2^up"""
    ln2 = 0.6931471805599453
    n = 192
    score, gain = torch.zeros(n), torch.ones(n)
    score[64:96] = 7.5 * ln2
    score[96] = (7.5 + 3.0) * ln2
    gain[96] = 2.0 ** (up - 3.0)
    check(case(score, gain, seed=int(up)), 3, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("at", [5, 100, 20000])
@pytest.mark.parametrize("D,vb,n", [(64, 8, 30000), (128, 4, 30000), (64, 8, 21000)])
def test_one_loud_key_over_a_long_context(at, D, vb, n, dtype):
    """2^13 heavier than the others and with a V scale 2^13 times theirs; the others hold most of the softmax's mass (one part: the longest length is a hint)"""
    ln2 = 0.6931471805599453
    g = torch.Generator().manual_seed(at)
    score, gain = torch.rand(n, generator=g) * 2 - 1, torch.full((n,), 1.0)
    score[at], gain[at] = 13 * ln2, 2.0 ** 13
    check(case(score, gain, D, vb, seed=at), 2, dtype, D, max_kv=1)


@pytest.mark.parametrize("at", [0, 5, 31, 32, 63, 64, 100, 199])
@pytest.mark.parametrize("D,vb", [(64, 8), (128, 8), (64, 4)])
def test_a_key_that_is_nearly_everything_comes_out_as_it_is(at, D, vb):
    """its weight is held exactly, so that only the output's own rounding is left (and e^-25 of the others, 2^-18 for the reciprocals and the exponential in fp32)"""
    n = 200
    score, gain = torch.zeros(n), torch.ones(n)
    score[at] = 25.0
    b = case(score, gain, D, vb, seed=at)
    v = torch.rand((1, 1, D), generator=torch.Generator().manual_seed(at + 1)) - 0.5
    b.cache.append(torch.full((1, 1, D), 25.0, device=DEV), v.to(DEV), b.slots[0][at:at + 1].to(DEV))
    q = torch.ones((3, 1, D), dtype=torch.float16, device=DEV)
    out, _ = b.attend(q, [3], 1.0 / D, causal=False)
    ref = b.cache.read(b.slots[0][at:at + 1].to(DEV))[1].double()
    assert ((out.double() - ref).abs() <= 2.0 ** -11 * ref.abs() + 2.0 ** -18 * ref.abs() + n * 2.0 ** -36 + 2.0 ** -25).all()
