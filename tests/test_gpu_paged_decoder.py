"""The operators of a paged cache together, as a server uses them: a decoder skeleton whose sequences are prefilled in chunks, decode next to one another,
leave, and whose pages others take over.

Two runs of a sequence differ in how attention rounds (weights in fp16, sums in another order) and in the codes of the layers behind: with bf16 activations
one rounding is 2^-8 of a value, a layer adds a few of them, and a code on a rounding boundary moves a value by 1/127 of its row's largest.  Hidden states are
of order 1: 0.08 in the 2-norm is ten roundings of each element, and a wrong key, slot or mask moves it by a multiple of that."""
import pytest
import torch

from VAR_Q import _cabi
from VAR_Q.harness import StandInDecoder

pytestmark = pytest.mark.gpu


def make(**kw):
    torch.manual_seed(0)
    return StandInDecoder(depth=2, width=256, heads=8, kv_heads=2, head_dim=64, num_pages=40, page_size=16, **kw).to(torch.bfloat16)


def inputs(n, seed):
    return torch.randn((n, 256), generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()


def off(a, b):
    return ((a.float() - b.float()).norm() / b.float().norm()).item()


@pytest.mark.parametrize("kw", [{}, {"window": 40, "sinks": 4}, {"k_bits": 8, "v_bits": 4}])
def test_chunks_and_company_do_not_change_a_sequence(kw):
    model, x, y, z = make(**kw), inputs(150, 1), inputs(90, 2), inputs(33, 3)
    whole = model.step(["x"], [x])[0]
    model.finish("x")
    first = model.step(["y", "x"], [y[:50], x[:70]])[1]
    second = model.step(["x", "y"], [x[70:71], y[50:51]])[0]
    third = model.step(["z", "x"], [z, x[71:130]])[1]
    model.finish("y")
    last = [model.step(["x", "z"], [x[i:i + 1], inputs(1, i)])[0] for i in range(130, 150)]
    parts = torch.cat([first, second, third, *last])
    assert parts.shape == whole.shape
    assert off(parts, whole) <= 0.08
    other = make(**kw)
    alone = other.step(["y"], [y[:50]])[0]
    assert off(model.step(["fresh"], [y[:50]])[0], alone) <= 0.08           # in pages that others have left
    assert _cabi.device_status() == 0


def test_a_full_pool_takes_nothing():
    model = make()
    free = model.table.free_pages
    with pytest.raises(RuntimeError, match="pages"):
        model.step(["big"], [inputs(40 * 16 + 1, 1)])
    assert model.table.free_pages == free
