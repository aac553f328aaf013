"""Rotary positions, trees of drafted tokens, forked and compacted sequences together, as a server uses them, on the decoder skeleton.
The tolerance of hidden states is that of test_gpu_paged_decoder.py, where it is derived."""
import pytest
import torch

from test_gpu_paged_decoder import inputs, off
from VAR_Q import _cabi
from VAR_Q.harness import StandInDecoder
from VAR_Q.rotary import Rotary

pytestmark = pytest.mark.gpu


def make(**kw):
    torch.manual_seed(0)
    args = dict(rotary=Rotary(64, rotary_dim=32), qk_norm="rms")
    args.update(kw)
    return StandInDecoder(depth=2, width=256, heads=8, kv_heads=2, head_dim=64, num_pages=60, page_size=16, **args).to(torch.bfloat16)


TREE, PATH = [-1, 0, 0, 1, 1, 2, 4, 4, 6, -1, 9], [0, 1, 4, 6, 8]


@pytest.mark.parametrize("kw", [{}, {"window": 40, "sinks": 4}, {"rotary": None, "qk_norm": None}, {"qk_norm": "l2", "k_bits": 8, "v_bits": 4}])
def test_a_draft_and_its_accepted_path(kw):
    model, plain = make(**kw), make(**kw)
    x, y, draft, more = inputs(75, 1), inputs(18, 2), inputs(len(TREE), 3), inputs(20, 4)
    for m in (model, plain):
        m.step(["x", "y"], [x, y])
    out = model.verify(["y", "x"], [more[:1], draft], [[-1], TREE])[1]
    ref = plain.step(["x", "y"], [draft[PATH], more[:1]])[0]
    assert off(out[PATH], ref) <= 0.08
    for i, p in enumerate(TREE):                                           # and every other branch of it
        chain = [i]
        while TREE[chain[0]] >= 0:
            chain.insert(0, TREE[chain[0]])
        other = make(**kw)
        other.step(["x"], [x])
        assert off(out[i:i + 1], other.step(["x"], [draft[chain]])[0][-1:]) <= 0.08
    model.accept(["x", "y"], [len(TREE), 1], [PATH, [0]])
    assert model.table.length("x") == plain.table.length("x") == 75 + len(PATH) and model.table.free_pages == plain.table.free_pages
    for i in range(10):
        a, b = (m.step(["x", "y"], [more[i:i + 1], more[i + 1:i + 2]]) for m in (model, plain))
        assert off(a[0], b[0]) <= 0.08 and off(a[1], b[1]) <= 0.08
    assert _cabi.device_status() == 0


def test_forked_sequences_go_their_own_ways():
    model, plain = make(), make()
    x, a, b = inputs(59, 1), inputs(30, 2), inputs(30, 3)
    model.step(["x"], [x])
    free = model.table.free_pages
    model.fork(["x", "x"], ["a", "b"])
    assert model.table.free_pages == free - 2                              # a copy of the last page each, three are shared
    plain.step(["a", "b"], [x, x])
    for i in range(0, 30, 10):
        got, ref = model.step(["b", "a"], [b[i:i + 10], a[i:i + 10]]), plain.step(["b", "a"], [b[i:i + 10], a[i:i + 10]])
        assert off(got[0], ref[0]) <= 0.08 and off(got[1], ref[1]) <= 0.08
        if i == 0:
            model.finish("x")
    for name in ("a", "b"):
        model.finish(name)
    assert model.table.free_pages == 60


def test_a_compacted_pool_answers_as_before():
    model = make()
    x, y, z = inputs(90, 1), inputs(50, 2), inputs(40, 3)
    model.step(["x", "y", "z"], [x, y, z])
    model.fork(["z"], ["w"])
    model.finish("x")
    before = [model.verify([s], [inputs(1, 9)], [[-1]])[0] for s in ("y", "z", "w")]
    model.accept(["y", "z", "w"], [1, 1, 1], [[], [], []])
    model.compact()
    used = 60 - model.table.free_pages
    assert all(p < used for s in ("y", "z", "w") for p in model.table._pages[s])
    for s, ref in zip(("y", "z", "w"), before):
        assert torch.equal(model.verify([s], [inputs(1, 9)], [[-1]])[0], ref)
    assert _cabi.device_status() == 0


def test_refusals():
    model = make()
    model.step(["x"], [inputs(5, 1)])
    for parents in ([[0]], [[1]], [[-2]], [[-1, 0]], []):
        with pytest.raises(ValueError, match="parent"):
            model.verify(["x"], [inputs(1, 1)], parents)
    assert model.table.length("x") == 5
    model = make(window=8)
    model.step(["x"], [inputs(5, 1)])
    with pytest.raises(ValueError, match="window"):                        # before its tokens have taken any room
        model.verify(["x"], [inputs(9, 1)], [[-1] * 9])
    assert model.table.length("x") == 5
    with pytest.raises(ValueError, match="rotary"):
        StandInDecoder(depth=1, width=64, heads=1, kv_heads=1, qk_norm="l2")
    with pytest.raises(ValueError, match="axis"):
        StandInDecoder(depth=1, width=64, heads=1, kv_heads=1, rotary=Rotary(64, sections=(16, 16)))
