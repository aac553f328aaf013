"""The learnt factor of each head in the shape in which an attention module holds it."""
import pytest
import torch

from test_gpu_rotary import DEV, rows
from VAR_Q.hooks import LayerKV
from VAR_Q.rotary import Rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["BLHc", "BHLc"])
@pytest.mark.parametrize("heads", [3, 64, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_four_dimensions_are_a_column(fmt, heads, dtype):
    rot = Rotary(64, sections=(16, 16), restart=True, interleaved=True)
    factor = (torch.rand(heads, generator=torch.Generator().manual_seed(9)) * 4 + 1).to(dtype).to(DEV)
    shapes = [factor.float().view(-1, 1), factor.view(1, -1, 1, 1), factor.view(1, 1, -1, 1), torch.nn.Parameter(factor.view(1, -1, 1, 1))]
    layers = [LayerKV(8, 'G_TOKEN_HEAD', fmt) for _ in shapes]
    for side in (1, 3):
        x = rows(2, side * side, 3 * heads, 64, dtype=torch.bfloat16, seed=side)
        q, k, v = (t.transpose(1, 2) if fmt == "BHLc" else t for t in x.split(heads, 2))
        pos = torch.stack([torch.arange(side * side) // side, torch.arange(side * side) % side]).to(torch.int32).to(DEV)
        outs = [layer.step_rotated(q, k, v, rot, pos, 1.0, torch.bfloat16, q_weight=w) for layer, w in zip(layers, shapes)]
        assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("shape", [(1, 5, 1, 1), (1, 1, 1, 1), (1, 3, 1, 64), (3, 1, 1, 3)])
def test_other_shapes_are_refused(shape):
    rot, layer = Rotary(64), LayerKV(8, 'G_TOKEN_HEAD', 'BLHc')
    q = rows(2, 4, 3, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="factor per head"):
        layer.step_rotated(q, q, q, rot, torch.arange(4, device=DEV), 1.0, q_weight=torch.ones(shape, device=DEV))
