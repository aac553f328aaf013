"""Factors behind the norm, element by element: what x * weight alone would lose in fp32 is not lost.  Tolerances: test_gpu_rotary.py."""
import pytest
import torch

from test_gpu_rotary import DEV, check
from VAR_Q.rotary import Rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("norm,gain,factor", [("l2", 1e-37, 1e-3), ("l2", 1e-30, 1e-12), ("l2", 1e16, 1e24), ("rms", 1e15, 1e25), ("rms", 1e-36, 1e-4)])
@pytest.mark.parametrize("shape", [(128,), (6, 128)])
def test_factors_are_behind_the_norm(dtype, norm, gain, factor, shape):
    """x / max(|x|, eps) * weight is an ordinary number where x * weight is subnormal or infinite"""
    rot = Rotary(128)
    g = torch.Generator().manual_seed(1)
    q, k = ((torch.randn((20, n, 128), generator=g, dtype=torch.float64) * gain).to(dtype).to(DEV) for n in (6, 6))
    weight = torch.randn(shape, generator=g) * factor
    pos = torch.arange(20, dtype=torch.int32) * 3
    out = torch.float32
    qo, ko = rot.rotate(q, k, pos.to(DEV), norm=norm, q_weight=weight.to(DEV), k_weight=weight.to(DEV), dtype=out)
    check(rot, q, qo, pos.view(1, -1), norm, weight)
    check(rot, k, ko, pos.view(1, -1), norm, weight)
