"""Angles of positions anywhere in 64 bits, against the table itself in whole numbers: turns * position modulo 2^64.

Tolerance: the kernel takes the upper 32 bits of that number (off by 2^-32 turns at most) rounded to fp32 (2^-26 turns, test_gpu_rotary.py counts 2^-25 of half a
turn), which its 2^-19 (|a| + |b|) covers with sine's and cosine's 2^-23."""
import math

import pytest
import torch

from test_gpu_rotary import DEV, rows
from VAR_Q.rotary import Rotary

pytestmark = pytest.mark.gpu


def turned(rot, x, positions):
    """y and |a| + |b| in float64 from the table"""
    x = x.double().cpu()
    y, both = x.clone(), x.abs()
    for i, (turn, axis) in enumerate(zip(rot.turns.tolist(), rot.axes)):
        t = torch.tensor([2 * math.pi * ((turn * p % 2 ** 64) / 2 ** 64) for p in positions[axis].tolist()], dtype=torch.float64).unsqueeze(-1)
        a, b = (2 * i, 2 * i + 1) if rot.interleaved else (i, i + rot.rotary_dim // 2)
        y[..., a] = x[..., a] * t.cos() - x[..., b] * t.sin()
        y[..., b] = x[..., b] * t.cos() + x[..., a] * t.sin()
        both[..., a] = both[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, both


FAR = [2 ** 40 + 12345, -2 ** 50, 2 ** 62, 0, 2 ** 63 - 1, -2 ** 63, 2 ** 33, -1, 2 ** 53 + 1, -2 ** 62 - 987654321]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("axes", [1, 2])
def test_positions_of_64_bits(interleaved, D, axes):
    rot = Rotary(D, interleaved=interleaved, sections=[D // 2] if axes == 1 else [D // 8, 3 * D // 8])
    pos = torch.tensor([FAR, FAR[::-1]][:axes], dtype=torch.int64)
    q, k = rows(len(FAR), 3, D), rows(len(FAR), 1, D, seed=1)
    for x, got in zip((q, k), rot.rotate(q, k, pos.to(DEV))):
        ref, both = turned(rot, x, pos)
        worst = ((got.double().cpu() - ref).abs() / (2.0 ** -19 * both + 2.0 ** -24 * ref.abs() * 1.01 + 1e-38)).max().item()
        assert worst <= 1.0, f"{worst:.3f} of the bound"


@pytest.mark.parametrize("positions", [[0, 1, -1, 2 ** 31 - 1, -2 ** 31, 123456789]])
def test_positions_of_32_bits(positions):
    rot = Rotary(64)
    pos = torch.tensor([positions], dtype=torch.int32)
    q = rows(6, 2, 64)
    ref, both = turned(rot, q, pos)
    got = rot.rotate(q, q, pos.to(DEV))[0].double().cpu()
    assert ((got - ref).abs() <= 2.0 ** -19 * both + 2.0 ** -24 * ref.abs() * 1.01 + 1e-38).all()
