"""Rotary positions of one or several axes, with the norms of queries and keys in front of them, in one pass.

A transformer does two things to Q and K between its projection and its cache: a norm per head (VAR and Infinity: to unit length, times a learnt factor
per head, VAR/models/basic_var.py:137-141, Infinity/infinity/models/basic.py:316-320; other decoders: by the root mean square, times a learnt factor
per element) and a rotation by position (Infinity: rows and columns of the image, :325-326; texts: one axis; videos: time, height, width).
``Rotary.rotate`` does both for any consumer; ``PagedCache.append_rotated`` does both and quantises K and V into their pages.

Inference only: outputs have no gradient, whether or not the inputs require one.
"""
import math
from fractions import Fraction
from typing import Optional, Sequence, Tuple

import torch

from . import _cabi
from .quant import _host

# 2 pi, to 50 digits (a double is 0.1 radians off at position 10^15)
_TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937510")
NORMS = {None: (0, 1.0), "l2": (1, 1e-12), "rms": (2, 1e-6)}


def _native():
    return _host if _host is not None else _cabi.lib()                    # which says what to build


def _norm(norm, eps):
    if norm not in NORMS:
        raise ValueError(f"[VAR-Q]: norm must be None, 'l2' or 'rms' (got {norm!r})")
    code, usual = NORMS[norm]
    return code, usual if eps is None else float(eps)


class Rotary:
    """Which pairs of a head's elements turn, how fast, and by which axis' positions.

    ``rotary_dim`` (a multiple of 16, default ``head_dim``): elements from there on are not turned.  Pair i of ``rotary_dim / 2`` is the elements
    ``(2i, 2i + 1)`` (``interleaved``) or ``(i, i + rotary_dim / 2)``; it turns by ``position * frequency`` radians.
    ``sections``: how many pairs, one after another, go by each axis (default: all by one).  ``axes`` instead names the axis of every pair.
    Frequencies: ``base ** (-2i / rotary_dim)`` for pair i; with ``restart`` a section of n pairs has ``base ** (-2j / 2n)`` for its pair j, as if it were
    a rotary embedding of its own; or ``frequencies``, one for every pair.

    A frequency (a double, ``frequencies``) is held as a 64-bit fraction of a turn: an angle is off by less than position * 2^-65 + 2^-32 turns, and is then rounded once, to
    fp32 (2^-26 turns), for sine and cosine."""

    def __init__(self, head_dim: int, base: float = 10000.0, sections: Optional[Sequence[int]] = None, interleaved: bool = False, restart: bool = False,
                 rotary_dim: Optional[int] = None, frequencies: Optional[Sequence[float]] = None, axes: Optional[Sequence[int]] = None, device="cuda"):
        if head_dim not in (64, 128):
            raise ValueError(f"[VAR-Q]: head_dim {head_dim} is not 64 or 128")
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if rotary_dim < 16 or rotary_dim > head_dim or rotary_dim % 16:
            raise ValueError(f"[VAR-Q]: rotary_dim {rotary_dim} is not a multiple of 16 up to head_dim {head_dim}")
        pairs = rotary_dim // 2
        if sections is not None and axes is not None:
            raise ValueError("[VAR-Q]: sections or axes, not both")
        if axes is None:
            sections = [int(n) for n in ((pairs,) if sections is None else sections)]
            if any(n < 1 for n in sections) or sum(sections) != pairs:
                raise ValueError(f"[VAR-Q]: sections {tuple(sections)} do not add up to {pairs} pairs")
            axes = [a for a, n in enumerate(sections) for _ in range(n)]
        elif restart:
            raise ValueError("[VAR-Q]: restart goes with sections")
        else:
            axes = [int(a) for a in axes]
            if len(axes) != pairs or min(axes) < 0:
                raise ValueError(f"[VAR-Q]: axes must name the axis (0, 1, ...) of {pairs} pairs")
        if frequencies is None:
            if not (base > 0 and math.isfinite(base)):
                raise ValueError(f"[VAR-Q]: base must be positive and finite (got {base})")
            if restart:
                frequencies = [float(base) ** (-2.0 * j / (2 * n)) for n in sections for j in range(n)]
            else:
                frequencies = [float(base) ** (-2.0 * i / rotary_dim) for i in range(pairs)]
        else:
            frequencies = [float(f) for f in frequencies]
            if len(frequencies) != pairs or not all(math.isfinite(f) for f in frequencies):
                raise ValueError(f"[VAR-Q]: frequencies must be {pairs} finite numbers")
        self.head_dim, self.rotary_dim, self.interleaved, self.n_axes = head_dim, rotary_dim, bool(interleaved), max(axes) + 1
        self.frequencies, self.axes = tuple(frequencies), tuple(axes)
        turns = [round(Fraction(f) / _TWO_PI * 2 ** 64) % 2 ** 64 for f in frequencies]
        self.turns = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64, device=device)
        self.axis = torch.tensor(axes, dtype=torch.int32, device=device)
        self._handle = (self.turns, self.axis, self.n_axes, rotary_dim, self.interleaved, head_dim)

    def rotate(self, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, *, norm: Optional[str] = None, q_weight: Optional[torch.Tensor] = None,
               k_weight: Optional[torch.Tensor] = None, eps: Optional[float] = None, dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """``q`` and ``k`` after norm, weights and rotation: new contiguous tensors of their shapes, in their type or in ``dtype`` = float32.

        ``q`` ``[tokens, heads, head_dim]`` or ``[batch, tokens, heads, head_dim]`` (float32, float16 or bfloat16, strided views are fine), ``k`` the same with
        heads of its own.  ``positions``: int32 or int64, ``[axes, tokens]``, ``[axes, batch, tokens]``, or ``[tokens]`` where there is one axis; negative
        ones turn backwards.

        ``norm``: ``"l2"`` x / max(|x|, eps), ``"rms"`` x / sqrt(mean x^2 + eps), or None.  ``q_weight`` / ``k_weight``: float32 factors behind the norm,
        ``[head_dim]``, or ``[heads, head_dim]`` with 1 in either place.  Sums and products are fp32; the result is rounded once."""
        code, eps = _norm(norm, eps)
        return _native().rotate(*self._handle, q, k, positions, code, eps, q_weight, k_weight, dtype)
