"""Rotary position plans: the frequency of every channel pair, its position axis and the
factor on the turned channels, as ``ops.rope`` and ``ops.norm_rope`` take them.

The world model turns a head's channels by the frame, row and column of a token
(``axes``, one run of channels each; P/matrix_curvature_phase_frame_weave.py:5394-5403
applies it ahead of the compact layer); a text stream turns them by one position.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Sequence

import torch

__all__ = ["RotaryPlan", "rotary_plan"]


class RotaryPlan(NamedTuple):
    """What a rotation keeps on the device."""
    turns: torch.Tensor             # float64 [R / 2]: whole turns per position
    axis: Optional[torch.Tensor]    # int32 [R / 2]: position axis of the pair (None: one axis)
    n_axes: int
    interleaved: bool
    scale: float                    # factor on the turned channels

    @property
    def rotary_dim(self) -> int:
        return 2 * self.turns.numel()


def rotary_plan(rotary_dim: int, *, base: float = 10000.0,
                axes: Optional[Sequence[int]] = None, interleaved: bool = False,
                scaling: Optional[str] = None, factor: float = 1.0,
                original_length: Optional[int] = None, low: float = 1.0, high: float = 32.0,
                scale: Optional[float] = None, device="cuda") -> RotaryPlan:
    """A plan that turns the first ``rotary_dim`` channels of a head.

    Pair i of n (of its axis) turns by ``base ** (-i / n)`` radians a position.  ``axes``
    gives the channels of each position axis (their sum is ``rotary_dim``; positions then
    have that many axes).  ``interleaved`` pairs channels (2i, 2i + 1), else
    (i, i + rotary_dim / 2).

    ``scaling`` stretches a context by ``factor``: "linear" divides the frequencies;
    "base" raises the base to ``base * factor ** (R / (R - 2))``, so that the slowest pair
    turns ``factor`` times slower and the fastest is kept; "ramp" keeps the pairs that turn
    more than ``high`` times in ``original_length`` positions, divides those that turn less
    than ``low`` times, blends between, and multiplies the turned channels by
    ``0.1 ln(factor) + 1`` (the published YaRN interpolation).  ``scale`` overrides that
    factor."""
    fn = "rotary_plan"
    rotary_dim = int(rotary_dim)
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f"{fn}: rotary_dim must be even, got {rotary_dim}")
    runs = [rotary_dim] if axes is None else [int(n) for n in axes]
    if not runs or any(n < 0 or n % 2 for n in runs) or sum(runs) != rotary_dim:
        raise ValueError(f"{fn}: axes {axes} must be even and sum to {rotary_dim}")
    if not (base > 0.0 and math.isfinite(base)):
        raise ValueError(f"{fn}: base must be positive, got {base}")
    if scaling not in (None, "linear", "base", "ramp"):
        raise ValueError(f"{fn}: unknown scaling {scaling!r}")
    if not (factor > 0.0 and math.isfinite(factor)):
        raise ValueError(f"{fn}: factor must be positive, got {factor}")
    if scaling is None and factor != 1.0:
        raise ValueError(f"{fn}: a factor needs a scaling")
    if scaling == "ramp" and not (original_length and original_length > 0 and high > low):
        raise ValueError(f"{fn}: ramp needs original_length and low < high")
    turns = []
    for n in runs:
        b = base
        if scaling == "base" and n > 2:
            b = base * factor ** (n / (n - 2.0))
        for i in range(n // 2):
            f = b ** (-2.0 * i / n)
            if scaling == "linear":
                f /= factor
            elif scaling == "ramp":
                whole = original_length * f / (2.0 * math.pi)
                keep = min(1.0, max(0.0, (whole - low) / (high - low)))
                f = f * keep + f / factor * (1.0 - keep)
            turns.append(f / (2.0 * math.pi))
    if scale is None:
        scale = 0.1 * math.log(factor) + 1.0 if scaling == "ramp" and factor > 1.0 else 1.0
    axis = None
    if len(runs) > 1:
        axis = torch.tensor([a for a, n in enumerate(runs) for _ in range(n // 2)],
                            dtype=torch.int32, device=device)
    return RotaryPlan(torch.tensor(turns, dtype=torch.float64, device=device), axis, len(runs),
                      bool(interleaved), float(scale))
