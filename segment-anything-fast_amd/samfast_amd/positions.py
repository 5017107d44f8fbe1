"""Positions and frequencies for ops.rotary."""

import math
from typing import Optional

import torch

SCALINGS = ("none", "linear", "bands")


def rotary_frequencies(pairs: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, trained_length: int = 4096,
                       slow_turns: float = 1.0, fast_turns: float = 32.0, device: Optional[torch.device] = None) -> torch.Tensor:
    """fp64 (pairs,): base^(-p / pairs) radians a position for pair p, stretched for contexts `factor` times as long as the trained ones:

    "none":   as they are;
    "linear": all of them `factor` times as slow (positions squeezed into the trained length);
    "bands":  pairs that make at least `fast_turns` turns within `trained_length` positions as they are, those that make at most `slow_turns`
              `factor` times as slow, the ones between by the share of the way that their turns lie on."""
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
    if pairs <= 0 or base <= 0 or factor <= 0 or trained_length <= 0 or not 0 <= slow_turns < fast_turns:
        raise ValueError("pairs, base, factor and trained_length must be positive, and slow_turns below fast_turns")
    f = torch.tensor(base, dtype=torch.float64, device=device) ** (-torch.arange(pairs, dtype=torch.float64, device=device) / pairs)
    if scaling == "linear":
        return f / factor
    if scaling == "bands":
        kept = ((trained_length * f / (2.0 * math.pi) - slow_turns) / (fast_turns - slow_turns)).clamp_(0.0, 1.0)
        return f * (kept + (1.0 - kept) / factor)
    return f


def grid_positions(height: int, width: int, device: Optional[torch.device] = None) -> torch.Tensor:
    """int64 (height * width, 2): row and column of each token of a grid, as the encoder orders them."""
    n = torch.arange(height * width, device=device)
    return torch.stack((n // width, n % width), -1)
