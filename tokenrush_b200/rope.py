"""Rotation frequencies for `fused.paged_append`: radians per position of each pair of dims, in float64, and the factor on
cos and sin, for a model's own context or one stretched beyond it.

    none     f_i = theta^(-2i / rd)
    linear   f_i / factor                                    (positions are squeezed)
    ntk      theta -> theta * factor^(rd / (rd - 2))         (the slowest pair is stretched by `factor`, the fastest stays)
    yarn     pairs that turn fewer than `slow` times over the trained context are stretched by `factor`, pairs that turn more than
             `fast` times stay, linear in the pair's index between; cos and sin times 0.1 ln(factor) + 1
"""
from __future__ import annotations

import math

import torch


def frequencies(rotary_dim: int, theta: float, scaling: str = "none", factor: float = 1.0, trained: int = 32768, fast: float = 32.0,
                slow: float = 1.0, device="cuda"):
    """(inv_freq float64 [rotary_dim / 2] on `device`, amplitude).  trained: the context the model was trained on (yarn)."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and positive")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if not factor >= 1.0:
        raise ValueError("factor must be at least 1")
    if scaling == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk scaling needs a rotary_dim of 4 or more")
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    f, amplitude = theta ** (-2.0 * i / rotary_dim), 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        def pair(turns):          # the (fractional) index of the pair that turns this often over the trained context
            return rotary_dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rotary_dim - 1)
        stretched = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        f = f / factor * stretched + f * (1 - stretched)
        amplitude = 0.1 * math.log(factor) + 1.0
    return f.to(device), amplitude
