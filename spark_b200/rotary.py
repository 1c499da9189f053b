"""Rotary positions: the table of cosines and sines, and the differentiable
application of it to q and k (ops.rope).
"""
from __future__ import annotations

import math

import torch

from . import ops


def rope_frequencies(rot_dim: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                     original_positions: int = 4096, fast: float = 32.0, slow: float = 1.0):
    """(angle per position of each pair, fp64 [rot_dim / 2]; factor on cosines and sines).

    scaling: None: base ** (-2 i / rot_dim);
    "linear": positions divided by `factor`;
    "ntk": the base grows so that the slowest pair turns `factor` times slower;
    "yarn": pairs that turn more than `fast` times within `original_positions` keep
    their angle, those that turn less than `slow` times are divided by `factor`, the
    ones between are blended linearly in the pair's index, and the attention's logits
    are sharpened by (0.1 ln(factor) + 1) on q and on k."""
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rope_frequencies: rot_dim must be even and positive, got {rot_dim}")
    if base <= 0 or factor <= 0:
        raise ValueError("rope_frequencies: base and factor must be positive")
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    if scaling == "ntk":
        base = base * factor ** (rot_dim / max(rot_dim - 2, 1))
    freq = base ** (-i / rot_dim)
    if scaling in (None, "ntk"):
        return freq, 1.0
    if scaling == "linear":
        return freq / factor, 1.0
    if scaling != "yarn":
        raise ValueError(f"rope_frequencies: scaling {scaling!r} is none of None, 'linear', 'ntk', 'yarn'")

    def pair(turns):
        """The (real) index of the pair that turns so often within original_positions."""
        return rot_dim * math.log(original_positions / (turns * 2 * math.pi)) / (2 * math.log(base))

    # (the blend may end behind the last pair, which then keeps a part of its angle)
    lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rot_dim - 1)
    blend = ((torch.arange(rot_dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
    return freq * (1 - blend) + freq / factor * blend, (0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0)


def rope_table(positions: int, rot_dim: int, base: float = 10000.0, device=None, **scaling) -> torch.Tensor:
    """fp32 [positions, rot_dim]: the cosines of every position's angles, then the
    sines, computed in fp64 (rope_frequencies; its keywords are passed on)."""
    freq, factor = rope_frequencies(rot_dim, base, **scaling)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return (torch.cat([angle.cos(), angle.sin()], 1) * factor).float().to(device or "cuda")


def apply_rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, table: torch.Tensor,
               interleaved: bool = False):
    """Differentiable ops.rope: (q', k'), gradients of gradients too.  The gradients of the
    positions and of the table are not computed; forward-mode differentiation is refused."""
    _, ws, stream = ops._place("rope", q)
    y, z, rc = ops._native().apply_rope(q, k, positions, table, interleaved, ws, stream)
    if rc:
        ops._check("spark_rope", rc)
    return y, z
