r"""Rotary positions on the CPU in torch operators: angles in float64, the turn in float32
(float64 for float64 features), one rounding. The backward is torch autograd."""

from __future__ import annotations

from collections.abc import Sequence

import torch
from torch import Tensor

from ...core.sanitize import rotary_sections
from ...registry import Backend, RotaryContext, rotary

__all__ = ["rotary_eager"]


def rotary_eager(x: Tensor, positions: Tensor, frequencies: Tensor, *, sections: Sequence[int] | None = None,
                 interleaved: bool = False) -> Tensor:
    """Run the rotary positions on the CPU in torch operators."""
    if x.device.type != "cpu":
        raise RuntimeError(f"the eager rotary backend runs on CPU tensors only; got a tensor on {x.device}")
    counts = rotary_sections(positions, frequencies, sections)
    compute = torch.float64 if x.dtype == torch.float64 else torch.float32
    axis = [a for a, n in enumerate(counts) for _ in range(n)]
    angles = positions.to(torch.float64)[..., axis] * frequencies.to(torch.float64)  # (L, R) or (B, L, R)
    cos, sin = torch.cos(angles).to(compute).unsqueeze(-2), torch.sin(angles).to(compute).unsqueeze(-2)
    pairs = len(axis)
    wide = x.to(compute)
    if interleaved:
        a, b = wide[..., 0:2 * pairs:2], wide[..., 1:2 * pairs:2]
    else:
        a, b = wide[..., :pairs], wide[..., pairs:2 * pairs]
    first, second = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([first, second], -1).flatten(-2) if interleaved else torch.cat([first, second], -1)
    return torch.cat([turned, wide[..., 2 * pairs:]], -1).to(x.dtype)


def supports_context(context: RotaryContext) -> bool:
    """CPU tensors of a floating dtype."""
    return context.device.type == "cpu" and context.dtype.is_floating_point


rotary.register(Backend.EAGER, rotary_eager, supports=supports_context)
