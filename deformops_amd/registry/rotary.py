r"""Rotary positions with several axes, for the queries and keys of attention.

A pyramid's positions have a place in the image and, in video, a time. Each axis turns
its own pairs of features. The reference has no counterpart.
"""

from __future__ import annotations

import dataclasses
from collections.abc import Sequence
from typing import Any

import torch
from torch import Tensor

from ..core.runtime import is_training_from
from ..core.sanitize import check_rotary_call, rotary_sections
from ._dispatch import Backend, Registry
from ._eager import plain_eager
from ._public import define_public_op

__all__ = ["RotaryContext", "rotary", "rotary_frequencies"]


@dataclasses.dataclass(frozen=True)
class RotaryContext:
    """What backend selection knows of a rotary call."""

    device: torch.device
    dtype: torch.dtype
    num_pairs: int
    row_elements: int
    is_training: bool


def select_backend(context: RotaryContext) -> list[Backend]:
    """GPU tensors run the HIP kernels and nothing else, CPU tensors the eager backend."""
    return [Backend.HIP] if context.device.type == "cuda" else [Backend.EAGER]


def rotary_frequencies(sections: Sequence[int], *, base: float = 10000.0, shared: bool = False,
                       device: torch.device | str | None = None) -> Tensor:
    """Float32 frequencies of ``sum(sections)`` pairs: ``base ** -(j / n)`` for pair ``j`` of
    an axis with ``n`` pairs, or with ``shared`` one ladder over all pairs in order."""
    counts = [sum(sections)] if shared else sections
    ladders = [torch.arange(n, dtype=torch.float64) / max(n, 1) for n in counts]
    exponents = torch.cat(ladders) if ladders else torch.zeros(0, dtype=torch.float64)
    return (base ** -exponents).float().to(device)


def _context_of(x: Tensor, positions: Tensor, frequencies: Tensor, *, sections: Sequence[int] | None = None,
                interleaved: bool = False) -> RotaryContext:  # noqa: ARG001
    check_rotary_call(x, positions, frequencies, sections)
    return RotaryContext(x.device, x.dtype, int(frequencies.shape[0]), int(x.shape[2]) * int(x.shape[3]),
                         is_training_from(x))


def _rotary_call(
    x: Tensor,
    positions: Tensor,
    frequencies: Tensor,
    /,
    *,
    sections: Sequence[int] | None = None,
    interleaved: bool = False,
    backend: Backend | None = None,
) -> Tensor:
    r"""Turn pairs of features by angles of the tokens' positions.

    Pair ``j`` of a token turns by ``position[axis of j] * frequencies[j]``:
    ``(a, b) -> (a cos - b sin, b cos + a sin)``.

    Parameters
    ----------
    x
        ``(B, L, H, D)``, float32, float16 or bfloat16 (float64 on the CPU too), in any
        memory layout.
    positions
        ``(L, A)`` or ``(B, L, A)`` (or ``(1, L, A)``), int32, int64, float32 or float64:
        the place of each token on each of ``A`` axes.
    frequencies
        ``(R,)`` float32, ``2 R <= D`` and ``R <= 256``, as :func:`rotary_frequencies`
        makes them.
    sections
        The pairs of each axis, ``A`` numbers that add up to ``R``: the first axis turns
        the first ``sections[0]`` pairs, and so on. ``None`` with one axis means ``(R,)``.
    interleaved
        Pairs are features ``(2 j, 2 j + 1)``; otherwise ``(j, j + R)``. Features past
        ``2 R`` pass through.
    backend
        A :class:`Backend` member, or ``None`` for the policy's choice.

    Returns
    -------
    The turned tensor, dense, with the shape and dtype of ``x``.

    Raises
    ------
    TypeError
        If ``backend`` is a raw string or a keyword is unknown.
    ValueError
        If the operands disagree in rank, size, dtype or device.
    NotImplementedError
        If ``positions`` or ``frequencies`` require a gradient, or an operand carries a
        forward-mode tangent.
    NoBackendError
        If no backend can run the call (float64, more than 256 pairs or tokens of more
        than 2^20 elements on the GPU).

    Notes
    -----
    Angles are formed in float64 and reduced to one turn there, so positions keep their
    precision however far they lie; the turn itself is in float32 and rounded once.
    """
    raise NotImplementedError


rotary = Registry("rotary", context_of=_context_of, select=select_backend, describe=_rotary_call)

_SCHEMA = "(Tensor x, Tensor positions, Tensor frequencies, int[] sections, bool interleaved) -> Tensor"


def _public_kernel(x: Tensor, positions: Tensor, frequencies: Tensor, sections: list[int], interleaved: bool) -> Tensor:
    return rotary.run_selected(x, positions, frequencies, sections=sections, interleaved=interleaved)


_PUBLIC = define_public_op("rotary", _SCHEMA, _public_kernel, fixed={2: "frequencies"})


def _route_selected(*args: Any, sections: Sequence[int] | None = None, interleaved: bool = False,
                    **unknown: Any) -> Tensor:
    if unknown:
        raise TypeError(f"rotary got unexpected keyword argument(s): {', '.join(sorted(unknown))}")
    if len(args) != 3 or any(a is None for a in args):  # noqa: PLR2004
        raise TypeError(f"rotary takes (x, positions, frequencies) positionally; got {len(args)} of them")
    x, positions, frequencies = args
    if (not torch.compiler.is_compiling() and isinstance(sections, (tuple, list))
            and all(type(n) is int and n >= 0 for n in sections)):
        direct = rotary.direct(Backend.HIP)
        if direct is not None:
            out = direct(x, positions, frequencies, sections, interleaved)
            if out is not None:
                return out
    if plain_eager(x, positions, frequencies):
        return rotary.run_selected(x, positions, frequencies, sections=sections, interleaved=interleaved)
    check_rotary_call(x, positions, frequencies, sections)
    counts = list(rotary_sections(positions, frequencies, sections))
    if positions.dim() == 2 or positions.shape[0] != x.shape[0]:  # noqa: PLR2004 - a batch axis, as vmap folds it
        positions = positions.expand(x.shape[0], *positions.shape[-2:])
    return _PUBLIC(x, positions, frequencies, counts, interleaved)


rotary.route_selected_calls(_route_selected)
