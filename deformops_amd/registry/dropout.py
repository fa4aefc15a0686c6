r"""Dropout whose mask is made again from a counter instead of being stored.

Deformable DETR's and Mask2Former's layers drop every block's output and add the
residual; this is that step as one pass. The reference has no counterpart.
"""

from __future__ import annotations

import dataclasses
from typing import Any

import torch
import torch.library
from torch import Tensor

from ..core.runtime import is_training_from
from ..core.sanitize import check_dropout_call
from ._dispatch import Backend, Registry
from ._eager import plain_eager
from ._public import define_public_op

__all__ = ["DropoutContext", "dropout"]


@dataclasses.dataclass(frozen=True)
class DropoutContext:
    """What backend selection knows of a dropout call."""

    device: torch.device
    dtype: torch.dtype
    is_training: bool


def select_backend(context: DropoutContext) -> list[Backend]:
    """GPU tensors run the HIP kernels and nothing else, CPU tensors the eager backend."""
    return [Backend.HIP] if context.device.type == "cuda" else [Backend.EAGER]


def _context_of(x: Tensor, p: float, *, seed: int | Tensor, offset: int = 0,
                residual: Tensor | None = None) -> DropoutContext:
    check_dropout_call(x, p, seed, offset, residual)
    return DropoutContext(x.device, x.dtype, is_training_from(x, *(() if residual is None else (residual,))))


def _dropout_call(
    x: Tensor,
    p: float,
    /,
    *,
    seed: int | Tensor,
    offset: int = 0,
    residual: Tensor | None = None,
    backend: Backend | None = None,
) -> Tensor:
    r"""Drop elements of ``x`` with probability ``p`` and add ``residual``.

    Element ``i`` (in row-major order) is kept, times ``1 / (1 - p)``, where word ``i %
    4`` of Philox4x32 with 7 rounds, of the counter ``(i // 4, offset)`` and the key
    ``seed``, is at least ``round(p * 2**32)`` (at most ``2**32 - 1``); ``p = 1`` drops
    everything. The mask depends on nothing else: a call with equal numbers drops the
    same elements on every device, and the backward makes it again.

    Parameters
    ----------
    x
        Any shape, float32, float16 or bfloat16 (float64 on the CPU too).
    p
        The probability, in ``[0, 1]``.
    seed
        An integer of 63 bits, or an int64 tensor of one element on ``x``'s device: a
        captured graph reads it at every replay. It has to keep its value until the
        backward has run.
    offset
        A second integer of 63 bits, to give the calls of one step masks of their own.
    residual
        Of ``x``'s shape and dtype, added to the result before its one rounding.
    backend
        A :class:`Backend` member, or ``None`` for the policy's choice.

    Returns
    -------
    A dense tensor with the shape and dtype of ``x``.

    Raises
    ------
    TypeError
        If ``backend`` is a raw string, ``seed`` is neither, or a keyword is unknown.
    ValueError
        If ``p``, ``seed`` or ``offset`` is out of range, or the operands disagree in
        size, dtype or device.
    NotImplementedError
        If an operand carries a forward-mode tangent.
    RuntimeError
        Under vmap: a mapped call's elements have no counters of their own.
    NoBackendError
        If no backend can run the call (float64 on the GPU).
    """
    raise NotImplementedError


dropout = Registry("dropout", context_of=_context_of, select=select_backend, describe=_dropout_call)

_SCHEMA = "(Tensor x, float p, int seed, Tensor? seed_at, int offset, Tensor? residual) -> Tensor"


def _public_kernel(x: Tensor, p: float, seed: int, seed_at: Tensor | None, offset: int,
                   residual: Tensor | None) -> Tensor:
    return dropout.run_selected(x, p, seed=seed if seed_at is None else seed_at, offset=offset, residual=residual)


def _no_vmap(*args: Any, **kwargs: Any) -> Any:  # noqa: ARG001
    raise RuntimeError("dropout cannot be mapped by vmap: the mask counts the elements of one call. Call it on "
                       "the whole tensor.")


_PUBLIC = define_public_op("dropout", _SCHEMA, _public_kernel, vmap=_no_vmap)


def _route_selected(*args: Any, seed: int | Tensor | None = None, offset: int = 0, residual: Tensor | None = None,
                    **unknown: Any) -> Tensor:
    if unknown:
        raise TypeError(f"dropout got unexpected keyword argument(s): {', '.join(sorted(unknown))}")
    if len(args) != 2 or seed is None:  # noqa: PLR2004
        raise TypeError(f"dropout takes (x, p) positionally and the keyword seed; got {len(args)} positional arguments")
    x, p = args
    number, at = (0, seed) if isinstance(seed, Tensor) else (seed, None)
    if not torch.compiler.is_compiling() and type(number) is int and type(offset) is int:
        direct = dropout.direct(Backend.HIP)
        if direct is not None and 0 <= number < 2**63 and 0 <= offset < 2**63 and type(p) in (float, int):
            out = direct(x, p, number, at, offset, residual)
            if out is not None:
                return out
    if plain_eager(x, at, residual):
        return dropout.run_selected(x, p, seed=seed, offset=offset, residual=residual)
    check_dropout_call(x, p, seed, offset, residual)
    return _PUBLIC(x, float(p), number, at, offset, residual)


dropout.route_selected_calls(_route_selected)
