r"""Cross attention: queries over an encoder's states of another length.

The dense neighbour of MSDA in a decoder (Mask2Former's masked attention over one
level, DETR's over the whole memory, a caption's token over its image's states). The
call goes the way an ``msda`` call goes: checked here, sent to the policy's backend,
through ``torch.ops.deformops.cross_attention`` where something watches the call. The
reference has no counterpart.
"""

from __future__ import annotations

import dataclasses
import math
from typing import Any

import torch
from torch import Tensor

from ..core.runtime import is_training_from
from ..core.sanitize import check_cross_attention_call
from ._dispatch import Backend, Registry
from ._eager import plain_eager
from ._public import define_public_op

__all__ = ["CrossAttentionContext", "cross_attention", "default_scale"]


def default_scale(head_dim: int) -> float:
    """The factor of the scores for ``scale=None``."""
    return 1.0 / math.sqrt(head_dim)


@dataclasses.dataclass(frozen=True)
class CrossAttentionContext:
    """What backend selection knows of a cross attention call."""

    device: torch.device
    dtype: torch.dtype
    head_dim: int
    is_training: bool


def select_backend(context: CrossAttentionContext) -> list[Backend]:
    """GPU tensors run the HIP kernels and nothing else, CPU tensors the eager backend."""
    return [Backend.HIP] if context.device.type == "cuda" else [Backend.EAGER]


def _context_of(query: Tensor, key: Tensor, value: Tensor, *, mask: Tensor | None = None,
                key_lengths: Tensor | None = None, scale: float | None = None) -> CrossAttentionContext:
    check_cross_attention_call(query, key, value, mask, key_lengths, scale)
    return CrossAttentionContext(query.device, query.dtype, int(query.shape[3]), is_training_from(query, key, value))


def _cross_attention_call(
    query: Tensor,
    key: Tensor,
    value: Tensor,
    /,
    *,
    mask: Tensor | None = None,
    key_lengths: Tensor | None = None,
    scale: float | None = None,
    backend: Backend | None = None,
) -> Tensor:
    r"""Softmax attention of queries over states of another length.

    ``B`` batch, ``Q`` queries, ``S`` states, ``H`` heads, ``K`` key heads (``H`` is a
    multiple of ``K``; heads ``h`` of a group of ``H / K`` share key head ``h // (H /
    K)``), ``D`` channels per head (at most 128 on the GPU). The operands may have any
    memory layout, and ``Q = 1`` is a single token's step over cached states.

    Parameters
    ----------
    query
        ``(B, Q, H, D)``, float32, float16 or bfloat16 (float64 on the CPU too).
    key, value
        ``(B, S, K, D)``, with the dtype of ``query``.
    mask
        ``(Q, S)`` or 4 axes that broadcast to ``(B, H, Q, S)``. Boolean: ``True`` where
        the query attends the state. Floating (float32, float16, bfloat16): added to the
        scaled scores, ``-inf`` removing the state. It gets no gradient.
    key_lengths
        ``(B,)`` integer: the states of each image; those at or past it are not read.
        Values are clamped to ``[0, S]``.
    scale
        Factor of the scores, positive; ``None`` means ``D ** -0.5``.
    backend
        A :class:`Backend` member, or ``None`` for the policy's choice.

    Returns
    -------
    ``(B, Q, H * D)`` in the dtype of ``query``. A query that no state is left for gets
    zeros, and neither gives nor takes a gradient.

    Raises
    ------
    TypeError
        If ``backend`` is a raw string or a keyword is unknown.
    ValueError
        If the operands disagree in rank, size, dtype or device, or ``scale`` is not
        positive and finite.
    NotImplementedError
        If ``mask`` requires a gradient, or an operand carries a forward-mode tangent.
    NoBackendError
        If no backend can run the call (float64 or more than 128 channels on the GPU).

    Notes
    -----
    Scores, softmax and every sum are in float32. 16-bit products are exact in it;
    float32 products are formed on the GPU of three bfloat16 parts each, to 2^-23 of
    their size, and an attended infinity, or a value past bfloat16's range (3.39e38),
    gives NaN there. The weights and their gradients are rounded to a 16-bit operands'
    type before the second products. Equal calls give equal bits. States that
    ``key_lengths`` removes, or a boolean mask of shape ``(.., 1, 1, S)``, may hold
    anything, NaN included; states that a mask removes from some queries only, or a
    floating mask removes, must be finite, as in the formula.
    """
    raise NotImplementedError


cross_attention = Registry("cross_attention", context_of=_context_of, select=select_backend,
                           describe=_cross_attention_call)

_SCHEMA = ("(Tensor query, Tensor key, Tensor value, Tensor? mask, Tensor? key_lengths, float scale) -> Tensor")


def _public_kernel(query: Tensor, key: Tensor, value: Tensor, mask: Tensor | None, key_lengths: Tensor | None,
                   scale: float) -> Tensor:
    return cross_attention.run_selected(query, key, value, mask=mask, key_lengths=key_lengths, scale=scale)


_PUBLIC = define_public_op("cross_attention", _SCHEMA, _public_kernel)


def _route_selected(*args: Any, mask: Tensor | None = None, key_lengths: Tensor | None = None,
                    scale: float | None = None, **unknown: Any) -> Tensor:
    if unknown:
        raise TypeError(f"cross_attention got unexpected keyword argument(s): {', '.join(sorted(unknown))}")
    if len(args) != 3 or any(a is None for a in args):  # noqa: PLR2004
        raise TypeError(f"cross_attention takes (query, key, value) positionally; got {len(args)} of them")
    if not torch.compiler.is_compiling() and (scale is None or (type(scale) in (float, int) and scale != 0)):
        direct = cross_attention.direct(Backend.HIP)
        if direct is not None:
            out = direct(*args, mask, key_lengths, 0.0 if scale is None else scale)
            if out is not None:
                return out
    query, key, value = args
    if plain_eager(query, key, value, mask, key_lengths):
        return cross_attention.run_selected(query, key, value, mask=mask, key_lengths=key_lengths, scale=scale)
    check_cross_attention_call(query, key, value, mask, key_lengths, scale)
    if mask is not None:  # a batch axis of its own, as vmap folds it
        mask = mask.expand(query.shape[0], query.shape[2], query.shape[1], key.shape[1])
    return _PUBLIC(query, key, value, mask, key_lengths, default_scale(query.shape[3]) if scale is None else float(scale))


cross_attention.route_selected_calls(_route_selected)
