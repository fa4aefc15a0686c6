"""Operator dispatch: the operators' registries, their call contexts and the public operators.

Import through this package, as with the reference::

    from deformops_amd.registry import Backend, msda

``cross_attention``, ``rotary`` and ``dropout`` are what a decoder around MSDA needs next to it.
"""

from __future__ import annotations

from ..core.runtime import resolve_method
from ._dispatch import Backend, LoadedBackend, Registry, Resolution
from .cross_attention import CrossAttentionContext, cross_attention
from .dropout import DropoutContext, dropout
from .msda import (
    MSDABackend,
    MSDAContext,
    MSDAMethod,
    apply_msda_method,
    msda,
    msda_method_to_aggregate,
    resolve_msda_attn,
    select_backend,
)
from .rotary import RotaryContext, rotary, rotary_frequencies

__all__ = [
    "Backend",
    "CrossAttentionContext",
    "DropoutContext",
    "LoadedBackend",
    "MSDABackend",
    "MSDAContext",
    "MSDAMethod",
    "Registry",
    "Resolution",
    "RotaryContext",
    "apply_msda_method",
    "cross_attention",
    "dropout",
    "msda",
    "msda_method_to_aggregate",
    "resolve_method",
    "resolve_msda_attn",
    "rotary",
    "rotary_frequencies",
    "select_backend",
]
