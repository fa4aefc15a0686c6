r"""Registry adapter of the HIP rotary kernels, and their private operator:

    deformops_hip::rotary(x, positions, frequencies, sections, interleaved, inverse) -> y

whose gradient is the same operator with ``inverse`` turned.
"""

from __future__ import annotations

from collections.abc import Sequence
from typing import Any

import torch
import torch.library
from torch import Tensor

from ...core.sanitize import rotary_sections
from ...registry import Backend, RotaryContext, rotary
from ...registry._eager import plain_eager
from . import _native
from ._bridge import NAMESPACE
from .cross_attention import load

__all__ = ["rotary_hip", "supports_context"]

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
_LIBRARY = torch.library.Library(NAMESPACE, "FRAGMENT")
_LIBRARY.define("rotary(Tensor x, Tensor positions, Tensor frequencies, int[] sections, bool interleaved, "
                "bool inverse) -> Tensor")


def _apply(x: Tensor, positions: Tensor, frequencies: Tensor, sections: Sequence[int], interleaved: bool,
           inverse: bool) -> Tensor:
    return _native.load().rotary_apply(x, positions, frequencies, list(sections), interleaved, inverse)


_LIBRARY.impl("rotary", _apply, "CUDA")


@torch.library.register_fake(f"{NAMESPACE}::rotary", lib=_LIBRARY)
def _fake(x, positions, frequencies, sections, interleaved, inverse):  # noqa: ANN001, ANN202, ARG001, PLR0913
    return x.new_empty(x.shape)


_op = torch.ops.deformops_hip.rotary.default


def _setup_context(ctx, inputs, output):  # noqa: ANN001, ANN202, ARG001
    _, positions, frequencies, sections, interleaved, inverse = inputs
    ctx.save_for_backward(positions, frequencies)
    ctx.options = (sections, interleaved, not inverse)


@torch.autograd.function.once_differentiable
def _autograd(ctx, grad_output):  # noqa: ANN001, ANN202
    positions, frequencies = ctx.saved_tensors
    return _op(grad_output, positions, frequencies, *ctx.options), None, None, None, None, None


torch.library.register_autograd(f"{NAMESPACE}::rotary", _autograd, setup_context=_setup_context, lib=_LIBRARY)


def rotary_hip(x: Tensor, positions: Tensor, frequencies: Tensor, *, sections: Sequence[int] | None = None,
               interleaved: bool = False) -> Tensor:
    """Run the rotary positions on the gfx950 HIP kernels."""
    counts = list(rotary_sections(positions, frequencies, sections))
    if plain_eager(x, positions, frequencies):
        return _native.load().rotary(x, positions, frequencies, counts, interleaved)
    return _op(x, positions, frequencies, counts, interleaved, False)


def supports_context(context: RotaryContext) -> bool:
    """GPU tensors of at most 256 pairs, in tokens of at most 2^20 elements."""
    return (context.device.type == "cuda" and torch.version.hip is not None and context.dtype in _DTYPES
            and context.num_pairs <= 256 and context.row_elements <= 2**20)  # noqa: PLR2004


def direct(*args: Any) -> Any:
    """A plain eager GPU call that the native bridge can check by itself, or ``None``;
    also ``None`` until ``load`` has loaded the bridge."""
    native = _native.loaded()
    return None if native is None else native.try_rotary(*args)


if torch.cuda.is_available() and torch.version.hip is not None:
    rotary.register(Backend.HIP, rotary_hip, supports=supports_context, load=load, direct=direct)
else:
    rotary.mark_unavailable(Backend.HIP, "no ROCm GPU is available to this process")
