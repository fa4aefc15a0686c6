r"""Registry adapter of the HIP dropout kernel, and its private operator:

    deformops_hip::dropout(x, p, seed, seed_at, offset, residual) -> y

whose gradient for ``x`` is the same operator on the output's gradient, without a
residual.
"""

from __future__ import annotations

from typing import Any

import torch
import torch.library
from torch import Tensor

from ...registry import Backend, DropoutContext, dropout
from ...registry._eager import plain_eager
from . import _native
from ._bridge import NAMESPACE
from .cross_attention import load

__all__ = ["dropout_hip", "supports_context"]

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
_LIBRARY = torch.library.Library(NAMESPACE, "FRAGMENT")
_LIBRARY.define("dropout(Tensor x, float p, int seed, Tensor? seed_at, int offset, Tensor? residual) -> Tensor")


def _apply(x: Tensor, p: float, seed: int, seed_at: Tensor | None, offset: int, residual: Tensor | None) -> Tensor:
    return _native.load().dropout_apply(x, p, seed, seed_at, offset, residual)


_LIBRARY.impl("dropout", _apply, "CUDA")


@torch.library.register_fake(f"{NAMESPACE}::dropout", lib=_LIBRARY)
def _fake(x, p, seed, seed_at, offset, residual):  # noqa: ANN001, ANN202, ARG001, PLR0913
    return x.new_empty(x.shape)


_op = torch.ops.deformops_hip.dropout.default


def _setup_context(ctx, inputs, output):  # noqa: ANN001, ANN202, ARG001
    _, p, seed, seed_at, offset, _ = inputs
    ctx.save_for_backward(seed_at)
    ctx.options = (p, seed, offset)


@torch.autograd.function.once_differentiable
def _autograd(ctx, grad_output):  # noqa: ANN001, ANN202
    p, seed, offset = ctx.options
    (seed_at,) = ctx.saved_tensors
    grad_x = _op(grad_output, p, seed, seed_at, offset, None) if ctx.needs_input_grad[0] else None
    return grad_x, None, None, None, None, grad_output if ctx.needs_input_grad[5] else None


torch.library.register_autograd(f"{NAMESPACE}::dropout", _autograd, setup_context=_setup_context, lib=_LIBRARY)


def dropout_hip(x: Tensor, p: float, *, seed: int | Tensor, offset: int = 0, residual: Tensor | None = None) -> Tensor:
    """Run dropout on the gfx950 HIP kernel."""
    number, at = (0, seed) if isinstance(seed, Tensor) else (seed, None)
    if plain_eager(x, at, residual):
        return _native.load().dropout(x, float(p), number, at, offset, residual)
    return _op(x, float(p), number, at, offset, residual)


def supports_context(context: DropoutContext) -> bool:
    """GPU tensors of float32, float16 or bfloat16."""
    return context.device.type == "cuda" and torch.version.hip is not None and context.dtype in _DTYPES


def direct(*args: Any) -> Any:
    """A plain eager GPU call that the native bridge can check by itself, or ``None``;
    also ``None`` until ``load`` has loaded the bridge."""
    native = _native.loaded()
    return None if native is None else native.try_dropout(*args)


if torch.cuda.is_available() and torch.version.hip is not None:
    dropout.register(Backend.HIP, dropout_hip, supports=supports_context, load=load, direct=direct)
else:
    dropout.mark_unavailable(Backend.HIP, "no ROCm GPU is available to this process")
