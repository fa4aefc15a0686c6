r"""Registry adapter of the HIP cross attention kernels, and their private operators:

    deformops_hip::cross_attention_forward(query, key, value, mask, key_lengths, scale)
        -> (out, row_stats)
    deformops_hip::cross_attention_backward(..., out, row_stats, grad_output)
        -> (grad_query, grad_key, grad_value)

Plain eager calls take the native autograd node (csrc/bridge_operators.cpp); traced,
compiled, exported and fake calls take the operators.
"""

from __future__ import annotations

from typing import Any

import torch
import torch.library
from torch import Tensor

from ...registry import Backend, CrossAttentionContext, cross_attention
from ...registry._eager import plain_eager
from ...registry.cross_attention import default_scale
from . import _lib, _native
from ._bridge import NAMESPACE

__all__ = ["cross_attention_hip", "supports_context"]

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
_LIBRARY = torch.library.Library(NAMESPACE, "FRAGMENT")
_OPERANDS = "Tensor query, Tensor key, Tensor value, Tensor? mask, Tensor? key_lengths, float scale"

_LIBRARY.define(f"cross_attention_forward({_OPERANDS}) -> (Tensor, Tensor)")
_LIBRARY.define(f"cross_attention_backward({_OPERANDS}, Tensor out, Tensor row_stats, Tensor grad_output) "
                "-> (Tensor, Tensor, Tensor)")


def _forward(query: Tensor, key: Tensor, value: Tensor, mask: Tensor | None, key_lengths: Tensor | None,
             scale: float) -> tuple[Tensor, Tensor]:
    return _native.load().cross_attention_forward(query, key, value, mask, key_lengths, scale, True)


def _backward(query: Tensor, key: Tensor, value: Tensor, mask: Tensor | None,  # noqa: PLR0913
              key_lengths: Tensor | None, scale: float, out: Tensor, row_stats: Tensor,
              grad_output: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    return _native.load().cross_attention_backward(query, key, value, mask, key_lengths, scale, out, row_stats,
                                                   grad_output)


_LIBRARY.impl("cross_attention_forward", _forward, "CUDA")
_LIBRARY.impl("cross_attention_backward", _backward, "CUDA")


@torch.library.register_fake(f"{NAMESPACE}::cross_attention_forward", lib=_LIBRARY)
def _forward_fake(query, key, value, mask, key_lengths, scale):  # noqa: ANN001, ANN202, ARG001
    B, Q, H, D = query.shape
    return query.new_empty((B, Q, H * D)), query.new_empty((B * H * Q, 2), dtype=torch.float32)


@torch.library.register_fake(f"{NAMESPACE}::cross_attention_backward", lib=_LIBRARY)
def _backward_fake(query, key, value, mask, key_lengths, scale, out, row_stats, grad_output):  # noqa: ANN001, ANN202, ARG001, PLR0913
    return query.new_empty(query.shape), key.new_empty(key.shape), value.new_empty(value.shape)


_forward_op = torch.ops.deformops_hip.cross_attention_forward.default
_backward_op = torch.ops.deformops_hip.cross_attention_backward.default


def _setup_context(ctx, inputs, output):  # noqa: ANN001, ANN202
    query, key, value, mask, key_lengths, scale = inputs
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(query, key, value, mask, key_lengths, *output)
    ctx.scale = scale


@torch.autograd.function.once_differentiable
def _autograd(ctx, grad_output, _grad_stats):  # noqa: ANN001, ANN202
    query, key, value, mask, key_lengths, out, stats = ctx.saved_tensors
    grads = _backward_op(query, key, value, mask, key_lengths, ctx.scale, out, stats, grad_output)
    return *grads, None, None, None


torch.library.register_autograd(f"{NAMESPACE}::cross_attention_forward", _autograd, setup_context=_setup_context,
                                lib=_LIBRARY)


def cross_attention_hip(query: Tensor, key: Tensor, value: Tensor, *, mask: Tensor | None = None,
                        key_lengths: Tensor | None = None, scale: float | None = None) -> Tensor:
    """Run cross attention on the gfx950 HIP kernels."""
    scale = default_scale(query.shape[3]) if scale is None else float(scale)
    if plain_eager(query, key, value, mask, key_lengths):
        return _native.load().cross_attention(query, key, value, mask, key_lengths, scale)
    return _forward_op(query, key, value, mask, key_lengths, scale)[0]


def supports_context(context: CrossAttentionContext) -> bool:
    """GPU tensors of a type the matrix cores sum in float32, heads of at most 128 channels."""
    return (context.device.type == "cuda" and torch.version.hip is not None and context.dtype in _DTYPES
            and context.head_dim <= 128)  # noqa: PLR2004


def load(*, download: bool | None = None, compile: bool | str | None = None) -> str:  # noqa: A002
    """Load libdeformops_amd.so and its native bridge; return the library's path."""
    path = str(_lib.load(download=download, compile=compile).path)
    _native.load(download=download, compile=compile)
    return path


def direct(*args: Any) -> Any:
    """A plain eager GPU call that the native bridge can check by itself, or ``None``;
    also ``None`` until ``load`` has loaded the bridge."""
    native = _native.loaded()
    return None if native is None else native.try_cross_attention(*args)


if torch.cuda.is_available() and torch.version.hip is not None:
    cross_attention.register(Backend.HIP, cross_attention_hip, supports=supports_context, load=load, direct=direct)
else:
    cross_attention.mark_unavailable(Backend.HIP, "no ROCm GPU is available to this process")
