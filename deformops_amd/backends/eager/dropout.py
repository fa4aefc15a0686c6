r"""Dropout on the CPU in torch operators, with the mask the GPU kernel makes. The backward
is torch autograd."""

from __future__ import annotations

import torch
from torch import Tensor

from ...registry import Backend, DropoutContext, dropout

__all__ = ["dropout_eager", "kept_elements"]

_WORD = 0xFFFFFFFF


def kept_elements(elements: int, p: float, seed: Tensor, offset: int) -> Tensor:
    """Which of ``elements`` are kept: words of Philox4x32 with 7 rounds (Salmon, Moraes,
    Dror and Shaw, SC 2011) of the counter ``(element // 4, offset)`` and the key ``seed``
    (an int64 tensor) against ``p``. Products of two 32-bit words wrap modulo 2^64 in
    int64, and the masked shift takes their high word."""
    block = torch.arange((elements + 3) // 4, dtype=torch.int64, device=seed.device)
    high = torch.full_like(block, offset >> 32)
    state = [block & _WORD, block >> 32, torch.full_like(block, offset & _WORD), high]
    seed = seed.reshape(())
    key = [seed & _WORD, (seed >> 32) & _WORD]
    for _ in range(7):
        a, b = state[0] * 0xD2511F53, state[2] * 0xCD9E8D57
        state = [((b >> 32) & _WORD) ^ state[1] ^ key[0], b & _WORD, ((a >> 32) & _WORD) ^ state[3] ^ key[1], a & _WORD]
        key = [(key[0] + 0x9E3779B9) & _WORD, (key[1] + 0xBB67AE85) & _WORD]
    return torch.stack(state, -1).reshape(-1)[:elements] >= min(round(p * 2**32), _WORD)


def dropout_eager(x: Tensor, p: float, *, seed: int | Tensor, offset: int = 0, residual: Tensor | None = None) -> Tensor:
    """Run dropout on the CPU in torch operators."""
    if x.device.type != "cpu":
        raise RuntimeError(f"the eager dropout backend runs on CPU tensors only; got a tensor on {x.device}")
    compute = torch.float64 if x.dtype == torch.float64 else torch.float32
    if p == 1:
        keep, scale = torch.zeros(x.shape, dtype=torch.bool), 0.0
    else:
        key = seed if isinstance(seed, Tensor) else torch.tensor(seed, dtype=torch.int64)
        keep, scale = kept_elements(x.numel(), p, key, offset).reshape(x.shape), 1.0 / (1.0 - p)
    wide = x.to(compute)
    out = torch.where(keep, wide * scale, wide.new_zeros(()))
    if residual is not None:
        out = out + residual.to(compute)
    return out.to(x.dtype)


def supports_context(context: DropoutContext) -> bool:
    """CPU tensors of a floating dtype."""
    return context.device.type == "cpu" and context.dtype.is_floating_point


dropout.register(Backend.EAGER, dropout_eager, supports=supports_context)
