"""The step that ends a block: its output, dropped, plus the residual."""

from __future__ import annotations

import torch
from torch import Tensor

from ..registry import Backend, dropout

__all__ = ["check_dropout", "drop_and_add"]


def check_dropout(p: float) -> float:
    """``p`` as a layer keeps it; ``ValueError`` outside ``[0, 1]``."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout must lie in [0, 1]; got {p}")
    return float(p)


def drop_and_add(x: Tensor, p: float, *, training: bool, seed: int | Tensor | None, residual: Tensor | None,
                 backend: Backend | None = None) -> Tensor:
    """``x``, dropped with probability ``p`` in training, plus ``residual``.

    ``seed=None`` draws one from torch's CPU generator, which a captured graph could not do
    again at a replay: there the caller passes a tensor.
    """
    if training and p > 0.0:
        if seed is None:
            if x.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("dropout under graph capture needs seed, an int64 tensor that the graph reads at "
                                   "every replay")
            seed = int(torch.randint(2**63 - 1, ()))
        if residual is not None and residual.dtype != x.dtype:  # as the sum without dropout
            wide = torch.promote_types(x.dtype, residual.dtype)
            x, residual = x.to(wide), residual.to(wide)
        return dropout(x, p, seed=seed, residual=residual, backend=backend)
    return x if residual is None else x + residual
