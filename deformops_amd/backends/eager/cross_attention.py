r"""Cross attention on the CPU in torch operators, with the kernels' semantics: sums in
float32 (float64 for float64 operands), zeros and no gradient for a query that no state
is left for, and states that the lengths or a mask of states removes left unread. The
backward is torch autograd."""

from __future__ import annotations

import torch
from torch import Tensor

from ...registry import Backend, CrossAttentionContext, cross_attention
from ...registry.cross_attention import default_scale

__all__ = ["cross_attention_eager"]


def _kept(mask: Tensor | None, key_lengths: Tensor | None, B: int, H: int, Q: int, S: int) -> Tensor | None:  # noqa: N803
    """``(B, S)``: the states that the lengths, or a mask that is one for all queries and
    heads, leave; ``None`` when both leave all."""
    kept = None
    if key_lengths is not None:
        kept = torch.arange(S, device=key_lengths.device) < key_lengths[:, None]
    if mask is not None and mask.dtype == torch.bool:
        full = mask if mask.dim() == 4 else mask[None, None]  # noqa: PLR2004
        if (full.shape[1] == 1 or H == 1) and (full.shape[2] == 1 or Q == 1):
            states = full[:, 0, 0].expand(B, S) if full.shape[2] else None
            if states is not None:
                kept = states if kept is None else kept & states
    return kept


def cross_attention_eager(query: Tensor, key: Tensor, value: Tensor, *, mask: Tensor | None = None,
                          key_lengths: Tensor | None = None, scale: float | None = None) -> Tensor:
    """Run cross attention on the CPU in torch operators."""
    if query.device.type != "cpu":
        raise RuntimeError(f"the eager cross attention backend runs on CPU tensors only; got a tensor on {query.device}")
    B, Q, H, D = query.shape
    S, K = key.shape[1], key.shape[2]
    compute = torch.float64 if query.dtype == torch.float64 else torch.float32
    scale = default_scale(D) if scale is None else float(scale)
    kept = _kept(mask, key_lengths, B, H, Q, S)

    def heads_first(x: Tensor) -> Tensor:  # (B, K, S, D)
        x = x.to(compute)
        if kept is not None:
            x = torch.where(kept[:, :, None, None], x, x.new_zeros(()))
        return x.transpose(1, 2)

    k, v = heads_first(key), heads_first(value)
    # The heads of a group are rows of one list: (B, K, G * Q, D).
    q = query.to(compute).reshape(B, Q, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(B, K, H // K * Q, D)
    scores = torch.matmul(q, k.transpose(2, 3)).reshape(B, H, Q, S) * scale
    off = None
    if mask is not None:
        if mask.dtype == torch.bool:
            off = ~mask
        else:
            scores = scores + mask.to(compute)
            off = mask == -torch.inf
    if kept is not None:
        beyond = ~kept[:, None, None, :]
        off = beyond if off is None else off | beyond
    if off is not None:
        scores = scores.masked_fill(off, -torch.inf)
    if S == 0:
        return query.new_zeros((B, Q, H * D)) + 0 * query.reshape(B, Q, H * D)
    top = scores.detach().amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -torch.inf, torch.zeros_like(top), top))
    total = weights.sum(-1, keepdim=True)
    weights = weights / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.matmul(weights.reshape(B, K, H // K * Q, S), v).reshape(B, H, Q, D)
    return out.transpose(1, 2).reshape(B, Q, H * D).to(query.dtype)


def supports_context(context: CrossAttentionContext) -> bool:
    """CPU tensors of a floating dtype."""
    return context.device.type == "cpu" and context.dtype.is_floating_point


cross_attention.register(Backend.EAGER, cross_attention_eager, supports=supports_context)
