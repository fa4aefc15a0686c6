"""Whether a call would be observed by anything but autograd."""

from __future__ import annotations

import torch
from torch import Tensor

__all__ = ["plain_eager"]


def plain_eager(*tensors: Tensor | None) -> bool:
    """Real tensors, no compiling or tracing, no dispatch or function mode (fake tensors,
    export), and no functorch transform (vmap, grad) around any of them."""
    if torch.compiler.is_compiling() or torch._C._len_torch_dispatch_stack():  # noqa: SLF001
        return False
    if torch._C._get_tracing_state() is not None:  # noqa: SLF001
        return False
    if torch._C._is_torch_function_mode_enabled():  # noqa: SLF001
        return False
    wrapped = torch._C._functorch.is_functorch_wrapped_tensor  # noqa: SLF001
    return all(t is None or (type(t) in (Tensor, torch.nn.Parameter) and not wrapped(t)) for t in tensors)
