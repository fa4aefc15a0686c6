"""Operand validation for the operators' entry points.

The contract is the reference's (sources/deformops/core/sanitize.py:56-146 for the
layer sizes, :276-436 for a call): a malformed call raises ``ValueError`` naming
the operand at fault, before any kernel launches, and reads tensor metadata only;
the level-table contents are read back to the host only when ``DEFORMOPS_VALIDATE``
is set, since that synchronizes the stream and breaks graph capture.

The structural check here is one pass of shape unification. Each operand has a
pattern over the symbols B (batch), S (positions), H (heads), D (channels), Q
(queries), L (levels) and P (points); a symbol is bound by the first operand that
has it and every later occurrence must agree. The HIP kernels treat a level whose
table entry does not fit the value tensor as empty, so a malformed table yields
zeros, never an out-of-bounds access, when the value checks are off.
"""

from __future__ import annotations

import math
import os
from typing import TYPE_CHECKING, Any

if TYPE_CHECKING:
    from collections.abc import Sequence

    from torch import Tensor

__all__ = [
    "VALIDATE_ENV_VAR",
    "check_2power",
    "check_cross_attention_call",
    "check_divisible",
    "check_dropout_call",
    "check_msda_call",
    "check_msda_params",
    "check_positive",
    "check_rotary_call",
    "rotary_sections",
    "value_checks_enabled",
]

#: Enables the level-table checks; any value but a falsy spelling turns them on.
VALIDATE_ENV_VAR = "DEFORMOPS_VALIDATE"


def value_checks_enabled() -> bool:
    """Whether the checks that read the level table back to the host run (off by default)."""
    return os.getenv(VALIDATE_ENV_VAR, "0").strip().lower() not in {"", "0", "false", "no", "off"}


# Layer sizes.


def check_positive(n: int, name: str) -> None:
    """``ValueError`` unless ``n`` is a positive integer."""
    if not n > 0:
        raise ValueError(f"{name} must be a positive integer; got {n}")


def check_divisible(a: int, b: int) -> None:
    """``ValueError`` unless ``b`` is non-zero and divides ``a``."""
    if b == 0 or a % b:
        raise ValueError(f"{a} is not divisible by {b}")


def check_2power(n: int) -> None:
    """``ValueError`` unless ``n`` is a positive power of 2."""
    if n <= 0 or n & (n - 1):
        raise ValueError(f"expected a positive power of 2; got {n}")


def check_msda_params(dim: int, num_heads: int, num_levels: int, num_points: int) -> None:
    """The integers that size an MSDA layer: all positive, ``dim`` split evenly over heads."""
    for name, n in (("dim", dim), ("num_heads", num_heads), ("num_levels", num_levels),
                    ("num_points", num_points)):
        check_positive(n, name)
    check_divisible(dim, num_heads)


# One call.

#: Axis patterns of the five operands: symbols bind on first sight, integers are
#: fixed sizes. attention_weights takes either pattern.
_PATTERNS: tuple[tuple[str, tuple[tuple[str | int, ...], ...]], ...] = (
    ("value", (("B", "S", "H", "D"),)),
    ("spatial_shapes", (("L", 2),)),
    ("level_start_index", (("L",),)),
    ("sampling_locations", (("B", "Q", "H", "L", "P", 2),)),
    ("attention_weights", (("B", "Q", "H", "LP"), ("B", "Q", "H", "L", "P"))),
)

_MEANING = {
    "B": "the batch of value",
    "H": "the heads of value",
    "L": "the levels (rows of spatial_shapes)",
    "Q": "the queries of sampling_locations",
    "P": "the points of sampling_locations",
    "LP": "levels x points of sampling_locations",
}


def _unify(name: str, shape: tuple[int, ...], patterns: tuple[tuple[str | int, ...], ...],
           bound: dict[str, int]) -> None:
    """Match ``shape`` to the pattern of its rank; bind new symbols, check old ones."""
    pattern = next((p for p in patterns if len(p) == len(shape)), None)
    if pattern is None:
        ranks = " or ".join(str(len(p)) for p in patterns)
        raise ValueError(f"{name} must have {ranks} dimensions; got shape {tuple(shape)}")
    for axis, (symbol, size) in enumerate(zip(pattern, shape)):
        if isinstance(symbol, int):
            want, why = symbol, "its fixed size"
        elif symbol in bound:
            want, why = bound[symbol], _MEANING.get(symbol, symbol)
        else:
            bound[symbol] = size
            continue
        if size != want:
            raise ValueError(
                f"{name} has {size} entries on axis {axis} where {want} are expected "
                f"({why}); its shape is {tuple(shape)}"
            )


def check_msda_call(
    value: Tensor,
    spatial_shapes: Tensor,
    level_start_index: Tensor,
    sampling_locations: Tensor,
    attention_weights: Tensor,
) -> None:
    """Validate the five MSDA operands; ``ValueError`` names the first operand at fault.

    value ``(B, S, H, D)`` floating; spatial_shapes ``(L, 2)`` and level_start_index
    ``(L,)`` integer; sampling_locations ``(B, Q, H, L, P, 2)`` floating;
    attention_weights ``(B, Q, H, L * P)`` or ``(B, Q, H, L, P)`` in value's dtype;
    one device for all.
    """
    operands = (value, spatial_shapes, level_start_index, sampling_locations, attention_weights)
    bound: dict[str, int] = {}
    for (name, patterns), tensor in zip(_PATTERNS, operands):
        if name == "attention_weights" and "L" in bound and "P" in bound:
            bound["LP"] = bound["L"] * bound["P"]
        _unify(name, tuple(tensor.shape), patterns, bound)

    for (name, _), tensor in zip(_PATTERNS, operands):
        integral = name in ("spatial_shapes", "level_start_index")
        if integral and (tensor.is_floating_point() or tensor.is_complex()):
            raise ValueError(f"{name} indexes the value tensor and must be integer; got {tensor.dtype}")
        if not integral and not tensor.is_floating_point():
            raise ValueError(f"{name} must be floating point; got {tensor.dtype}")
    if attention_weights.dtype != value.dtype:
        raise ValueError(
            f"attention_weights is {attention_weights.dtype} while value is {value.dtype}; "
            f"give both one dtype (or run the call under autocast)"
        )
    devices = {tensor.device for tensor in operands}
    if len(devices) > 1:
        where = ", ".join(f"{name} on {t.device}" for (name, _), t in zip(_PATTERNS, operands))
        raise ValueError(f"the operands must share one device; got {where}")

    if value_checks_enabled() and _readable(spatial_shapes, level_start_index):
        _check_level_table(value, spatial_shapes, level_start_index)


def _readable(*tensors: Tensor) -> bool:
    """Whether the tensors hold data the host can read: not traced, fake or meta."""
    import torch  # noqa: PLC0415
    from torch._subclasses.fake_tensor import is_fake  # noqa: PLC0415

    if torch.compiler.is_compiling():
        return False
    return all(t.device.type != "meta" and not is_fake(t) for t in tensors)


def _check_level_table(value: Tensor, spatial_shapes: Tensor, level_start_index: Tensor) -> None:
    """The levels are non-empty, laid end to end from 0, and exactly fill value's S axis."""
    sizes = [(int(h), int(w)) for h, w in spatial_shapes.detach().cpu().tolist()]
    starts = [int(s) for s in level_start_index.detach().cpu().tolist()]
    empty = [i for i, (h, w) in enumerate(sizes) if h <= 0 or w <= 0]
    if empty:
        raise ValueError(f"spatial_shapes has an empty level at row {empty[0]}: {sizes[empty[0]]}")
    offsets = [0]
    for h, w in sizes:
        offsets.append(offsets[-1] + h * w)
    if starts != offsets[:-1]:
        raise ValueError(
            f"level_start_index is {starts}, but levels of sizes {[h * w for h, w in sizes]} laid end "
            f"to end start at {offsets[:-1]}"
        )
    if offsets[-1] != value.shape[1]:
        raise ValueError(
            f"spatial_shapes covers {offsets[-1]} positions but value has {value.shape[1]} on its "
            f"spatial axis"
        )


# The operators beside MSDA.


def _check_tensor(name: str, value: Any) -> None:
    import torch  # noqa: PLC0415

    if not isinstance(value, torch.Tensor):
        raise TypeError(f"{name} must be a tensor; got {type(value).__name__}")


def _same_device(**tensors: Tensor | None) -> None:
    given = {name: t for name, t in tensors.items() if t is not None}
    if len({t.device for t in given.values()}) > 1:
        where = ", ".join(f"{name} on {t.device}" for name, t in given.items())
        raise ValueError(f"the operands must share one device; got {where}")


def _floating(**tensors: Tensor) -> None:
    """All floating and of the first one's dtype."""
    first, dtype = None, None
    for name, t in tensors.items():
        if not t.is_floating_point():
            raise ValueError(f"{name} must be floating point; got {t.dtype}")
        if dtype is None:
            first, dtype = name, t.dtype
        elif t.dtype != dtype:
            raise ValueError(f"{name} is {t.dtype} while {first} is {dtype}; give both one dtype")


def _no_gradient(name: str, t: Tensor | None) -> None:
    import torch  # noqa: PLC0415

    if t is not None and t.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"{name} gets no gradient from this operator; detach it")


def check_cross_attention_call(query: Tensor, key: Tensor, value: Tensor, mask: Tensor | None,
                               key_lengths: Tensor | None, scale: float | None) -> None:
    """Validate the operands of a cross attention call; the error names the one at fault.

    query ``(B, Q, H, D)``, key and value ``(B, S, K, D)`` of one floating dtype, ``H`` a
    multiple of ``K``; mask boolean or floating, ``(Q, S)`` or 4 axes that broadcast to
    ``(B, H, Q, S)``; key_lengths ``(B,)`` integer; scale positive and finite.
    """
    import torch  # noqa: PLC0415

    for name, t in (("query", query), ("key", key), ("value", value)):
        _check_tensor(name, t)
        if t.dim() != 4:  # noqa: PLR2004
            raise ValueError(f"{name} must have 4 dimensions; got shape {tuple(t.shape)}")
    B, Q, H, D = query.shape
    _, S, K, _ = key.shape
    if key.shape[0] != B or key.shape[3] != D:
        raise ValueError(f"key has batch {key.shape[0]} and {key.shape[3]} channels where query has {B} and {D}")
    if value.shape != key.shape:
        raise ValueError(f"value has shape {tuple(value.shape)} where key has {tuple(key.shape)}")
    if D == 0 or H == 0 or K == 0:
        raise ValueError(f"query and key must have heads and channels; got {H} and {K} heads of {D} channels")
    if H % K:
        raise ValueError(f"query has {H} heads, which is not a multiple of the {K} heads of key")
    _floating(query=query, key=key, value=value)
    if mask is not None:
        _check_tensor("mask", mask)
        if mask.dtype != torch.bool and mask.dtype not in (torch.float32, torch.float16, torch.bfloat16, query.dtype):
            raise ValueError(f"mask must be bool, float32, float16 or bfloat16; got {mask.dtype}")
        full = (B, H, Q, S)
        if mask.dim() not in (2, 4) or any(n not in (1, m) for n, m in zip(mask.shape[::-1], full[::-1])):
            raise ValueError(f"mask must have 2 or 4 dimensions that broadcast to {full}; got shape {tuple(mask.shape)}")
        _no_gradient("mask", mask)
    if key_lengths is not None:
        _check_tensor("key_lengths", key_lengths)
        if key_lengths.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"key_lengths must be int64 or int32; got {key_lengths.dtype}")
        if tuple(key_lengths.shape) != (B,):
            raise ValueError(f"key_lengths must have one entry for each of {B} images; got shape "
                             f"{tuple(key_lengths.shape)}")
    # The kernels hold the scale in float32, where 1e-50 is 0.
    if scale is not None and not (math.isfinite(scale) and 2.0**-149 <= scale <= 3.4028234663852886e38):
        raise ValueError(f"scale must be positive and finite (in float32); got {scale}")
    _same_device(query=query, key=key, value=value, mask=mask, key_lengths=key_lengths)


def rotary_sections(positions: Tensor, frequencies: Tensor, sections: Sequence[int] | None) -> tuple[int, ...]:
    """``sections`` of a rotary call; one axis takes every pair when it is ``None``."""
    if sections is None:
        if positions.shape[-1] != 1:
            raise ValueError(f"sections are needed: positions have {positions.shape[-1]} axes")
        return (int(frequencies.shape[0]),)
    counts = tuple(sections)
    if any(not isinstance(n, int) or n < 0 for n in counts):
        raise ValueError(f"sections must be integers, none negative; got {counts}")
    return counts


def check_rotary_call(x: Tensor, positions: Tensor, frequencies: Tensor, sections: Sequence[int] | None) -> None:
    """Validate the operands of a rotary call; the error names the one at fault.

    x ``(B, L, H, D)`` floating; positions ``(L, A)``, ``(B, L, A)`` or ``(1, L, A)`` of
    int32, int64, float32 or float64; frequencies ``(R,)`` float32 with ``2 R <= D``;
    sections ``A`` counts that add up to ``R``.
    """
    import torch  # noqa: PLC0415

    for name, t in (("x", x), ("positions", positions), ("frequencies", frequencies)):
        _check_tensor(name, t)
    if x.dim() != 4:  # noqa: PLR2004
        raise ValueError(f"x must have 4 dimensions; got shape {tuple(x.shape)}")
    _floating(x=x)
    B, L, _, D = x.shape
    if positions.dim() not in (2, 3) or positions.shape[-2] != L or (
            positions.dim() == 3 and positions.shape[0] not in (1, B)):  # noqa: PLR2004
        raise ValueError(f"positions must be ({L}, axes) or ({B}, {L}, axes); got shape {tuple(positions.shape)}")
    if positions.dtype not in (torch.int32, torch.int64, torch.float32, torch.float64):
        raise ValueError(f"positions must be int32, int64, float32 or float64; got {positions.dtype}")
    if frequencies.dim() != 1 or frequencies.dtype != torch.float32:
        raise ValueError(f"frequencies must be one float32 axis; got {frequencies.dtype} of shape "
                         f"{tuple(frequencies.shape)}")
    counts = rotary_sections(positions, frequencies, sections)
    R = frequencies.shape[0]
    if not counts or len(counts) != positions.shape[-1] or sum(counts) != R:
        raise ValueError(f"sections must give {positions.shape[-1]} axes (at least one) {R} pairs together; got {counts}")
    if len(counts) > 255:  # noqa: PLR2004
        raise ValueError(f"positions must have at most 255 axes; got {len(counts)}")
    if 2 * R > D:
        raise ValueError(f"frequencies turn {2 * R} features where x has {D}")
    _no_gradient("positions", positions)
    _no_gradient("frequencies", frequencies)
    _same_device(x=x, positions=positions, frequencies=frequencies)


def check_dropout_call(x: Tensor, p: float, seed: int | Tensor, offset: int, residual: Tensor | None) -> None:
    """Validate the operands of a dropout call; the error names the one at fault."""
    import torch  # noqa: PLC0415

    _check_tensor("x", x)
    _floating(x=x)
    if isinstance(p, bool) or not isinstance(p, (int, float)):
        raise TypeError(f"p must be a number; got {type(p).__name__}")
    if not 0 <= p <= 1:
        raise ValueError(f"p must lie in [0, 1]; got {p}")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ValueError(f"seed must be one int64; got {seed.dtype} of shape {tuple(seed.shape)}")
    elif isinstance(seed, bool) or not isinstance(seed, int):
        raise TypeError(f"seed must be an integer or an int64 tensor; got {type(seed).__name__}")
    elif not 0 <= seed < 2**63:
        raise ValueError(f"seed must be in [0, 2^63); got {seed}")
    if isinstance(offset, bool) or not isinstance(offset, int):
        raise TypeError(f"offset must be an integer; got {type(offset).__name__}")
    if not 0 <= offset < 2**63:
        raise ValueError(f"offset must be in [0, 2^63); got {offset}")
    if residual is not None:
        _check_tensor("residual", residual)
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"residual is {residual.dtype} of shape {tuple(residual.shape)} where x is {x.dtype} of "
                             f"shape {tuple(x.shape)}")
    _same_device(x=x, residual=residual, seed=seed if isinstance(seed, torch.Tensor) else None)
