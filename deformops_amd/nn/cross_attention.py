"""Attention of a decoder's queries over an encoder's states, with rotary positions and
dropout: :data:`~deformops_amd.registry.rotary`, :data:`~deformops_amd.registry.cross_attention`
and :data:`~deformops_amd.registry.dropout` as one layer. The reference has no counterpart.
"""

from __future__ import annotations

from collections.abc import Sequence

from torch import Tensor, nn

from ..core.sanitize import check_divisible, check_positive
from ..registry import Backend, cross_attention, rotary, rotary_frequencies
from ._dropout import check_dropout, drop_and_add

__all__ = ["CrossAttention"]


class CrossAttention(nn.Module):
    r"""Multi-head attention of queries over states of another length.

    Queries, keys and values are linear maps of the two inputs. With ``rotary_sections``,
    queries and keys turn by their places (:func:`~deformops_amd.registry.rotary`), so
    that a score depends on the places' difference on every axis. The heads are projected
    out, dropped in training, and added to the residual.

    Parameters
    ----------
    dim
        Query and hidden width, split evenly over the heads.
    dim_context
        Width of the encoder's states; ``None`` means ``dim``.
    dim_output
        Output width; ``None`` means ``dim``.
    num_heads
        Query heads.
    num_key_heads
        Heads of the keys and values, a divisor of ``num_heads``; ``None`` means as many.
    rotary_sections
        Turned pairs of features of each position axis, at most half of a head's channels
        together; ``None`` turns nothing.
    rotary_base
        The ladder's base (:func:`~deformops_amd.registry.rotary_frequencies`).
    dropout
        Probability with which the output's elements are dropped in training.
    bias
        Whether the projections have biases.
    backend
        A :class:`~deformops_amd.registry.Backend` member, or ``None`` for the registry's
        choice.

    Raises
    ------
    ValueError
        If a size is not positive, heads do not divide evenly, the sections turn more
        than a head, or ``dropout`` is out of range.
    """

    def __init__(
        self,
        dim: int,
        dim_context: int | None = None,
        dim_output: int | None = None,
        *,
        num_heads: int,
        num_key_heads: int | None = None,
        rotary_sections: Sequence[int] | None = None,
        rotary_base: float = 10000.0,
        dropout: float = 0.0,
        bias: bool = True,
        backend: Backend | None = None,
    ) -> None:
        super().__init__()
        key_heads = num_heads if num_key_heads is None else num_key_heads
        for name, n in (("dim", dim), ("num_heads", num_heads), ("num_key_heads", key_heads)):
            check_positive(n, name)
        check_divisible(dim, num_heads)
        check_divisible(num_heads, key_heads)
        self.dim = dim
        self.num_heads = num_heads
        self.num_key_heads = key_heads
        self.head_dim = dim // num_heads
        self.dropout = check_dropout(dropout)
        self.backend = backend
        self.rotary_sections = None if rotary_sections is None else tuple(rotary_sections)
        if self.rotary_sections is not None:
            if any(n < 0 for n in self.rotary_sections) or 2 * sum(self.rotary_sections) > self.head_dim:
                raise ValueError(f"rotary_sections {self.rotary_sections} turn more than the {self.head_dim} channels "
                                 f"of a head, or are negative")
            self.register_buffer("frequencies", rotary_frequencies(self.rotary_sections, base=rotary_base),
                                 persistent=False)
        self.proj_query = nn.Linear(dim, dim, bias=bias)
        self.proj_key = nn.Linear(dim_context or dim, key_heads * self.head_dim, bias=bias)
        self.proj_value = nn.Linear(dim_context or dim, key_heads * self.head_dim, bias=bias)
        self.proj_output = nn.Linear(dim, dim_output or dim, bias=bias)

    def _turned(self, x: Tensor, positions: Tensor | None, name: str) -> Tensor:
        if self.rotary_sections is None:
            if positions is not None:
                raise ValueError(f"{name} are given to a layer without rotary_sections")
            return x
        if positions is None:
            raise ValueError(f"{name} are needed: the layer turns {self.rotary_sections} pairs")
        # Module.to(dtype) narrows every floating buffer; the angles keep float32.
        return rotary(x, positions, self.frequencies.float(), sections=self.rotary_sections, backend=self.backend)

    def states(self, context: Tensor, context_positions: Tensor | None = None) -> tuple[Tensor, Tensor]:
        """The keys and values ``(B, S, num_key_heads, head_dim)`` of ``context`` ``(B, S,
        dim_context)``: what a decoder computes once and passes to every step."""
        B, S, _ = context.shape
        shape = (B, S, self.num_key_heads, self.head_dim)
        key = self._turned(self.proj_key(context).view(shape), context_positions, "context_positions")
        return key, self.proj_value(context).view(shape)

    def forward(  # noqa: PLR0913
        self,
        q: Tensor,
        context: Tensor | tuple[Tensor, Tensor],
        *,
        positions: Tensor | None = None,
        context_positions: Tensor | None = None,
        mask: Tensor | None = None,
        key_lengths: Tensor | None = None,
        residual: Tensor | None = None,
        seed: int | Tensor | None = None,
    ) -> Tensor:
        """Attend ``context`` from ``q``.

        Parameters
        ----------
        q
            Queries ``(B, Q, dim)``.
        context
            The encoder's states ``(B, S, dim_context)``, or what :meth:`states` made of
            them.
        positions, context_positions
            Places of the queries and of the states, ``(Q, axes)`` or ``(B, Q, axes)``;
            needed with ``rotary_sections`` (``context_positions`` not with ready states).
        mask, key_lengths
            As :data:`~deformops_amd.registry.cross_attention` takes them.
        residual
            ``(B, Q, dim_output)``, added to the result; or ``None``.
        seed
            The dropout's seed (:data:`~deformops_amd.registry.dropout`); ``None`` draws
            one from torch's CPU generator.

        Returns
        -------
        ``(B, Q, dim_output)``.
        """
        B, Q, _ = q.shape
        if isinstance(context, tuple):
            if context_positions is not None:
                raise ValueError("context_positions are given with states that are ready")
            key, value = context
        else:
            key, value = self.states(context, context_positions)
        query = self._turned(self.proj_query(q).view(B, Q, self.num_heads, self.head_dim), positions, "positions")
        out = cross_attention(query, key, value, mask=mask, key_lengths=key_lengths, backend=self.backend)
        return drop_and_add(self.proj_output(out), self.dropout, training=self.training, seed=seed, residual=residual,
                            backend=self.backend)

    def extra_repr(self) -> str:
        return (f"dim={self.dim}, num_heads={self.num_heads}, num_key_heads={self.num_key_heads}, "
                f"rotary_sections={self.rotary_sections}, dropout={self.dropout}")
