"""Layers over the operators (reference ``sources/deformops/nn/__init__.py``)."""

from __future__ import annotations

from .cross_attention import CrossAttention
from .msda import MSDAMethod, MultiScaleDeformAttn2d

__all__ = ["CrossAttention", "MSDAMethod", "MultiScaleDeformAttn2d"]
