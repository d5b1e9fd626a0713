"""Layer norm over the last axis, forward and backward, on HIP kernels.

The reference's blocks call ``nn.LayerNorm`` for the token rows of a ViT
(``opentad/models/backbones/vit_sparse_adapter_poguise.py:869-1010``) and for
the query and key rows of the adapter's heads (``:598-606``).
"""
from __future__ import annotations

import torch

from . import opentad_sparse_ops as _ops


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis of
    ``x`` (any leading axes, strides included), mean and variance in float32.

    ``x`` is float16, bfloat16 or float32 with 1 to 8192 channels; the output
    has its dtype, also under autocast (where ``torch`` returns float32).
    ``weight`` and ``bias`` are ``[channels]``, in x's dtype or float32 (any
    other is widened to float32), or None. Their gradients are summed over all
    rows in float32 in a fixed order and rounded once. Differentiable once, in
    reverse mode; a second derivative and forward mode raise."""
    given = [p for p in (weight, bias) if p is not None]
    if any(p.dtype not in (x.dtype, torch.float32) for p in given) or len({p.dtype for p in given}) > 1:
        weight, bias = (None if p is None else p.float() for p in (weight, bias))
        given = [p for p in (weight, bias) if p is not None]
    if torch.is_grad_enabled() and (x.requires_grad or any(p.requires_grad for p in given)):
        return _ops.layer_norm_grad(x, weight, bias, eps)
    return _ops.layer_norm(x, weight, bias, eps, False)[0]
