"""The norm over all gradients of a model, and clipping to a limit, on HIP
kernels, without host synchronisation: two launches for every 160 tensors of one
dtype that follow one another (a list that alternates between dtypes takes two for
every run of them).

The reference's training loop clips with ``torch.nn.utils.clip_grad_norm_``
(``opentad/cores/train_engine.py:706-731``).
"""
from __future__ import annotations

import math
from typing import Iterable, Sequence

import torch

from . import opentad_sparse_ops as _ops


def _is_inf(norm_type) -> bool:
    norm_type = float(norm_type)
    if norm_type not in (2.0, math.inf):
        raise ValueError(f"gradient norm: norm_type must be 2 or inf, got {norm_type}")
    return norm_type == math.inf


def grad_norm(grads: Sequence[torch.Tensor], norm_type: float = 2.0, scale: float = 1.0) -> torch.Tensor:
    """``|scale|`` times the 2-norm (or, for ``inf``, the largest magnitude) of
    all elements of ``grads``: a float32 scalar on the GPU."""
    return _ops.grad_clip(grads, None, False, -1.0, scale, _is_inf(norm_type))


def clip_grads(grads: Sequence[torch.Tensor], max_norm: float, norm_type: float = 2.0,
               out: Sequence[torch.Tensor] | None = None, scale: float = 1.0) -> torch.Tensor:
    """Scale ``grads`` by ``scale`` and down to a norm of ``max_norm``: each
    becomes ``g * scale * min(1, max_norm / (norm + 1e-6))``, in place or in
    ``out`` (tensors of the same shapes, of any of the dtypes). Returns the norm
    before clipping (of the scaled gradients), a float32 scalar on the GPU.

    ``grads`` is a sequence of float16, bfloat16 or float32 tensors on one GPU;
    ``scale`` removes a loss scale in the same pass. Norms are summed in float64
    over all tensors, in a fixed order. A gradient that is listed twice counts and
    is scaled once per mention; a tensor of ``out`` shares no memory with another
    tensor. A norm of NaN makes every gradient NaN
    and an infinite one zeros and NaN, as ``torch`` has it."""
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"clip_grads: max_norm must not be negative, got {max_norm}")
    return _ops.grad_clip(grads, out, True, max_norm, scale, _is_inf(norm_type))


def clip_grad_norm_(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_`` for norm types 2 and inf: clips the
    ``grad`` of every parameter in place by their common norm and returns it.
    ``error_if_nonfinite`` reads the norm back before anything is scaled."""
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad for p in params if p.grad is not None]
    if not grads:
        _is_inf(norm_type)
        return torch.tensor(0.0)
    if error_if_nonfinite and not math.isfinite(norm := grad_norm(grads, norm_type).item()):
        raise RuntimeError(f"The total norm of order {float(norm_type)} for gradients from `parameters` is non-finite "
                           f"({norm}), so it cannot be clipped.")
    return clip_grads(grads, max_norm, norm_type)
