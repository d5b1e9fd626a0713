"""Attention of queries to the tokens of another sequence, on HIP kernels.

Action queries of a decoder, key tokens or the tokens of one window attend to
the kept tokens of an encoder, whose number differs between samples. The
reference evaluates such attention with ``F.scaled_dot_product_attention``
(``opentad/models/backbones/vit_sparse_adapter_poguise.py:607-640``).
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from . import opentad_sparse_ops as _ops
from .adapter import _is_plain
from .layer_norm import layer_norm


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, key_lengths: torch.Tensor | None = None,
                    key_mask: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """``softmax(scale q k^T) v`` of ``q [B, Nq, H, D]`` over ``k, v [B, Nk, KH,
    D]``; the result is ``[B, Nq, H, D]``.

    ``H`` is a multiple of ``KH``: query head ``h`` reads key head ``h // (H //
    KH)``. ``D`` is 1 to 128, the dtype float16, bfloat16 or float32; any
    strides (a last axis that is strided is copied), any token counts, 0
    included. Sample ``b`` sees its first ``key_lengths[b]`` tokens (int32 or
    int64 ``[B]`` on the GPU) where ``key_mask[b]`` (bool ``[B, Nk]``) is true;
    a query that sees none gives zeros and no gradient, and what unseen tokens
    hold, infinities and NaN included, reaches no result. ``scale`` defaults to
    ``D ** -0.5`` and must be positive.

    Softmax statistics and sums are float32; probabilities and score gradients
    are rounded to the inputs' dtype as operands of the matrix units (scaled by
    powers of two in float16, so that small ones keep their bits). For the
    backward the call keeps its result, in 16 bits a second tensor like it (what
    the result's rounding took), and 4 bytes per query and head. Gradients come without
    atomics: equal inputs give equal bits. Differentiable once, in reverse mode;
    a second derivative and forward mode raise."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if key_lengths is not None and key_lengths.dtype == torch.int64:
        key_lengths = key_lengths.clamp(0, k.shape[1]).to(torch.int32)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _ops.cross_attention_grad(q, k, v, key_lengths, key_mask, scale)
    return _ops.cross_attention(q, k, v, key_lengths, key_mask, scale, False)[0]


class CrossAttention(nn.Module):
    """Pre-norm cross attention with a residual: ``x + proj(attention(norm(x),
    context))``, with per-head norms of queries and keys as the adapter's
    attention has them.

    ``x [B, Nq, embed_dims]``, ``context [B, Nk, context_dims]`` (``embed_dims``
    by default). ``kv_heads`` below ``num_heads`` shares key heads. For serving,
    ``project_context`` gives the keys and values once per context, and
    ``forward(x, kv=...)`` attends to them token by token."""

    def __init__(self, embed_dims: int, num_heads: int, context_dims: int | None = None, kv_heads: int | None = None,
                 eps: float = 1e-6):
        super().__init__()
        kv_heads = num_heads if kv_heads is None else kv_heads
        if embed_dims % num_heads or num_heads % kv_heads:
            raise ValueError(f"CrossAttention: {embed_dims} channels, {num_heads} heads and {kv_heads} key heads do not divide")
        self.num_heads, self.kv_heads, self.head_dim = num_heads, kv_heads, embed_dims // num_heads
        if self.head_dim > 128:
            raise ValueError(f"CrossAttention: a head dimension of {self.head_dim} (at most 128)")
        context_dims = embed_dims if context_dims is None else context_dims
        self.norm = nn.LayerNorm(embed_dims, eps=eps)
        self.context_norm = nn.LayerNorm(context_dims, eps=eps)
        self.q_norm = nn.LayerNorm(self.head_dim, eps=eps)
        self.k_norm = nn.LayerNorm(self.head_dim, eps=eps)
        self.q = nn.Linear(embed_dims, embed_dims)
        self.kv = nn.Linear(context_dims, 2 * kv_heads * self.head_dim)
        self.proj = nn.Linear(embed_dims, embed_dims)

    @staticmethod
    def _norm(layer, x):
        """The layer's norm in x's dtype. A layer whose call does more than compute
        it, or another layer in its place, is called."""
        if _is_plain(layer, nn.LayerNorm) and layer.normalized_shape == x.shape[-1:]:
            return layer_norm(x, layer.weight, layer.bias, layer.eps)
        return layer(x).to(x.dtype)

    def project_context(self, context: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys (normalised) and values ``[B, Nk, kv_heads, head_dim]`` of a context."""
        kv = self.kv(self._norm(self.context_norm, context)).unflatten(-1, (2, self.kv_heads, self.head_dim))
        return self._norm(self.k_norm, kv[:, :, 0]), kv[:, :, 1]

    def forward(self, x: torch.Tensor, context: torch.Tensor | None = None, key_lengths: torch.Tensor | None = None,
                key_mask: torch.Tensor | None = None, kv: tuple[torch.Tensor, torch.Tensor] | None = None) -> torch.Tensor:
        if (context is None) == (kv is None):
            raise ValueError("CrossAttention: give either context or kv")
        k, v = self.project_context(context) if kv is None else kv
        q = self.q(self._norm(self.norm, x)).unflatten(-1, (self.num_heads, self.head_dim))
        out = cross_attention(self._norm(self.q_norm, q), k, v, key_lengths, key_mask, 1.0 / math.sqrt(self.head_dim))
        return x + self.proj(out.flatten(2))
