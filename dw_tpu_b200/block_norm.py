"""The norms before and after a block on B200, fused with the block's gate, its
scale and the residual's scale."""

from __future__ import annotations

import torch

from . import _lib as L
from .ops import NORMS, code_of


def pre_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
             eps: float = 1e-6, kind: str = "rms", out_dtype: torch.dtype = torch.bfloat16,
             out: torch.Tensor | None = None) -> torch.Tensor:
    """The norm before a block: ``norm(x) * weight (+ bias)`` of x [t, h] (bf16
    or f32), ``kind`` "rms" or "layer"; statistics in f32. ``out`` (which may
    be ``x``) is written and returned if given. Inference only: no gradient."""
    if weight is None:
        raise ValueError("pre_norm needs a weight")
    return L.bind().block_norm(x, None, None, None, None, 1.0, 1.0, weight, bias, eps,
                               code_of(NORMS, kind, "norm kind"), None, out,
                               code_of(L.FLOATS, out_dtype, "out_dtype"), True, None)[1]


def post_norm(y: torch.Tensor, residual: torch.Tensor, *,
              norm_weight: torch.Tensor | None = None, norm_bias: torch.Tensor | None = None,
              gate: torch.Tensor | None = None, scale: float = 1.0, residual_scale: float = 1.0,
              next_weight: torch.Tensor | None = None, next_bias: torch.Tensor | None = None,
              eps: float = 1e-6, kind: str = "rms", out_dtype: torch.dtype = torch.bfloat16,
              residual_out: torch.Tensor | None = None, out: torch.Tensor | None = None):
    """After a block with output y [t, h], in one pass:

        r = residual_scale * residual + scale * gate * norm(y)
        h = norm(r)

    Returns (r in residual's dtype, h in ``out_dtype``). norm(y) has
    ``norm_weight`` / ``norm_bias`` and is y itself without a weight; h has
    ``next_weight`` / ``next_bias`` (the next block's ``pre_norm``) and is None
    without a weight. gate (y's dtype): one value a token [t, 1], a channel
    [h], or an element [t, h]. h is formed from the f32 r. ``residual_out`` may be
    ``residual`` (the stream updated in place) and ``out`` may be ``y``.
    Inference only: no gradient."""
    if next_weight is None and (out is not None or next_bias is not None):
        raise ValueError("out and next_bias need next_weight")
    if y is None:
        raise ValueError("post_norm needs y")
    return L.bind().block_norm(residual, y, norm_weight, norm_bias, gate, scale, residual_scale,
                               next_weight, next_bias, eps, code_of(NORMS, kind, "norm kind"),
                               residual_out, out, code_of(L.FLOATS, out_dtype, "out_dtype"),
                               next_weight is not None, None)
