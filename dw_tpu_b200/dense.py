"""Dense products of the MoE block on B200: the router's logits and the shared
expert's projections, with bias, activation and residual in the epilogue."""

from __future__ import annotations

import torch

from . import _lib as L
from .ops import code_of

_ACTS = {None: L.ACT_NONE, "silu": L.ACT_SILU, "gelu": L.ACT_GELU,
         "gelu_tanh": L.ACT_GELU_TANH, "swiglu": L.ACT_SWIGLU,
         "swiglu_clamp": L.ACT_SWIGLU_CLAMP}


def dense_matmul(x: torch.Tensor, w: torch.Tensor, *, bias: torch.Tensor | None = None,
                 act: str | None = None, act_limit: float | None = None,
                 residual: torch.Tensor | None = None, residual_scale: float = 1.0,
                 out_dtype: torch.dtype | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """``residual_scale * residual + act(x @ w.T + bias)``, rounded once.

    x bf16 [m, k]; w bf16 [n, k] (a Linear layer's layout); k a multiple of 8,
    rows of both on 16 bytes. ``act``: None, "silu", "gelu" (erf), "gelu_tanh",
    each element by itself, or "swiglu" / "swiglu_clamp" on the [gate | up]
    halves of n (then the result has n / 2 columns; the clamp is gate <=
    ``act_limit``, |up| <= ``act_limit``). Note that ``gmm_v2``'s ``fuse_act``
    calls SwiGLU "silu". bias [n], residual and the result [m, n or n / 2] are
    bf16 or f32; ``out_dtype`` is bf16 by default. ``out`` (which may be
    ``residual``) is written and returned if given. Inference only: no
    gradient."""
    code = _ACTS.get(act, -1)
    if code < 0:
        raise ValueError(f"act {act!r} not supported (one of {sorted(k for k in _ACTS if k)})")
    if code == L.ACT_SWIGLU_CLAMP and act_limit is None:
        raise ValueError("swiglu_clamp needs act_limit")
    if out is not None and out_dtype is not None and out.dtype != out_dtype:
        raise ValueError(f"out is {out.dtype}, out_dtype {out_dtype}")
    return L.bind().dense_matmul(x, w, bias, code, act_limit or 0.0, residual, residual_scale, out,
                                 code_of(L.FLOATS, out_dtype or torch.bfloat16, "out_dtype"), None)
