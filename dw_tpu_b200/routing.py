"""Top-k routing on B200, as fused_moe_func computes it for the GMM path
(E0901:656-687; weights cast to the activation dtype, X0101:131)."""

from __future__ import annotations

import torch

from . import _lib as L
from . import ops


def route_topk(gating_output: torch.Tensor, top_k: int, renormalize: bool = True,
               scoring_fn: str = "sigmoid", dtype: torch.dtype = torch.bfloat16,
               bias: torch.Tensor | None = None, num_valid_tokens: int | None = None):
    """Returns (topk_weights in ``dtype``, topk_ids int32) like
    ``_fused_moe_fp4_routing``: scores in f32, ties to the lower expert index,
    bias for selection only, renormalised, rows >= num_valid_tokens -> expert
    0 with weight 0."""
    logits = gating_output.contiguous()
    if logits.dtype not in (torch.bfloat16, torch.float32):
        logits = logits.float()
    t = logits.shape[0]
    ids = torch.empty((t, top_k), dtype=torch.int32, device=logits.device)
    w32 = torch.empty((t, top_k), dtype=torch.float32, device=logits.device)
    w16 = (torch.empty((t, top_k), dtype=torch.bfloat16, device=logits.device)
           if dtype == torch.bfloat16 else None)
    ops.route_topk_out(logits, top_k, ids, w32_out=w32, w16_out=w16, scoring_fn=scoring_fn,
                       renormalize=renormalize,
                       bias=None if bias is None else bias.float().contiguous(),
                       num_valid_tokens=num_valid_tokens)
    if dtype == torch.bfloat16:
        return w16, ids
    return w32.to(dtype), ids


def route_grouped_topk(gating_output: torch.Tensor, top_k: int, num_groups: int,
                       topk_groups: int, renormalize: bool = True, scoring_fn: str = "sigmoid",
                       group_score: str = "top2", routed_scale: float = 1.0,
                       dtype: torch.dtype = torch.bfloat16, bias: torch.Tensor | None = None,
                       num_valid_tokens: int | None = None):
    """Group-limited ``route_topk``: (topk_weights in ``dtype``, topk_ids int32).

    The experts are ``num_groups`` (at most 32) groups of consecutive ones; the
    ``topk_groups`` best groups stay open and the ``top_k`` best experts are
    chosen in them, best first, ties to the lower index. An expert's choice
    value is its score plus ``bias`` (the balance bias, taken in f32: selection
    only; without one the experts are in their logits' order), a group's the
    best choice in it (``group_score="max"``) or the sum of its two best
    ("top2"). The weights are the scores, divided by their sum if
    ``renormalize``, times ``routed_scale``. Selection is that of 64-bit scores
    whatever the logits' dtype (f64 logits take several times as long).
    Inference only: no gradient."""
    logits = gating_output
    if logits.dtype not in L.FLOATS and logits.dtype is not torch.float64:
        # f32 holds the 16- and 8-bit floats whole, f64 the integers.
        logits = logits.float() if logits.is_floating_point() else logits.double()
    if bias is not None and (bias.dtype is not torch.float32 or not bias.is_contiguous()):
        bias = bias.float().contiguous()
    w_ids = ops.route_grouped_topk_new(logits, top_k, num_groups, topk_groups,
                                       L.FLOATS.get(dtype, L.F32), scoring_fn, group_score,
                                       renormalize, routed_scale, bias, num_valid_tokens)
    return w_ids if dtype in L.FLOATS else (w_ids[0].to(dtype), w_ids[1])


def route_hash(gating_output: torch.Tensor, hash_ids: torch.Tensor, renormalize: bool = True,
               scoring_fn: str = "sigmoid", dtype: torch.dtype = torch.bfloat16,
               num_valid_tokens: int | None = None):
    """Hash routing of ``_fused_moe_fp4_routing`` (E0901:667-671): the ids
    are ``hash_ids`` [t, top_k]; the weights are the scores at those ids,
    renormalised, padding rows -> expert 0 with weight 0."""
    logits = gating_output.contiguous()
    if logits.dtype not in (torch.bfloat16, torch.float32):
        logits = logits.float()
    t, top_k = hash_ids.shape
    ids = torch.empty((t, top_k), dtype=torch.int32, device=logits.device)
    w32 = torch.empty((t, top_k), dtype=torch.float32, device=logits.device)
    ops.route_hash_out(logits, hash_ids.to(torch.int32).contiguous(), ids, w32,
                       scoring_fn=scoring_fn, renormalize=renormalize,
                       num_valid_tokens=num_valid_tokens)
    return w32.to(dtype), ids


def dedupe_topk(topk_weights: torch.Tensor, topk_ids: torch.Tensor, num_experts: int):
    """E0901:98-121: makes each token's expert ids distinct. Returns new
    (f32 weights, int32 ids)."""
    w = topk_weights.float().contiguous().clone()
    ids = topk_ids.to(torch.int32).contiguous().clone()
    ops.dedupe_topk_(w, ids, num_experts)
    return w, ids
