"""A transformer block's MoE half on one device, around ``MoELayer``:

    h = norm(x)                                  pre_norm
    logits = h Wr^T                              dense_matmul, f32
    ids, w = group-limited top-k of the logits   route_grouped_topk
    y = sum_k w_k expert_k(h)                    MoELayer.experts (FP4)
      + shared expert(h)                         dense_matmul x 2 (SwiGLU; y added in the second)
    x' = residual_scale x + scale gate norm(y)   post_norm, with the next block's
    h' = norm(x')                                norm in the same pass
"""

from __future__ import annotations

import torch

from .block_norm import post_norm, pre_norm
from .dense import dense_matmul
from .fused_moe import MoELayer
from . import ops


class MoEBlock:
    """The block over ``layer`` (its weights, top_k, scoring_fn, renormalize,
    SwiGLU limit and workspace), all other weights bf16 on its device:

    router [E, H]; norm_weight [H] of the norm before the block; shared_w13
    [2 I, H] = [gate | up] and shared_w2 [H, I], both or neither; post_weight
    [H] of a norm of the block's output (none without it); next_weight [H] of
    the norm before the next block (then ``forward`` returns h'). router_bias
    f32 [E] is the balance bias (selection only). One block serves one sequence
    of calls at a time, like its layer."""

    def __init__(self, layer: MoELayer, router: torch.Tensor, norm_weight: torch.Tensor, *,
                 num_groups: int = 1, topk_groups: int = 1, group_score: str = "top2",
                 routed_scale: float = 1.0, router_bias: torch.Tensor | None = None,
                 shared_w13: torch.Tensor | None = None, shared_w2: torch.Tensor | None = None,
                 post_weight: torch.Tensor | None = None,
                 next_weight: torch.Tensor | None = None, scale: float = 1.0,
                 residual_scale: float = 1.0, eps: float = 1e-6, kind: str = "rms"):
        e, h = layer.w.num_experts, layer.w.hidden_size
        if router.shape != (e, h):
            raise ValueError(f"router must be [{e}, {h}], got {list(router.shape)}")
        if (shared_w13 is None) != (shared_w2 is None):
            raise ValueError("shared_w13 and shared_w2 go together")
        if shared_w13 is not None and (
                shared_w13.dim() != 2 or shared_w2.dim() != 2 or shared_w13.shape[1] != h or
                shared_w2.shape != (h, shared_w13.shape[0] // 2) or shared_w13.shape[0] % 2):
            raise ValueError(f"shared_w13 must be [2 I, {h}] and shared_w2 [{h}, I]")
        self.layer = layer
        self.router, self.router_bias = router, router_bias
        self.norm_weight, self.post_weight, self.next_weight = norm_weight, post_weight, next_weight
        self.shared_w13, self.shared_w2 = shared_w13, shared_w2
        self.num_groups, self.topk_groups, self.group_score = num_groups, topk_groups, group_score
        self.routed_scale = routed_scale
        self.scale, self.residual_scale, self.eps, self.kind = scale, residual_scale, eps, kind
        t, dev = layer.max_tokens, router.device
        self.h = torch.empty((t, h), dtype=torch.bfloat16, device=dev)
        self.logits = torch.empty((t, e), dtype=torch.float32, device=dev)
        # With a shared expert the routed sum is added to it in f32.
        self.routed = torch.empty((t, h), device=dev,
                                  dtype=torch.bfloat16 if shared_w13 is None else torch.float32)
        if shared_w13 is not None:
            self.s1 = torch.empty((t, shared_w13.shape[0] // 2), dtype=torch.bfloat16, device=dev)
            self.y = torch.empty((t, h), dtype=torch.bfloat16, device=dev)

    def forward(self, x: torch.Tensor, h: torch.Tensor | None = None,
                gate: torch.Tensor | None = None, num_valid_tokens: int | None = None,
                out: torch.Tensor | None = None):
        """x [t, H] (bf16 or f32): the residual stream; h: its norm where the
        block before has formed it already; gate as in ``post_norm`` (bf16).
        Returns (x' in x's dtype, h' or None); ``out`` may be x (in place).
        Tokens from ``num_valid_tokens`` on get no routed expert."""
        t, layer = x.shape[0], self.layer
        if t > layer.max_tokens:
            raise ValueError(f"{t} tokens exceed max_tokens={layer.max_tokens}")
        if h is None:
            h = pre_norm(x, self.norm_weight, eps=self.eps, kind=self.kind, out=self.h[:t])
        elif h.shape != x.shape or h.dtype != torch.bfloat16 or not h.is_contiguous():
            raise ValueError("h must be a contiguous bf16 tensor of x's shape")
        logits = dense_matmul(h, self.router, out=self.logits[:t])
        ids, w16 = layer.ids[:t], layer.w16[:t]
        ops.route_grouped_topk_out(logits, layer.top_k, self.num_groups, self.topk_groups, ids,
                                   w16_out=w16, scoring_fn=layer.scoring_fn,
                                   group_score=self.group_score, renormalize=layer.renormalize,
                                   routed_scale=self.routed_scale, bias=self.router_bias,
                                   num_valid_tokens=num_valid_tokens)
        y = self.routed[:t]
        if t:
            layer.experts(h, ids, w16, y)
        if self.shared_w13 is not None:
            clamp = layer.act_limit > 0.0
            s1 = dense_matmul(h, self.shared_w13, act="swiglu_clamp" if clamp else "swiglu",
                              act_limit=layer.act_limit, out=self.s1[:t])
            y = dense_matmul(s1, self.shared_w2, residual=y, out=self.y[:t])
        return post_norm(y, x, norm_weight=self.post_weight, gate=gate, scale=self.scale,
                         residual_scale=self.residual_scale, next_weight=self.next_weight,
                         eps=self.eps, kind=self.kind, residual_out=out)

    __call__ = forward
