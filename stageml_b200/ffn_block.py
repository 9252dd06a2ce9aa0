"""The feed-forward sublayer of a decoder block around the routed experts.

One call runs what stands between a block's attention and the next block:

    ids, weights = router(normed)                           (ops.route_topk)
    y = SwiGLU experts on block-scaled e4m3 weights          (ops.moe_forward_blocks)
    residual' = residual_scale * residual + gate * post_norm(y)
    normed'   = next_pre_weight * rms_norm(residual')        (ops.norm_residual, one pass)

and, for router training, the balance loss with its counts (``balance``). Weights are quantized
once, when the module is built. Tenants with LoRA adapters stay with ``ops.moe_forward``.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops


class _Route(torch.autograd.Function):
    """ops.route_topk (ids, renormalised weights, logits) with the gradients of its weights and logits."""

    @staticmethod
    def forward(ctx, rows, router_w, k):
        ctx.set_materialize_grads(False)
        ids, weights, logits = ops.route_topk(rows, router_w, k)
        ctx.save_for_backward(rows, router_w, ids, weights)
        ctx.mark_non_differentiable(ids)
        return ids, weights, logits

    @staticmethod
    @once_differentiable
    def backward(ctx, _ids, d_weights, d_logits):
        rows, router_w, ids, weights = ctx.saved_tensors
        if d_weights is not None:  # a softmax over the chosen logits
            d = weights * (d_weights - (d_weights * weights).sum(1, keepdim=True))
            chosen = d.new_zeros(d.shape[0], router_w.shape[0]).scatter_(1, ids.long(), d)
            d_logits = chosen if d_logits is None else d_logits + chosen
        if d_logits is None:
            return None, None, None
        d_rows = (d_logits @ router_w).to(rows.dtype) if ctx.needs_input_grad[0] else None
        d_router_w = d_logits.t() @ rows.float() if ctx.needs_input_grad[1] else None
        return d_rows, d_router_w, None


class FeedForwardBlock(torch.nn.Module):
    """Router, block-scaled experts, post norm, gate, residual sum and the next block's pre norm.

    router_w [E, H] float32; gate_up [E + n_shared, 2I, H] (rows [:I] the SiLU branch) and down
    [E + n_shared, H, I] in float32, bfloat16 or float16; H and I multiples of 16. post_weight [H], gate
    [H] and pre_weight [H] are optional (no norm, gate 1, no norm). balance_coefficient scales the loss
    of ``balance``.
    """

    def __init__(self, router_w, gate_up, down, k: int, *, n_shared: int = 0, pre_weight=None, post_weight=None,
                 gate=None, residual_scale: float = 1.0, balance_coefficient: float = 0.01, eps: float = 1e-6):
        super().__init__()
        if gate_up.dim() != 3 or down.dim() != 3 or gate_up.shape[0] != down.shape[0]:
            raise ValueError("FeedForwardBlock: gate_up [E, 2I, H] and down [E, H, I]")
        if router_w.shape != (gate_up.shape[0] - n_shared, gate_up.shape[2]):
            raise ValueError(f"FeedForwardBlock: router_w {tuple(router_w.shape)} does not match "
                             f"{gate_up.shape[0] - n_shared} experts of width {gate_up.shape[2]}")
        self.k, self.n_shared = int(k), int(n_shared)
        self.residual_scale, self.balance_coefficient, self.eps = residual_scale, balance_coefficient, eps
        self.router_w = torch.nn.Parameter(router_w.detach().float().contiguous())
        with torch.no_grad():
            codes = [ops.quantize_e4m3_blocks(w, tiles=True) for w in (gate_up, down)]
        self.gate_up, self.gate_up_scale = codes[0]
        self.down, self.down_scale = codes[1]
        for name, w in (("pre_weight", pre_weight), ("post_weight", post_weight), ("gate", gate)):
            self.register_parameter(name, None if w is None else torch.nn.Parameter(w.detach().clone()))

    def start(self, x):
        """(residual, normed) of the stack's first block: x and its pre norm."""
        return x, ops.norm_residual(None, x, pre_weight=self.pre_weight, eps=self.eps)[1]

    def experts(self, normed):
        """The routed experts' output for normed [..., H]."""
        rows = normed.detach().reshape(-1, normed.shape[-1])
        ids, weights, _ = ops.route_topk(rows, self.router_w.detach(), self.k)
        y = ops.moe_forward_blocks(rows, self.gate_up, self.gate_up_scale, self.down, self.down_scale, topk_ids=ids,
                                   topk_weights=weights, n_shared=self.n_shared)
        return y.view(normed.shape)

    def forward(self, residual, normed, next_pre_weight=None):
        """-> (residual', normed') with next_pre_weight (the next block's pre norm), else (residual',).

        Gradients reach the residual stream, the norms' weights and the gate; the experts are frozen.
        """
        return ops.norm_residual(self.experts(normed), residual, post_weight=self.post_weight, gate=self.gate,
                                 residual_scale=self.residual_scale, pre_weight=next_pre_weight, eps=self.eps)

    def balance(self, normed, valid=None):
        """The router's balance loss on normed [..., H] -> (loss, counts per expert, tokens); differentiable in
        router_w and normed. The counts are of the experts that ``experts`` runs for the same rows."""
        rows = normed.reshape(-1, normed.shape[-1]).contiguous()
        ids, _, logits = _Route.apply(rows, self.router_w, self.k)
        return ops.balance_loss(logits, ids, self.balance_coefficient, valid=valid)


__all__ = ["FeedForwardBlock"]
