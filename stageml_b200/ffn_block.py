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

from . import ops
from .ops import differentiable_once


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
    @differentiable_once
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


def _row_values(x):
    """x [rows, cols] as its codes hold it, fp32."""
    q, scale = ops.quantize_e4m3_blocks(x)
    return q.float() * scale.repeat_interleave(128, 1)[:, : x.shape[1]]


def _tile_values(q, scale):
    """A matrix of codes with a scale per 128 x 128 tile, fp32."""
    rows, cols = q.shape
    return q.float() * scale.repeat_interleave(128, 1)[:, :cols].repeat_interleave(128, 0)[:rows]


class _Experts(torch.autograd.Function):
    """ops.moe_forward_blocks with the gradients of its rows and routing weights; the experts are frozen.

    The gradient passes the two roundings to e4m3 codes (rows, silu(gate) * up) as if they were not there, at the
    values that the codes hold. It is the plain chain in fp32, one expert at a time: that expert's weights are
    dequantized (12 H I bytes at a time) and multiplied by library products, and the host reads the rows per expert
    once, so the backward pass cannot be captured in a graph. Forward products are the framework's kernels.
    """

    @staticmethod
    def forward(ctx, rows, weights, ids, gate_up, gate_up_scale, down, down_scale, n_shared):
        ctx.save_for_backward(rows, weights, ids, gate_up, gate_up_scale, down, down_scale)
        ctx.n_shared = n_shared
        return ops.moe_forward_blocks(rows, gate_up, gate_up_scale, down, down_scale, topk_ids=ids, topk_weights=weights,
                                      n_shared=n_shared)

    @staticmethod
    @differentiable_once
    def backward(ctx, dy):
        rows, weights, ids, gate_up, gate_up_scale, down, down_scale = ctx.saved_tensors
        routed, k = gate_up.shape[0] - ctx.n_shared, weights.shape[1]
        x, dy = _row_values(rows), dy.float()
        dx, dw = torch.zeros_like(x), torch.zeros_like(weights)

        def expert(j, x, dy, w):
            """Gradients of the rows x and, one per row, of w in w * W2 (silu(W1 x) * (W3 x))."""
            w13 = _tile_values(gate_up[j], gate_up_scale[j])
            gate, up = (x @ w13.t()).chunk(2, 1)
            sig = torch.sigmoid(gate)
            act = gate * sig
            dh = dy @ _tile_values(down[j], down_scale[j])
            d_weight = (dh * _row_values(act * up)).sum(1)
            dh = dh * w
            d_gate = dh * up * (sig + act * (1 - sig))
            return torch.cat((d_gate, dh * act), 1) @ w13, d_weight

        flat = ids.reshape(-1).long()
        flat = torch.where((flat >= 0) & (flat < routed), flat, routed)  # a slot without an expert
        order = flat.argsort(stable=True)
        at = 0
        for j, n in enumerate(torch.bincount(flat, minlength=routed + 1).tolist()[:routed]):
            if n == 0:
                continue
            pair = order[at:at + n]
            at += n
            token = pair // k
            d_rows, d_weight = expert(j, x[token], dy[token], weights.view(-1)[pair][:, None])
            dx.index_add_(0, token, d_rows)  # the router names an expert once per token: no two rows meet
            dw.view(-1)[pair] = d_weight
        for j in range(routed, gate_up.shape[0]):
            dx += expert(j, x, dy, 1.0)[0]
        return dx.to(rows.dtype), dw, None, None, None, None, None, None


CODE_BUFFERS = ("gate_up", "gate_up_scale", "down", "down_scale")


class FeedForwardBlock(torch.nn.Module):
    """Router, block-scaled experts, post norm, gate, residual sum and the next block's pre norm.

    router_w [E, H] float32; gate_up [E + n_shared, 2I, H] (rows [:I] the SiLU branch) and down
    [E + n_shared, H, I] in float32, bfloat16 or float16; H and I multiples of 16. post_weight [H], gate
    [H] and pre_weight [H] are optional (no norm, gate 1, no norm). balance_coefficient scales the loss
    of ``balance``. The quantized weights are buffers: saved, loaded and moved with the module, never cast. A router
    cast to 16 bits is read as fp32.
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
        for names, pair in zip((CODE_BUFFERS[:2], CODE_BUFFERS[2:]), codes):
            for name, t in zip(names, pair):
                self.register_buffer(name, t)
        for name, w in (("pre_weight", pre_weight), ("post_weight", post_weight), ("gate", gate)):
            self.register_parameter(name, None if w is None else torch.nn.Parameter(w.detach().clone()))

    def _apply(self, fn, recurse=True):
        """Moves as Module has them; casts leave the codes and their fp32 scales what they are."""
        held = {name: self._buffers.pop(name) for name in CODE_BUFFERS}
        try:
            super()._apply(fn, recurse)
        finally:
            self._buffers.update(held)
        for name, t in held.items():
            bits = t.view(torch.uint8)  # an integer tensor: casts of floating-point tensors pass it by
            moved = fn(bits)
            self._buffers[name] = (moved if moved.dtype == torch.uint8 else bits.to(moved.device)).view(t.dtype)
        return self

    def start(self, x, normed_dtype=None):
        """(residual, normed) of the stack's first block: x and its pre norm (x itself without pre_weight).

        The experts read 16-bit rows: normed_dtype names their type, x's own by default, bfloat16 beside an fp32 x.
        """
        if normed_dtype is None:
            normed_dtype = torch.bfloat16 if x.dtype == torch.float32 else x.dtype
        if self.pre_weight is None:
            return x, x.to(normed_dtype)
        return x, ops.norm_residual(None, x, pre_weight=self.pre_weight, eps=self.eps, normed_dtype=normed_dtype)[1]

    def experts(self, normed):
        """The routed experts' output for normed [..., H]; differentiable in normed and router_w."""
        rows = normed.reshape(-1, normed.shape[-1]).contiguous()
        router_w = self.router_w.float()
        codes = (self.gate_up, self.gate_up_scale, self.down, self.down_scale)
        if torch.is_grad_enabled() and (rows.requires_grad or router_w.requires_grad):
            ids, weights, _ = _Route.apply(rows, router_w, self.k)
            y = _Experts.apply(rows, weights, ids, *codes, self.n_shared)
        else:  # decoding: without the autograd functions' host code
            ids, weights, _ = ops.route_topk(rows, router_w, self.k)
            y = ops.moe_forward_blocks(rows, *codes, topk_ids=ids, topk_weights=weights, n_shared=self.n_shared)
        return y.view(normed.shape)

    def forward(self, residual, normed, next_pre_weight=None):
        """-> (residual', normed') with next_pre_weight (the next block's pre norm), else (residual',).

        Gradients reach both inputs, the norms' weights, the gate and the router; the experts' weights are frozen.
        """
        return ops.norm_residual(self.experts(normed), residual, post_weight=self.post_weight, gate=self.gate,
                                 residual_scale=self.residual_scale, pre_weight=next_pre_weight, eps=self.eps)

    def balance(self, normed, valid=None):
        """The router's balance loss on normed [..., H] -> (loss, counts per expert, tokens); differentiable in
        router_w and normed. The counts are of the experts that ``experts`` runs for the same rows."""
        rows = normed.reshape(-1, normed.shape[-1]).contiguous()
        ids, _, logits = _Route.apply(rows, self.router_w.float(), self.k)
        return ops.balance_loss(logits, ids, self.balance_coefficient, valid=valid)


__all__ = ["FeedForwardBlock"]
