"""Python entry points of the B200 residual path.

Thin functions over ``torch.ops.stageml.*`` (csrc/torch_ops.cpp -> C ABI ->
sm_100a kernels). Each one takes CUDA tensors and launches on the current
stream. Fake (meta) implementations are registered so the ops trace under
``torch.compile`` / FakeTensor without running.
"""

from __future__ import annotations

import functools
from typing import Optional

import torch

from ._native import ensure_cuda_device, load_torch_ops

load_torch_ops()
_ops = torch.ops.stageml
# overloads resolved once: the calls below are launch-bound for small batches
_quantize_e4m3_blocks = _ops.quantize_e4m3_blocks.default
_block_matmul = _ops.block_matmul.default
_moe_forward_blocks = _ops.moe_forward_blocks.default
_norm_residual = _ops.norm_residual.default
_norm_residual_backward = _ops.norm_residual_backward.default
_balance_loss = _ops.balance_loss.default
_balance_loss_backward = _ops.balance_loss_backward.default


def _register_fakes() -> None:
    lib = torch.library

    @lib.register_fake("stageml::residual_moe")
    def _(hidden, gate_up, down, topk_weights, topk_ids):
        return hidden.new_empty((hidden.shape[0], down.shape[1]))

    @lib.register_fake("stageml::moe_forward")
    def _(x, gate_up, down, topk_weights, topk_ids, router_w, k, n_shared, renormalize, tenant_ids, n_tenants, rank,
          lora_a13, lora_b13, lora_a2, lora_b2, lora_scale, gate_up_scale, down_scale, T_dev=None, fold_slot=None,
          n_fold=0, down_group=None):
        return x.new_empty((x.shape[0], x.shape[1]))

    @lib.register_fake("stageml::route_topk")
    def _(x, gate_w, k, renormalize):
        T = x.shape[0]
        return (x.new_empty((T, k), dtype=torch.int32), x.new_empty((T, k), dtype=torch.float32),
                x.new_empty((T, gate_w.shape[0]), dtype=torch.float32))

    @lib.register_fake("stageml::topk_from_logits")
    def _(logits, k, renormalize):
        T = logits.shape[0]
        return logits.new_empty((T, k), dtype=torch.int32), logits.new_empty((T, k), dtype=torch.float32)

    @lib.register_fake("stageml::lora_fold")
    def _(W, A, B, scale, layout):
        if A.dim() == 3:
            return W.new_empty((A.shape[0], W.shape[-2], W.shape[-1]))
        return W.new_empty(W.shape)

    @lib.register_fake("stageml::lora_linear")
    def _(x, w_bank, bias, row_group, row_tenant, n_tenants, rank, lora_a, lora_b, lora_scale):
        return x.new_empty((x.shape[0], w_bank.shape[1]))

    @lib.register_fake("stageml::moe_linear")
    def _(x, weight, bias, topk_ids, topk_weights, tenant_ids, n_experts, group_by_tenant, n_tenants, rank, lora_a,
          lora_b, lora_scale):
        return x.new_empty((x.shape[0], weight.shape[1]))

    @lib.register_fake("stageml::combine_rows")
    def _(y, pair_row, T, kk):
        return y.new_empty((T, y.shape[1]))

    @lib.register_fake("stageml::lora_gemv_f32")
    def _(x, W, A, B, scale):
        return x.new_empty((x.shape[0], W.shape[1]))

    def blocks(n):
        return (n + 127) // 128

    @lib.register_fake("stageml::quantize_e4m3_blocks")
    def _(x, tiles):
        shape = list(x.shape)
        shape[-1] = blocks(shape[-1])
        if tiles:
            shape[-2] = blocks(shape[-2])
        return x.new_empty(x.shape, dtype=torch.float8_e4m3fn), x.new_empty(shape, dtype=torch.float32)

    @lib.register_fake("stageml::block_matmul")
    def _(x, x_scale, w, w_scale, out_dtype):
        return x.new_empty((x.shape[0], w.shape[0]), dtype=out_dtype)

    @lib.register_fake("stageml::moe_forward_blocks")
    def _(x, gate_up, gate_up_scale, down, down_scale, topk_ids, topk_weights, n_shared):
        return x.new_empty(x.shape)

    @lib.register_fake("stageml::norm_residual")
    def _(block_out, residual, post_weight, gate, pre_weight, residual_scale, eps, quantize, normed_dtype=None):
        shape = tuple(residual.shape)
        out = [residual.new_empty(shape)]
        if quantize:
            out.append(residual.new_empty(shape, dtype=torch.float8_e4m3fn))
            out.append(residual.new_empty(shape[:-1] + (blocks(shape[-1]),), dtype=torch.float32))
        elif pre_weight is not None:
            dtype = block_out.dtype if block_out is not None else normed_dtype or residual.dtype
            out.append(residual.new_empty(shape, dtype=dtype))
        return out

    @lib.register_fake("stageml::norm_residual_backward")
    def _(grad_residual, grad_normed, block_out, residual, post_weight, gate, pre_weight, residual_scale, eps):
        return [t.new_empty(t.shape) for t in (residual, block_out, post_weight, gate, pre_weight) if t is not None]

    @lib.register_fake("stageml::balance_loss")
    def _(logits, topk_ids, coefficient, valid):
        return (logits.new_empty((), dtype=torch.float32), logits.new_empty((logits.shape[1],), dtype=torch.int32),
                logits.new_empty((), dtype=torch.int32))

    @lib.register_fake("stageml::balance_loss_backward")
    def _(grad_loss, logits, counts, tokens, k, coefficient, valid):
        return torch.empty_like(logits)


try:
    _register_fakes()
except Exception:  # pragma: no cover - re-registration in the same process
    pass


def residual_moe(hidden, gate_up, down, topk_weights, topk_ids):
    """The reference's ``stageml::residual_moe`` (csrc/stageml_residual_op.cpp:17-19), semantics of
    ``_fallback_moe`` (stageml/custom_op_registry.py:23-37)."""
    ensure_cuda_device(hidden)
    return _ops.residual_moe(hidden, gate_up.contiguous(), down.contiguous(), topk_weights.contiguous(),
                             topk_ids.contiguous())


def moe_forward(x, gate_up, down, *, topk_weights=None, topk_ids=None, router_w=None, k: int = 2, n_shared: int = 0,
                renormalize: bool = True, tenant_ids=None, n_tenants: int = 0, rank: int = 0, lora_a13=None,
                lora_b13=None, lora_a2=None, lora_b2=None, lora_scale=None, gate_up_scale=None, down_scale=None,
                T_dev=None, fold_slot=None, n_fold: int = 0, down_group=None):
    """One MoE-LoRA FFN layer (router -> permutation -> SwiGLU experts with per-tenant LoRA -> combine).

    T_dev: optional CUDA int32 tensor; only the first T_dev[0] tokens are valid (the rest are skipped and
    their output rows are left unwritten), for token counts known only on the device.
    fold_slot: optional CUDA int32 [n_tenants, E_tot]; entry (a, e) = s >= 0 runs tenant a's pairs of
    expert e on folded weight set s, stored as group E_tot + s of gate_up / down ([E_tot + n_fold, ...]),
    without dynamic LoRA; -1 = base weights plus the tenant's LoRA. One permutation, one set of GEMMs.
    down_group: optional CUDA int32 [E_tot + n_fold] with entries in [0, E_tot): weight group g takes
    down[down_group[g]] (down then holds the E_tot base experts), for folded sets whose adapters leave
    w2 unchanged.
    """
    ensure_cuda_device(x)
    if topk_ids is not None:
        k = int(topk_ids.shape[1])
    return _ops.moe_forward(x, gate_up, down, topk_weights, topk_ids, router_w, int(k), int(n_shared),
                            bool(renormalize), tenant_ids, int(n_tenants), int(rank), lora_a13, lora_b13, lora_a2,
                            lora_b2, lora_scale, gate_up_scale, down_scale, T_dev, fold_slot, int(n_fold),
                            down_group)


def route_topk(x, gate_w, k: int, renormalize: bool = True):
    """Router logits (fp32), softmax, top-k, renormalisation -> (ids int32, weights fp32, logits fp32)."""
    ensure_cuda_device(x)
    return _ops.route_topk(x, gate_w, int(k), bool(renormalize))


def topk_from_logits(logits, k: int, renormalize: bool = True):
    ensure_cuda_device(logits)
    return _ops.topk_from_logits(logits, int(k), bool(renormalize))


PLAN_FIELDS = ("row_token", "row_tenant", "row_weight", "row_pair", "pair_row", "tile_group", "group_offsets",
               "group_counts", "num_tiles")


def permute(ids, weights=None, tenant_ids=None, *, n_experts_total: int, n_shared: int = 0, n_tenants: int = 0,
            group_by_tenant: bool = False) -> dict:
    """Stable (expert, tenant) permutation with 128-row padded expert segments; returns the plan arrays."""
    ensure_cuda_device(ids)
    out = _ops.permute(ids, weights, tenant_ids, int(n_experts_total), int(n_shared), int(n_tenants),
                       bool(group_by_tenant))
    return dict(zip(PLAN_FIELDS, out))


def lora_fold(W, A, B, scale, layout: int = 0):
    """W' = W + s * B @ A (layout 0, [out,in]) or W + s * A @ B (layout 1, [in,out]); batched over A/B."""
    ensure_cuda_device(W)
    if not torch.is_tensor(scale):
        n = A.shape[0] if A.dim() == 3 else 1
        scale = torch.full((n,), float(scale), dtype=torch.float32, device=W.device)
    return _ops.lora_fold(W.contiguous(), A.contiguous(), B.contiguous(), scale.to(torch.float32).contiguous(),
                          int(layout))


def lora_linear(x, w_bank, *, bias=None, row_group=None, row_tenant=None, n_tenants: int = 0, rank: int = 0,
                lora_a=None, lora_b=None, lora_scale=None):
    """Mixed-adapter dense linear: folded weights by row group, dynamic LoRA by row tenant."""
    ensure_cuda_device(x)
    return _ops.lora_linear(x, w_bank, bias, row_group, row_tenant, int(n_tenants), int(rank), lora_a, lora_b,
                            lora_scale)


def moe_linear(x, weight, topk_ids, topk_weights, *, bias=None, tenant_ids=None, n_experts: int,
               group_by_tenant: bool = False, n_tenants: int = 0, rank: int = 0, lora_a=None, lora_b=None,
               lora_scale=None):
    """Routed single-linear MoE-LoRA layer (DynamicMoELoRALayer / MaterializedMoELoRALayer)."""
    ensure_cuda_device(x)
    return _ops.moe_linear(x, weight, bias, topk_ids, topk_weights, tenant_ids, int(n_experts), bool(group_by_tenant),
                           int(n_tenants), int(rank), lora_a, lora_b, lora_scale)


def lora_gemv_f32(x, W, A=None, B=None, scale: float = 1.0):
    """fp32 y = x W + s (x A) B with W [in,out] (A None: y = x W)."""
    ensure_cuda_device(x)
    return _ops.lora_gemv_f32(x, W, A, B, float(scale))


def quantize_e4m3_rows(w):
    """Per-output-channel e4m3 quantization -> (q float8_e4m3fn, scale fp32)."""
    ensure_cuda_device(w)
    return _ops.quantize_e4m3_rows(w.contiguous())


def quantize_e4m3_blocks(x, tiles: bool = False):
    """e4m3 codes with one fp32 scale per 128 values -> (q float8_e4m3fn, scale fp32).

    x [..., K] float32/bfloat16/float16. tiles False (activations): scale [..., ceil(K/128)], one per 128
    values of a row. tiles True (weights [..., N, K]): scale [..., ceil(N/128), ceil(K/128)], one per
    128 x 128 tile. scale = max|x| / 448 (1 for a block of zeros), q = e4m3(x / scale), nearest even.
    """
    ensure_cuda_device(x)
    _no_grad("quantize_e4m3_blocks", x)
    return _quantize_e4m3_blocks(x.contiguous(), tiles)


def block_matmul(x, x_scale, w, w_scale, out_dtype=torch.bfloat16):
    """x w^T on block-scaled e4m3 operands, fp32 sums rounded once to out_dtype.

    x [M, K] with x_scale [M, ceil(K/128)], w [N, K] with w_scale [ceil(N/128), ceil(K/128)], as
    ``quantize_e4m3_blocks`` (tiles False / True) makes them; K a multiple of 16. -> [M, N].
    """
    ensure_cuda_device(x)
    return _block_matmul(x.contiguous(), x_scale.contiguous(), w.contiguous(), w_scale.contiguous(), out_dtype)


def moe_forward_blocks(x, gate_up, gate_up_scale, down, down_scale, *, topk_ids=None, topk_weights=None,
                       n_shared: int = 0):
    """One routed SwiGLU FFN layer on block-scaled e4m3 weights, both products on e4m3 operands.

    x [T, H] bfloat16/float16; gate_up [E + n_shared, 2I, H] and down [E + n_shared, H, I] e4m3 with the
    scales of ``quantize_e4m3_blocks(w, tiles=True)``; topk_ids [T, k] and topk_weights [T, k] as
    ``route_topk`` gives them (None: only the shared experts). H and I are multiples of 16. x and
    silu(gate) * up are quantized per 128 values of a row on the way. No LoRA: tenants with adapters
    take ``moe_forward``.
    """
    ensure_cuda_device(x)
    _no_grad("moe_forward_blocks", x, topk_weights)
    return _moe_forward_blocks(x.contiguous(), gate_up, gate_up_scale, down, down_scale, topk_ids, topk_weights,
                               n_shared)


def norm_residual_backward(grad_residual, grad_normed, block_out, residual, *, post_weight=None, gate=None,
                           residual_scale: float = 1.0, pre_weight=None, eps: float = 1e-6):
    """Gradients of ``norm_residual`` from those of its outputs (either may be None = zero) and its inputs.

    -> (d_residual, d_block_out, d_post_weight, d_gate, d_pre_weight), None for inputs that are None. Each
    has its input's shape and dtype; sums over tokens are fp32 in a fixed order.
    """
    ensure_cuda_device(residual)
    out = iter(_norm_residual_backward(grad_residual, grad_normed, block_out, residual, post_weight, gate, pre_weight,
                                       residual_scale, eps))
    return (next(out), None if block_out is None else next(out), None if post_weight is None else next(out),
            None if gate is None else next(out), None if pre_weight is None else next(out))


def _any_grad(*tensors) -> bool:
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


def _no_grad(name: str, *tensors) -> None:
    if torch.is_grad_enabled() and _any_grad(*tensors):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad() or on detached tensors")


class _Last(torch.autograd.Function):
    """Hands the first n tensors on; a gradient of them is an error."""

    @staticmethod
    def forward(ctx, n, *tensors):
        ctx.set_materialize_grads(False)
        return tuple(None if t is None else t.view_as(t) for t in tensors[:n])

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("this operator is differentiable once: its gradient has no gradient of its own")


def differentiable_once(backward):
    """For an autograd function's backward: it runs without a graph, and under create_graph its results refuse a
    gradient, also where the incoming gradients are constants."""

    @functools.wraps(backward)
    def wrapped(ctx, *grads):
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not torch.is_grad_enabled():
            return out
        single = not isinstance(out, tuple)
        out = (out,) if single else out
        out = _Last.apply(len(out), *out, *ctx.saved_tensors, *grads)
        return out[0] if single else out

    return wrapped


class _NormResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, block_out, residual, post_weight, gate, pre_weight, residual_scale, eps, normed_dtype):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(block_out, residual, post_weight, gate, pre_weight)
        ctx.numbers = {"residual_scale": residual_scale, "eps": eps}
        return tuple(_norm_residual(block_out, residual, post_weight, gate, pre_weight, residual_scale, eps, False,
                                    normed_dtype))

    @staticmethod
    @differentiable_once
    def backward(ctx, *grads):
        if all(g is None for g in grads):  # its consumers have passed none on
            return (None,) * 8
        block_out, residual, post_weight, gate, pre_weight = ctx.saved_tensors
        grad_normed = grads[1] if len(grads) > 1 else None
        d = norm_residual_backward(grads[0], grad_normed, block_out, residual, post_weight=post_weight, gate=gate,
                                   pre_weight=pre_weight, **ctx.numbers)
        return d[1], d[0], d[2], d[3], d[4], None, None, None


def norm_residual(block_out, residual, *, post_weight=None, gate=None, residual_scale: float = 1.0, pre_weight=None,
                  eps: float = 1e-6, quantize: bool = False, normed_dtype=None):
    """The norm after a block, its gate, the residual sum and the next block's norm in one pass.

    u = post_weight * rms_norm(block_out) (block_out itself without post_weight),
    new_residual = residual_scale * residual + gate * u (without block_out: residual_scale * residual),
    normed = pre_weight * rms_norm(new_residual).

    residual [..., H] float32/bfloat16/float16; block_out of the same shape, in residual's dtype or, beside a
    float32 residual, in any of the three; gate [H], [..., 1] or [..., H]; weights [H]. fp32 arithmetic, each
    output rounded once. -> (new_residual, normed), (new_residual,) without pre_weight. quantize=True returns
    (new_residual, codes, scale) instead: normed as ``quantize_e4m3_blocks`` would hold it, the operand of the
    block-scaled products. normed_dtype (block_out's dtype by default, else residual's) names normed's type.
    Differentiable once, except with quantize. H <= 16384.
    """
    ensure_cuda_device(residual)
    if torch.is_grad_enabled() and _any_grad(block_out, residual, post_weight, gate, pre_weight):
        if quantize:
            raise ValueError("norm_residual: the codes of quantize=True carry no gradient")
        return _NormResidual.apply(block_out, residual, post_weight, gate, pre_weight, residual_scale, eps,
                                   normed_dtype)
    return tuple(_norm_residual(block_out, residual, post_weight, gate, pre_weight, residual_scale, eps, quantize,
                                normed_dtype))


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, topk_ids, coefficient, valid):
        loss, counts, tokens = _balance_loss(logits, topk_ids, coefficient, valid)
        ctx.save_for_backward(logits, counts, tokens, valid)
        ctx.numbers = (topk_ids.shape[1], coefficient)
        ctx.mark_non_differentiable(counts, tokens)
        return loss, counts, tokens

    @staticmethod
    @differentiable_once
    def backward(ctx, grad_loss, _counts, _tokens):
        logits, counts, tokens, valid = ctx.saved_tensors
        return balance_loss_backward(grad_loss, logits, counts, tokens, *ctx.numbers, valid=valid), None, None, None


def balance_loss(logits, topk_ids, coefficient: float = 1.0, *, valid=None):
    """The router's balance loss with the counts per expert -> (loss fp32 [], counts int32 [E], tokens int32 []).

    loss = coefficient * E * sum_e f_e P_e: f_e the share of the chosen slots that went to expert e, P_e the mean
    softmax probability of e, both over the tokens with valid[t] (all without valid); tokens is their number.
    logits [T, E] as ``route_topk`` returns them (or bfloat16/float16), topk_ids [T, k] (negative: no expert).
    Differentiable once, in logits; the counts carry no gradient.
    """
    ensure_cuda_device(logits)
    logits, topk_ids = logits.contiguous(), topk_ids.contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        return _BalanceLoss.apply(logits, topk_ids, coefficient, valid)
    return _balance_loss(logits, topk_ids, coefficient, valid)


def balance_loss_backward(grad_loss, logits, counts, tokens, k: int, coefficient: float = 1.0, *, valid=None):
    """Gradient of ``balance_loss``'s logits for grad_loss (CUDA fp32 scalar), from the forward's counts and tokens."""
    ensure_cuda_device(logits)
    return _balance_loss_backward(grad_loss.contiguous(), logits.contiguous(), counts, tokens, k, coefficient, valid)


def combine_rows(y, pair_row, T: int, kk: int):
    """out[t] = sum_j y[pair_row[t*kk + j]] (rows < 0 skipped), fp32 sum, one rounding."""
    ensure_cuda_device(y)
    return _ops.combine_rows(y.contiguous(), pair_row.to(torch.int32).contiguous(), int(T), int(kk))


def take_status(like) -> int:
    """Synchronise and return (then clear) the device status word of like's device (0 = ok)."""
    return int(_ops.take_status(like))


__all__ = [
    "residual_moe",
    "moe_forward",
    "route_topk",
    "topk_from_logits",
    "permute",
    "lora_fold",
    "lora_linear",
    "moe_linear",
    "lora_gemv_f32",
    "quantize_e4m3_rows",
    "quantize_e4m3_blocks",
    "block_matmul",
    "moe_forward_blocks",
    "norm_residual",
    "norm_residual_backward",
    "balance_loss",
    "balance_loss_backward",
    "combine_rows",
    "take_status",
    "PLAN_FIELDS",
]
