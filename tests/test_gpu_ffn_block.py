"""The feed-forward sublayer (stageml_b200.ffn_block): gradients, state, types, and the experts that its loss counts."""

import copy

import pytest
import torch

from test_gpu_block_ops import (BF16, DEV, F16, F32, LAYER_TOL, blocks, clean_status, close, dequant, ops, randn,  # noqa: F401
                                ref_codes)

pytestmark = pytest.mark.gpu
E, K, H, I = 8, 2, 256, 160


def make_block(seed=80, e=E, k=K, shared=1, h=H, i=I, **kw):
    from stageml_b200.ffn_block import FeedForwardBlock

    args = dict(pre_weight=1 + randn(h, seed=seed + 3, scale=0.1), post_weight=1 + randn(h, seed=seed + 4, scale=0.1),
                gate=randn(h, seed=seed + 5, scale=0.3), residual_scale=0.9)
    args.update(kw)
    return FeedForwardBlock(randn(e, h, seed=seed, scale=h ** -0.5),
                            randn(e + shared, 2 * i, h, seed=seed + 1, scale=h ** -0.5, dtype=BF16),
                            randn(e + shared, h, i, seed=seed + 2, scale=i ** -0.5, dtype=BF16), k, n_shared=shared, **args)


@pytest.mark.parametrize("t", [5, 300, 5000])
def test_balance_counts_the_experts_that_ran(ops, t):
    """Ties between experts up to the order of a sum: the loss counts what the experts' router chose, not what another
    order of the sum would choose."""
    h, e, k = 512, 32, 3  # an odd k: one of a pair is left out
    block = make_block(e=e, k=k, h=h, i=32, shared=0)
    with torch.no_grad():  # the second of two experts has the first one's row, turned by half as x's halves are equal
        block.router_w[1::2] = block.router_w[0::2].roll(h // 2, 1)
    x = randn(t, h // 2, seed=101, dtype=BF16).repeat(1, 2)
    ids, _, logits = ops.route_topk(x, block.router_w.detach(), k)
    loss, counts, tokens = block.balance(x)
    assert int(tokens) == t
    assert torch.equal(counts.long(), torch.bincount(ids.reshape(-1).long(), minlength=e))
    # its gradient: that of the loss in float64 through the logits
    xd = x.clone().requires_grad_(True)
    block.zero_grad()
    loss, counts, _ = block.balance(xd)
    loss.backward()
    x64, r64 = x.double().requires_grad_(True), block.router_w.detach().double().requires_grad_(True)
    p = (x64 @ r64.t()).softmax(1).mean(0)
    ref = block.balance_coefficient * e * (counts.double() / (k * t) * p).sum()
    ref.backward()
    close(loss, ref)
    close(block.router_w.grad, r64.grad, 1e-4)
    close(xd.grad, x64.grad, LAYER_TOL[BF16])


def test_balance_takes_fp32_rows(ops):
    block = make_block()
    x = randn(30, H, seed=102)
    loss, counts, tokens = block.balance(x)
    assert int(counts.sum()) == K * 30 and int(tokens) == 30 and loss.requires_grad
