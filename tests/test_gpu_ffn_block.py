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


def straight(x):
    """x as its codes hold it, in float64; its gradient passes the rounding."""
    q = dequant(*ref_codes(x.detach().float(), 1), 1)
    return x + (q - x).detach()


def ref_experts(block, normed, router_w, ids):
    """The routed experts in float64 with the experts chosen as `ids`, differentiable in normed and router_w."""
    e = block.router_w.shape[0]
    weights = torch.gather(normed @ router_w.t(), 1, ids.long()).softmax(1)
    x = straight(normed)
    out = torch.zeros_like(normed)
    for j in range(block.gate_up.shape[0]):
        if j < e:
            token, slot = (ids == j).nonzero(as_tuple=True)
            w = weights[token, slot][:, None]
        else:
            token, w = torch.arange(normed.shape[0], device=DEV), 1.0
        if token.numel() == 0:
            continue
        y = x[token] @ dequant(block.gate_up[j], block.gate_up_scale[j], 128).t()
        i = y.shape[1] // 2
        act = straight(torch.nn.functional.silu(y[:, :i]) * y[:, i:])
        out = out.index_add(0, token, (act @ dequant(block.down[j], block.down_scale[j], 128).t()) * w)
    return out


def ref_rms(x, w, eps=1e-6):
    return x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w


@pytest.mark.parametrize("t", [6, 200])
def test_gradients_reach_the_input_and_the_router(ops, t):
    """The experts' own gradient: of the rows that they read and of the router that weighs them."""
    block = make_block()
    x = randn(t, H, seed=90, dtype=BF16).requires_grad_(True)
    g = randn(t, H, seed=91, dtype=BF16)
    y = block.experts(x)
    y.backward(g)
    ids, _, _ = ops.route_topk(x.detach(), block.router_w.detach(), K)
    xd, rd = x.detach().double().requires_grad_(True), block.router_w.detach().double().requires_grad_(True)
    ref = ref_experts(block, xd, rd, ids)
    close(y, ref, LAYER_TOL[BF16])
    ref.backward(g.double())
    close(x.grad, xd.grad, LAYER_TOL[BF16])
    close(block.router_w.grad, rd.grad, LAYER_TOL[BF16])


def test_gradients_of_two_blocks(ops):
    """A stack: what an earlier block's inputs and weights get through the later block's experts."""
    a, b = make_block(seed=100), make_block(seed=120)
    x = randn(40, H, seed=92).requires_grad_(True)  # an fp32 stream, so that the roundings between the blocks are few
    residual, normed = x, ops.norm_residual(None, x, pre_weight=a.pre_weight, normed_dtype=BF16)[1]
    residual, normed2 = a(residual, normed, next_pre_weight=b.pre_weight)
    out, = b(residual, normed2)
    g = randn(40, H, seed=93)
    out.backward(g)
    names = ["pre_weight", "post_weight", "gate", "router_w"]
    p = [{n: getattr(m, n).detach().double().requires_grad_(True) for n in names} for m in (a, b)]
    xd = x.detach().double().requires_grad_(True)
    r, n, pre = xd, None, p[0]["pre_weight"]
    for m, q, got in ((a, p[0], normed), (b, p[1], normed2)):
        n = ref_rms(r, q["pre_weight"])
        n = n + (got.detach().double() - n).detach()  # the rows that the experts read, as the 16-bit type holds them
        ids, _, _ = ops.route_topk(got.detach(), m.router_w.detach(), K)
        y = ref_experts(m, n, q["router_w"], ids)
        y = y + (m.experts(got.detach()).detach().double() - y).detach()
        r = 0.9 * r + q["gate"] * ref_rms(y, q["post_weight"])
    close(out, r, 1e-4)
    r.backward(g.double())
    close(x.grad, xd.grad, LAYER_TOL[BF16])
    for m, q in ((a, p[0]), (b, p[1])):
        for name in names:
            close(getattr(m, name).grad, q[name].grad, LAYER_TOL[BF16])


def test_gradient_is_the_same_every_run(ops):
    block = make_block()
    x = randn(150, H, seed=94, dtype=BF16)
    g = randn(150, H, seed=95, dtype=BF16)
    grads = []
    for _ in range(3):
        leaf = x.clone().requires_grad_(True)
        block.zero_grad()
        block.experts(leaf).backward(g)
        grads.append((leaf.grad, block.router_w.grad.clone()))
    for a, b in grads[1:]:
        assert torch.equal(a, grads[0][0]) and torch.equal(b, grads[0][1])


def test_the_same_with_and_without_grad_mode(ops):
    block = make_block()
    x = randn(9, H, seed=104, dtype=BF16)
    want = block.experts(x)
    assert want.requires_grad
    with torch.no_grad():
        assert torch.equal(block.experts(x), want.detach())
    block.requires_grad_(False)
    assert not block.experts(x).requires_grad and block.experts(x.clone().requires_grad_(True)).requires_grad


def test_state_holds_the_experts(ops):
    a, b = make_block(seed=80), make_block(seed=140)
    names = {"gate_up", "gate_up_scale", "down", "down_scale"}
    assert names <= set(a.state_dict())
    x = randn(12, H, seed=96, dtype=BF16)
    assert not torch.equal(a.experts(x), b.experts(x))
    b.load_state_dict({k: v.cpu() for k, v in a.state_dict().items()})
    assert torch.equal(a.experts(x), b.experts(x))
    c = copy.deepcopy(a)
    assert torch.equal(a.experts(x), c.experts(x))


def test_moves_and_casts_keep_the_codes(ops):
    block = make_block()
    x = randn(12, H, seed=97, dtype=BF16)
    want = block.experts(x)
    block.cpu()
    assert all(getattr(block, n).device.type == "cpu" for n in ("gate_up", "gate_up_scale", "down", "down_scale"))
    block.to(DEV)
    assert torch.equal(block.experts(x), want)
    for cast in (lambda m: m.double(), lambda m: m.float(), lambda m: m.to(F16), lambda m: m.float()):
        cast(block)
        assert block.gate_up.dtype == block.down.dtype == torch.float8_e4m3fn
        assert block.gate_up_scale.dtype == block.down_scale.dtype == F32
    block.to(torch.device(DEV), F32)
    assert block.experts(x).isfinite().all()
    assert block.bfloat16().experts(x).isfinite().all()  # a router in 16 bits is read as fp32


def test_start_without_a_norm_and_with_an_fp32_stream(ops):
    block = make_block(pre_weight=None)
    x = randn(10, H, seed=98, dtype=BF16)
    residual, normed = block.start(x)
    assert residual is x and torch.equal(normed, x)
    assert len(block(residual, normed)) == 1
    x32 = randn(10, H, seed=99)
    assert block.start(x32)[1].dtype == BF16
    block = make_block()
    for dtype, want in ((None, BF16), (F16, F16), (BF16, BF16)):
        residual, normed = block.start(x32, normed_dtype=dtype)
        assert residual is x32 and normed.dtype == want
        close(normed, ref_rms(x32.double(), block.pre_weight.double()))
        new, nxt = block(residual, normed, next_pre_weight=block.pre_weight)
        assert new.dtype == F32 and nxt.dtype == want


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


def test_second_order_gradients_are_refused(ops):
    block = make_block()
    x = randn(8, H, seed=103, dtype=BF16).requires_grad_(True)
    g, = torch.autograd.grad(block.experts(x).float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        (g.float().square().sum() + x.float().square().sum()).backward()
