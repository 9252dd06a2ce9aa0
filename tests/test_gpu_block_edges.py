"""Edges of the block-scaled operators, the block norm and the balance loss, on the GPU.

References are those of test_gpu_block_ops.py: the definitions in float64 on the same inputs.
"""

import math

import pytest
import torch

from test_gpu_block_ops import (BF16, DEV, F16, F32, LAYER_TOL, TOL, blocks, clean_status, close, dequant,  # noqa: F401
                                layer_weights, norm_inputs, ops, randn, ref_codes, ref_layer, ref_norm)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ routed layer
@pytest.mark.parametrize("t", [8, 200])
def test_slots_are_summed_before_the_rounding(ops, t):
    """A token's slots meet in fp32: one rounding to 16 bits. What is left beside it are h's codes that fall on the
    other side of a rounding boundary (at most one in 10^4 by 2^-4 of a value: 6e-4) and outputs that these
    differences carry over a boundary of theirs, together below one rounding (2^-9 of a bf16 value)."""
    e, k, h, i = 16, 8, 512, 384
    gu, gus, dn, dns = layer_weights(e + 1, h, i, seed=21)
    x = randn(t, h, seed=22, dtype=BF16)
    top = randn(t, e, seed=23).topk(k, 1)
    ids, w = top.indices.to(torch.int32), top.values.softmax(1)
    y = ops.moe_forward_blocks(x, gu, gus, dn, dns, topk_ids=ids, topk_weights=w, n_shared=1)
    close(y, ref_layer(x, gu, gus, dn, dns, ids, w, 1), TOL[BF16])


@pytest.mark.parametrize("t", [8, 200])
def test_slots_beyond_the_16_bit_range(ops, t):
    """Weighted rows past float16's 65504 whose sum is not: two copies of an expert at weights c + 1 and -c."""
    h, i = 256, 128
    gu, gus, dn, dns = (p[:1].expand(2, *p.shape[1:]).contiguous() for p in layer_weights(1, h, i, seed=24))
    dns = dns * 1024.0
    x = randn(t, h, seed=25, dtype=F16)
    ids = torch.tensor([0, 1], dtype=torch.int32, device=DEV).repeat(t, 1)
    w = torch.tensor([1025.0, -1024.0], device=DEV).repeat(t, 1)
    ref = ref_layer(x, gu, gus, dn, dns, ids, w, 0)
    assert ref.abs().max() < 60000 and 1024 * ref.abs().max() > 65504
    y = ops.moe_forward_blocks(x, gu, gus, dn, dns, topk_ids=ids, topk_weights=w)
    # each slot's fp32 error is 1e-5 of 1024 times the sum: 1e-5 * 1024 * sqrt 2
    close(y, ref, TOL[F16] + 1.5e-2)


@pytest.mark.parametrize("t", [16, 200])
@pytest.mark.parametrize("scale", [1e-18, 1e-19, 1e-20, 1e-21, 1e-22, 1e-23])
def test_rows_of_small_numbers(ops, t, scale):
    """h at the bottom of fp32's range, with a channel of zeros: finite, and its definition's value. From 1e-21 on h
    itself has only a few bits and the scale's rounding decides; there the output is only bounded."""
    e, k, h, i = 4, 2, 192, 160
    gu, gus, dn, dns = layer_weights(e, h, i, seed=26)
    gu.view(torch.uint8)[:, 5] = 0  # a pruned gate channel: h[5] = 0
    dns = torch.full_like(dns, 16.0)  # a power of two: the product of the two scales is exact
    x = (randn(t, h, seed=27) * scale).to(BF16)
    ids = randn(t, e, seed=28).topk(k, 1).indices.to(torch.int32)
    w = torch.full((t, k), 0.5, device=DEV)
    y = ops.moe_forward_blocks(x, gu, gus, dn, dns, topk_ids=ids, topk_weights=w)
    assert y.isfinite().all()
    ref = ref_layer(x, gu, gus, dn, dns, ids, w, 0)
    if scale >= 1e-20:
        close(y, ref, LAYER_TOL[BF16])
    else:
        wide = torch.nn.functional.silu(x.double()).abs().max()  # bound: |h| <= (|W| |x|)^2 / 2 over 192 terms of 4 / sqrt h
        assert y.double().abs().max() <= 16 * 448 * i * max(float((8 * wide * math.sqrt(h)) ** 2), 2.0 ** -149 * 448)


@pytest.mark.parametrize("t", [17, 32, 64, 128])
@pytest.mark.parametrize("shared", [1, 3])
def test_shared_experts_alone(ops, t, shared):
    h, i = 256, 144
    gu, gus, dn, dns = layer_weights(shared, h, i, seed=29)
    x = randn(t, h, seed=30, dtype=BF16)
    close(ops.moe_forward_blocks(x, gu, gus, dn, dns, n_shared=shared),
          ref_layer(x, gu, gus, dn, dns, None, None, shared), LAYER_TOL[BF16])


@pytest.mark.parametrize("t,e", [(8, 64), (40, 64), (200, 8), (3000, 64)])
def test_layer_same_bits_every_run(ops, t, e):
    h, i, k = 512, 272, 6
    gu, gus, dn, dns = layer_weights(e + 1, h, i, seed=80)
    x = randn(t, h, seed=81, dtype=BF16)
    top = randn(t, e, seed=82).topk(k, 1)
    ids, w = top.indices.to(torch.int32), top.values.softmax(1)
    first = ops.moe_forward_blocks(x, gu, gus, dn, dns, topk_ids=ids, topk_weights=w, n_shared=1)
    for _ in range(5):
        assert torch.equal(ops.moe_forward_blocks(x, gu, gus, dn, dns, topk_ids=ids, topk_weights=w, n_shared=1), first)


# ------------------------------------------------------------------ gradients that are not there
@pytest.mark.parametrize("constant", [False, True])
def test_second_order_gradients_are_refused(ops, constant):
    """Under create_graph the gradients refuse one of their own, with incoming gradients that need one and constant
    ones, and do not drop out of a sum without a word."""
    v = norm_inputs(6, 64, F32, F32, "channel", True, True, seed=31)
    leaves = {k: x.clone().requires_grad_(True) for k, x in v.items()}
    new, z = ops.norm_residual(leaves["y"], leaves["r"], post_weight=leaves["post"], gate=leaves["gate"],
                               pre_weight=leaves["pre"])
    first = torch.autograd.grad((new.sum() + z.sum()) if constant else (new * z).sum(), list(leaves.values()),
                                create_graph=True)
    for g in first:
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(g.square().sum() + leaves["r"].square().sum(), leaves["r"], retain_graph=True)
    logits = randn(9, 8, seed=32).requires_grad_(True)
    loss, _, _ = ops.balance_loss(logits, logits.detach().topk(2, 1).indices.to(torch.int32))
    g, = torch.autograd.grad(loss if constant else loss * loss, logits, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        (g.square().sum() + logits.square().sum()).backward()


def test_norm_residual_backward_without_any_gradient(ops):
    """A consumer without a gradient of its own: the norm's node is reached with none, and passes none on."""

    class Cut(torch.autograd.Function):
        @staticmethod
        def forward(ctx, a):
            return a.clone()

        @staticmethod
        def backward(ctx, g):
            return None

    r = randn(4, 64, seed=40).requires_grad_(True)
    y = randn(4, 64, seed=41)
    new, z = ops.norm_residual(y, r, pre_weight=torch.ones(64, device=DEV))
    (Cut.apply(new).sum() + Cut.apply(z).sum()).backward()
    assert r.grad is None


def _calls(ops):
    """(name, call with the tensors of `t`, names of the tensors that could ask for a gradient)"""
    raw = torch.ops.stageml
    x, xs = ref_codes(randn(5, 128, seed=33), 1)
    w, ws = ref_codes(randn(32, 128, seed=34), 128)
    gu, gus, dn, dns = layer_weights(2, 128, 64, seed=35)
    ids = torch.tensor([[0, 1]], dtype=torch.int32, device=DEV).repeat(5, 1)
    logits, counts, tokens = randn(5, 8, seed=36), torch.ones(8, dtype=torch.int32, device=DEV), \
        torch.full((), 5, dtype=torch.int32, device=DEV)
    v = norm_inputs(5, 128, F32, F32, "channel", True, True, seed=37)
    rows = randn(5, 128, seed=38)
    t = {"x_scale": xs, "w_scale": ws, "gus": gus, "dns": dns, "h": randn(5, 128, seed=39, dtype=BF16),
         "tw": torch.ones(5, 2, device=DEV), "logits": logits, "rows": rows, "g": torch.ones((), device=DEV), **v}
    norm = lambda t: (t["y"], t["r"], t["post"], t["gate"], t["pre"])  # noqa: E731
    kw = lambda t: {"post_weight": t["post"], "gate": t["gate"], "pre_weight": t["pre"]}  # noqa: E731
    five = ["y", "r", "post", "gate", "pre"]
    return t, [
        ("quantize", lambda t: ops.quantize_e4m3_blocks(t["rows"]), ["rows"]),
        ("matmul", lambda t: ops.block_matmul(x, t["x_scale"], w, t["w_scale"]), ["x_scale", "w_scale"]),
        ("layer", lambda t: ops.moe_forward_blocks(t["h"], gu, t["gus"], dn, t["dns"], topk_ids=ids, topk_weights=t["tw"]),
         ["h", "gus", "dns", "tw"]),
        ("norm backward", lambda t: ops.norm_residual_backward(t["rows"], t["rows"], t["y"], t["r"], **kw(t)),
         ["rows"] + five),
        ("balance backward", lambda t: ops.balance_loss_backward(t["g"], t["logits"], counts, tokens, 2), ["g", "logits"]),
        ("raw quantize", lambda t: raw.quantize_e4m3_blocks(t["rows"], False), ["rows"]),
        ("raw norm", lambda t: raw.norm_residual(*norm(t), 1.0, 1e-6, False, None), five),
        ("raw norm backward", lambda t: raw.norm_residual_backward(t["rows"], t["rows"], *norm(t), 1.0, 1e-6), five),
        ("raw balance", lambda t: raw.balance_loss(t["logits"], ids, 1.0, None), ["logits"]),
        ("raw balance backward", lambda t: raw.balance_loss_backward(t["g"], t["logits"], counts, tokens, 2, 1.0, None),
         ["g", "logits"]),
    ]


def test_gradients_that_an_op_does_not_have_are_refused(ops):
    """Every input that asks for a gradient where there is none, the raw ops' too; without grad mode they run."""
    t, calls = _calls(ops)
    for name, call, inputs in calls:
        call(t)
        for key in inputs:
            asking = {**t, key: t[key].clone().requires_grad_(True)}
            with pytest.raises(RuntimeError, match="gradient"):
                call(asking)
            with torch.no_grad():
                call(asking)


def test_tangents_are_refused(ops):
    import torch.autograd.forward_ad as fwd

    t, calls = _calls(ops)
    calls += [("norm", lambda t: ops.norm_residual(t["y"], t["r"], post_weight=t["post"], gate=t["gate"],
                                                   pre_weight=t["pre"]), ["y", "r", "post", "gate", "pre"]),
              ("balance", lambda t: ops.balance_loss(t["logits"], torch.zeros(5, 2, dtype=torch.int32, device=DEV)),
               ["logits"])]
    for name, call, inputs in calls:
        for key in inputs:
            with fwd.dual_level():
                dual = {**t, key: fwd.make_dual(t[key], torch.ones_like(t[key]))}
                with pytest.raises((RuntimeError, NotImplementedError), match="gradient|forward"):
                    call(dual)


# ------------------------------------------------------------------ sizes
def test_quantize_columns_past_32_bits(ops):
    cols = (1 << 32) + 1000 + 3  # not a multiple of 8 or 128: the kernel that keeps a row and a column index
    x = torch.zeros(1, cols, device=DEV, dtype=BF16)
    x[0, :512] = randn(512, seed=42, dtype=BF16)
    x[0, -1003:] = randn(1003, seed=43, dtype=BF16)
    q, s = ops.quantize_e4m3_blocks(x)
    first = (cols - 1003) // 128 * 128
    for lo, hi in ((0, 512), (first, cols)):
        rq, rs = ref_codes(x[:, lo:hi], 1)
        assert torch.equal(s[:, lo // 128: lo // 128 + blocks(hi - lo)], rs)
        assert torch.equal(q[:, lo:hi].contiguous().view(torch.uint8), rq.view(torch.uint8))


def test_balance_backward_refuses_a_k_past_its_range(ops):
    logits = randn(4, 8, seed=44)
    _, counts, tokens = ops.balance_loss(logits, logits.topk(2, 1).indices.to(torch.int32))
    for k in (0, 9, -1, (1 << 32) + 2):
        with pytest.raises(RuntimeError, match="k="):
            ops.balance_loss_backward(torch.ones((), device=DEV), logits, counts, tokens, k)


def test_norm_workspace_is_the_launched_grid(ops):
    """The backward's partial sums: one row per CTA of the launch, of which no SM holds more than four here."""
    v = norm_inputs(8192, 4096, BF16, BF16, "channel", True, True, wd=BF16, seed=45)
    g = randn(8192, 4096, seed=46, dtype=BF16)
    torch.cuda.synchronize()
    kept = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    d = ops.norm_residual_backward(g, g, v["y"], v["r"], post_weight=v["post"], gate=v["gate"], pre_weight=v["pre"])
    outputs = sum(t.numel() * t.element_size() for t in d if t is not None)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert torch.cuda.max_memory_allocated() - kept - outputs <= 4 * sms * 2 * 4096 * 4 + (1 << 20)


# ------------------------------------------------------------------ tracing, streams
def test_fake_implementations_match(ops):
    """Under a fake tensor mode each op gives what it really gives: shapes, types, strides."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    raw = torch.ops.stageml
    x, xs = ref_codes(randn(5, 200, seed=50), 1)
    w, ws = ref_codes(randn(130, 200, seed=51), 128)
    x, w = x[:, :192].contiguous(), w[:, :192].contiguous()
    gu, gus, dn, dns = layer_weights(3, 144, 80, seed=52)
    ids = torch.tensor([[0, 1]], dtype=torch.int32, device=DEV).repeat(5, 1)
    rows, wide = randn(5, 144, seed=53, dtype=BF16), randn(3, 5, 300, seed=54, dtype=BF16)
    v = norm_inputs(5, 300, F32, BF16, "token", True, True, seed=55)
    norm = (v["y"], v["r"], v["post"], v["gate"], v["pre"])
    bare = (None, v["r"], None, None, v["pre"])
    dr, dz = randn(5, 300, seed=56), randn(5, 300, seed=57, dtype=BF16)
    logits = randn(5, 9, seed=58, dtype=F16)
    counts, tokens = torch.ones(9, dtype=torch.int32, device=DEV), torch.full((), 5, dtype=torch.int32, device=DEV)
    calls = [
        (raw.quantize_e4m3_blocks, (wide, False)), (raw.quantize_e4m3_blocks, (wide, True)),
        (raw.quantize_e4m3_blocks, (wide[0, 0], False)),
        (raw.block_matmul, (x, xs, w, ws, F16)), (raw.block_matmul, (x, xs, w, ws, F32)),
        (raw.moe_forward_blocks, (rows, gu, gus, dn, dns, ids, torch.ones(5, 2, device=DEV), 1)),
        (raw.moe_forward_blocks, (rows, gu, gus, dn, dns, None, None, 3)),
        (raw.norm_residual, (*norm, 0.5, 1e-6, False, None)), (raw.norm_residual, (*norm, 0.5, 1e-6, True, BF16)),
        (raw.norm_residual, (*bare, 1.0, 1e-6, False, F16)), (raw.norm_residual, (*bare, 1.0, 1e-6, False, None)),
        (raw.norm_residual, (v["y"], v["r"], None, None, None, 1.0, 1e-6, False, None)),
        (raw.norm_residual, (v["y"].t().contiguous().t(), v["r"].t().contiguous().t(), None, None, v["pre"], 1.0, 1e-6,
                             False, None)),
        (raw.norm_residual_backward, (dr, dz, *norm, 0.5, 1e-6)),
        (raw.norm_residual_backward, (dr, None, *bare, 0.5, 1e-6)),
        (raw.balance_loss, (logits, ids, 0.1, None)),
        (raw.balance_loss_backward, (torch.ones((), device=DEV), logits, counts, tokens, 2, 0.1, None)),
    ]
    for op, args in calls:
        real = op(*args)
        with FakeTensorMode() as mode:
            fake = op(*[mode.from_tensor(a) if isinstance(a, torch.Tensor) else a for a in args])
        real, fake = ([o] if isinstance(o, torch.Tensor) else list(o) for o in (real, fake))
        assert len(real) == len(fake)
        for a, b in zip(real, fake):
            assert (a.shape, a.dtype, a.device, a.stride()) == (b.shape, b.dtype, b.device, b.stride()), op


def test_products_on_two_streams_at_once(ops):
    """The tile kernels of two streams share the device and nothing else: the bits of each alone."""
    small, large = [], []
    for m, n, k in ((64, 4096, 4096), (300, 1000, 2048)):  # several CTA pairs to a tile
        xs = ref_codes(randn(m, k, seed=m), 1)
        small.append((*xs, *ref_codes(randn(n, k, seed=n, scale=k ** -0.5), 128)))
    m, n, k = 1500, 2824, 1424
    large.append((*ref_codes(randn(m, k, seed=m), 1), *ref_codes(randn(n, k, seed=n, scale=k ** -0.5), 128)))
    gu, gus, dn, dns = layer_weights(6, 256, 208, seed=60)
    x = randn(700, 256, seed=61, dtype=BF16)
    top = randn(700, 6, seed=62).topk(3, 1)
    ids, w = top.indices.to(torch.int32), top.values.softmax(1)
    work = [lambda: [ops.block_matmul(*o, out_dtype=F32) for o in small],
            lambda: [ops.block_matmul(*o) for o in large] +
                    [ops.moe_forward_blocks(x, gu, gus, dn, dns, topk_ids=ids, topk_weights=w)]]
    want = [f() for f in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    got = [[], []]
    for _ in range(20):
        for s, f, g in zip(streams, work, got):
            with torch.cuda.stream(s):
                g.append(f())
    torch.cuda.synchronize()
    for g, ref in zip(got, want):
        for outs in g:
            for a, b in zip(outs, ref):
                assert torch.equal(a, b)


# ------------------------------------------------------------------ offsets past 32 bits
def test_norm_rows_past_32_bits(ops):
    """2.3e9 values: the last rows are those of the same rows alone, outputs and gradients."""
    t, h, n = 140000, 16384, 300
    g = torch.Generator(device=DEV).manual_seed(70)
    r, y, dr, dz = (torch.empty(t, h, device=DEV, dtype=BF16).normal_(generator=g) for _ in range(4))
    pre, post = 1 + randn(h, seed=71, scale=0.1), 1 + randn(h, seed=72, scale=0.1)
    args = dict(post_weight=post, pre_weight=pre)
    tail = {"y": y[-n:], "r": r[-n:], "post": post, "gate": None, "pre": pre}
    new, z = ops.norm_residual(y, r, **args)
    _, q, s = ops.norm_residual(y, r, quantize=True, **args)
    rn, rz, ref = ref_norm(tail, 1.0, 1e-6, (dr[-n:], dz[-n:]))
    close(new[-n:], rn), close(z[-n:], rz)
    assert float((dequant(q[-n:], s[-n:], 1) - rz).norm() / rz.norm()) < 0.04  # half a step of e4m3 at most: 2^-4
    del new, z, q, s
    d = ops.norm_residual_backward(dr, dz, y, r, **args)
    close(d[0][-n:], ref["r"]), close(d[1][-n:], ref["y"])


def test_layer_rows_past_32_bits(ops):
    """560000 slots of 4096 columns: the fp32 rows that are summed lie past 2^31 values; tokens of both ends."""
    t, e, k, h, i = 70000, 16, 8, 4096, 128
    gu, gus, dn, dns = layer_weights(e, h, i, seed=73)
    x = randn(t, h, seed=74, dtype=BF16)
    ids = torch.rand(t, e, generator=torch.Generator(device=DEV).manual_seed(75), device=DEV).topk(k, 1).indices.to(torch.int32)
    w = torch.rand(t, k, generator=torch.Generator(device=DEV).manual_seed(76), device=DEV)
    y = ops.moe_forward_blocks(x, gu, gus, dn, dns, topk_ids=ids, topk_weights=w)
    for part in (slice(0, 100), slice(t - 100, t)):
        close(y[part], ref_layer(x[part], gu, gus, dn, dns, ids[part], w[part], 0), LAYER_TOL[BF16])


def test_balance_logits_past_32_bits(ops):
    t, e = 8500000, 256  # 2.2e9 logits
    g = torch.Generator(device=DEV).manual_seed(77)
    logits = torch.empty(t, e, device=DEV, dtype=BF16).normal_(generator=g)
    ids = torch.randint(0, e, (t, 1), generator=g, device=DEV, dtype=torch.int32)
    loss, counts, tokens = ops.balance_loss(logits, ids)
    assert int(tokens) == t and torch.equal(counts.long(), torch.bincount(ids.view(-1), minlength=e))
    p = torch.zeros(e, dtype=torch.float64, device=DEV)
    for lo in range(0, t, 500000):
        p += torch.softmax(logits[lo:lo + 500000].double(), 1).sum(0)
    f = counts.double() / t
    # fp32 partial sums of about 150 tokens' probabilities per lane, then 3500 of those: sqrt(3500) * 2^-24
    close(loss, e * (f * p / t).sum())
    grad = ops.balance_loss_backward(torch.full((), 1e6, device=DEV), logits, counts, tokens, 1)
    x = torch.softmax(logits[-200:].double(), 1)
    ref = 1e6 * e / t * x * (f - (x * f).sum(1, keepdim=True))
    close(grad[-200:], ref)
