"""GPU tests of the block-scaled FP8 operators, the block norm and the router balance loss.

References are plain torch code in float64 on the same inputs. Tolerances (rel-L2 unless said):
- codes and scales of the quantizer: bit for bit.
- fp32 outputs: 1e-5. Sums of up to 2^14 terms in fp32 err like sqrt(terms) * 2^-24 < 8e-6.
- 16-bit outputs: the reference is rounded to the same type; what is left are values whose fp32 error
  crosses a rounding boundary. 2^-9 (bf16) and 2^-12 (f16), plus the fp32 part.
- the routed layer: each slot's row is rounded to 16 bits before the sum over slots and the sum is
  rounded again (sqrt 2 of the above), and a code of the fp32 h can fall on the other side of a
  rounding boundary than the reference's: at most one in 10^4 codes by 2^-4, 6e-4. 5e-3 and 2e-3.
"""

import math

import numpy as np
import pytest
import torch

from conftest import rel_l2

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOL32 = 1e-5
TOL = {torch.float32: TOL32, torch.bfloat16: 2.0 ** -9 + TOL32, torch.float16: 2.0 ** -12 + TOL32}
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops():
    import stageml_b200.ops as o

    return o


@pytest.fixture(autouse=True)
def clean_status(ops):
    yield
    assert ops.take_status(torch.empty(1, device=DEV)) == 0


def randn(*shape, seed=0, scale=1.0, dtype=F32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def close(got, ref, tol=None):
    tol = TOL[got.dtype] if tol is None else tol
    got, ref = got.detach().double(), ref.detach().to(got.dtype).double()
    assert got.shape == ref.shape
    assert torch.equal(got.isfinite(), ref.isfinite())
    m = ref.isfinite()
    err = float((got[m] - ref[m]).norm() / ref[m].norm().clamp(min=1e-300)) if m.any() and ref[m].norm() > 0 else \
        float(got[m].abs().sum())
    assert err <= tol, f"rel-L2 {err:.3e} > {tol:.3e}"


def blocks(n):
    return (n + 127) // 128


def ref_codes(x, high):
    """Codes (float8) and scales of x [rows, cols] in blocks of high x 128, by definition."""
    rows, cols = x.shape
    r = torch.arange(rows, device=DEV) // high
    c = torch.arange(cols, device=DEV) // 128
    nb = blocks(cols)
    a = torch.zeros((blocks(rows) if high == 128 else rows) * nb, dtype=torch.float64, device=DEV)
    a.scatter_reduce_(0, (r[:, None] * nb + c).reshape(-1), x.double().abs().reshape(-1), "amax")
    s = (a / 448).float().view(-1, nb)
    s[s == 0] = 1
    q = (x.double() / s.double()[r][:, c]).float().clamp(-448, 448).to(torch.float8_e4m3fn)
    return q, s


def dequant(q, s, high):
    rows, cols = q.shape
    r = torch.arange(rows, device=DEV) // high
    c = torch.arange(cols, device=DEV) // 128
    return q.double() * s.double()[r][:, c]


def same_bits(a, b):
    """Equal codes; a NaN's sign is free."""
    a, b = a.view(torch.uint8), b.view(torch.uint8)
    return bool(((a == b) | ((a & 0x7f == 0x7f) & (b & 0x7f == 0x7f))).all())


# ------------------------------------------------------------------ quantizer
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 7), (2, 8), (130, 129), (257, 136), (5, 1000), (64, 384),
                                       (129, 2048), (700, 4096)])
def test_quantize_codes_are_exact(ops, dtype, tiles, rows, cols):
    x = randn(rows, cols, seed=rows + cols) * torch.exp2(randn(rows, cols, seed=1) * 3)
    x[:, : min(cols, 128)][rows // 2:] = 0.0  # blocks of zeros
    x = x.to(dtype)
    q, s = ops.quantize_e4m3_blocks(x, tiles=tiles)
    rq, rs = ref_codes(x, 128 if tiles else 1)
    assert torch.equal(s, rs)
    assert same_bits(q, rq)


@pytest.mark.parametrize("exponent", [-148, -133, -120, -100, -91, -80, 40, 89, 92, 120])
def test_quantize_far_from_one(ops, exponent):
    """Scales at the ends of fp32's range, where the reciprocal is not used."""
    x = (randn(64, 512, seed=2).double() * 2.0 ** exponent).float()
    x = torch.where(x.isfinite(), x, torch.zeros_like(x))
    q, s = ops.quantize_e4m3_blocks(x)
    rq, rs = ref_codes(x, 1)
    assert torch.equal(s, rs)
    assert same_bits(q, rq)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tiles", [False, True])
def test_quantize_keeps_nan_and_infinity_visible(ops, dtype, tiles):
    x = randn(256, 384, seed=3).to(dtype)
    x[3, 5], x[200, 140], x[7, 383] = math.nan, math.inf, -math.inf
    q, s = ops.quantize_e4m3_blocks(x, tiles=tiles)
    at = (lambda r, c: (r // 128, c // 128)) if tiles else (lambda r, c: (r, c // 128))
    assert s[at(3, 5)].isnan() and s[at(200, 140)].isinf() and s[at(7, 383)].isinf()
    assert q[3, 5].float().isnan() and q[200, 140].float().isnan() and q[7, 383].float().isnan()
    clean = torch.ones_like(s, dtype=torch.bool)
    for r, c in ((3, 5), (200, 140), (7, 383)):
        clean[at(r, c)] = False
    assert s[clean].isfinite().all()


def test_quantize_batched_strided_and_empty(ops):
    w = randn(3, 200, 300, seed=4, dtype=BF16)
    q, s = ops.quantize_e4m3_blocks(w, tiles=True)
    assert q.shape == w.shape and s.shape == (3, 2, 3)
    for i in range(3):
        rq, rs = ref_codes(w[i], 128)
        assert same_bits(q[i], rq) and torch.equal(s[i], rs)
    x = randn(64, 512, seed=5, dtype=BF16)
    for view in (x[:, 1:513:2], x.t(), x[3:, 129:]):  # other strides and alignments
        q, s = ops.quantize_e4m3_blocks(view)
        rq, rs = ref_codes(view.contiguous(), 1)
        assert same_bits(q, rq) and torch.equal(s, rs)
    flat = torch.empty(64 * 256 + 3, device=DEV, dtype=BF16)[3:].view(64, 256).copy_(x[:, :256])  # rows off 16 bytes
    assert same_bits(ops.quantize_e4m3_blocks(flat)[0], ref_codes(flat, 1)[0])
    for shape in ((0, 128), (4, 0)):
        q, s = ops.quantize_e4m3_blocks(torch.empty(shape, device=DEV))
        assert q.shape == shape and s.numel() == 0


# ------------------------------------------------------------------ dense product
def operands(m, n, k, seed=0):
    x, xs = ref_codes(randn(m, k, seed=seed), 1)
    w, ws = ref_codes(randn(n, k, seed=seed + 1, scale=k ** -0.5), 128)
    return x, xs, w, ws


@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 520, 1024), (3, 130, 144), (8, 4096, 512), (9, 257, 2064), (16, 16, 48),
                                   (17, 1, 128), (17, 520, 16), (128, 256, 1152), (129, 130, 144), (300, 700, 400),
                                   (513, 127, 640), (1000, 2000, 80)])
def test_block_matmul(ops, m, n, k, out):
    x, xs, w, ws = operands(m, n, k, seed=m + n + k)
    y = ops.block_matmul(x, xs, w, ws, out_dtype=out)
    assert y.dtype == out
    close(y, dequant(x, xs, 1) @ dequant(w, ws, 128).t())


@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("m,n,k", [(17, 130, 1536), (64, 4096, 1552), (300, 500, 2048), (257, 1001, 1616), (500, 4095, 2064),
                                   (33, 8, 14336), (2048, 1027, 272), (300, 500, 3200), (257, 131, 4112)])
def test_block_matmul_shared_k_and_odd_widths(ops, m, n, k, out):
    """Few tiles with a long K, whose blocks several CTA pairs share, and rows that do not start at 16 bytes."""
    x, xs, w, ws = operands(m, n, k, seed=m + n + k)
    y = ops.block_matmul(x, xs, w, ws, out_dtype=out)
    close(y, dequant(x, xs, 1) @ dequant(w, ws, 128).t())
    for _ in range(3):
        assert torch.equal(ops.block_matmul(x, xs, w, ws, out_dtype=out), y)


@pytest.mark.parametrize("m", [1, 16, 17, 400])
def test_block_matmul_rows_do_not_mix(ops, m):
    """A row of NaN codes, or of an infinite scale, stays in its own output row."""
    x, xs, w, ws = operands(m, 300, 512, seed=9)
    ref = ops.block_matmul(x, xs, w, ws, out_dtype=F32)
    bad = x.view(torch.uint8).clone()
    bad[m // 2] = 0x7f
    y = ops.block_matmul(bad.view(torch.float8_e4m3fn), xs, w, ws, out_dtype=F32)
    keep = torch.arange(m, device=DEV) != m // 2
    assert torch.equal(y[keep], ref[keep]) and y[m // 2].isnan().all()
    xs = xs.clone()
    xs[m // 2] = 0.0
    y = ops.block_matmul(x, xs, w, ws, out_dtype=F32)
    assert torch.equal(y[keep], ref[keep]) and (y[m // 2] == 0).all()


@pytest.mark.parametrize("m", [1, 40])
def test_block_matmul_zero_rows_and_strides(ops, m):
    x, xs, w, ws = operands(m, 64, 256, seed=11)
    wt = w.view(torch.uint8).t().contiguous().t().view(torch.float8_e4m3fn)  # column-major weights
    assert torch.equal(ops.block_matmul(x, xs, wt, ws, out_dtype=F32), ops.block_matmul(x, xs, w, ws, out_dtype=F32))
    assert ops.block_matmul(x[:0], xs[:0], w, ws).shape == (0, 64)
    assert ops.block_matmul(x, xs, w[:0], ws[:0]).shape == (m, 0)


@pytest.mark.parametrize("m", [1, 24])
def test_block_matmul_offsets_past_32_bits(ops, m):
    n, k = 140000, 16384  # 2.3e9 bytes of weights
    g = torch.Generator(device=DEV).manual_seed(5)
    w = torch.randint(0, 0x78, (n, k), generator=g, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn)
    ws = torch.rand(blocks(n), k // 128, generator=g, device=DEV) + 0.5
    x, xs = ref_codes(randn(m, k, seed=6), 1)
    y = ops.block_matmul(x, xs, w, ws, out_dtype=F32)
    xd = dequant(x, xs, 1)
    for lo in (0, 131072 - 64, n - 100):  # 131072 rows are 2^31 bytes
        hi = min(lo + 128, n)
        cols = torch.arange(lo, hi, device=DEV)
        wd = w[lo:hi].double() * ws.double()[cols // 128].repeat_interleave(128, 1)
        close(y[:, lo:hi], xd @ wd.t())


# ------------------------------------------------------------------ routed layer
def ref_layer(x, gu, gus, dn, dns, ids, weights, n_shared):
    t, h = x.shape
    e_tot, two_i, _ = gu.shape
    i = two_i // 2
    xd = dequant(*ref_codes(x.float(), 1), 1)
    out = torch.zeros(t, h, dtype=torch.float64, device=DEV)

    def expert(j, rows, w):
        y = xd[rows] @ dequant(gu[j], gus[j], 128).t()
        act = torch.nn.functional.silu(y[:, :i]) * y[:, i:]
        act = dequant(*ref_codes(act.float(), 1), 1)
        out.index_add_(0, rows, (act @ dequant(dn[j], dns[j], 128).t()) * w[:, None])

    for j in range(e_tot - n_shared):
        if ids is not None:
            token, slot = (ids == j).nonzero(as_tuple=True)
            if token.numel():
                expert(j, token, weights.double()[token, slot])
    for j in range(e_tot - n_shared, e_tot):
        expert(j, torch.arange(t, device=DEV), torch.ones(t, dtype=torch.float64, device=DEV))
    return out


def layer_weights(e, h, i, seed=0):
    def stack(shape, scale):
        parts = [ref_codes(randn(*shape, seed=seed + j, scale=scale), 128) for j in range(e)]
        return (torch.stack([q.view(torch.uint8) for q, _ in parts]).view(torch.float8_e4m3fn),
                torch.stack([s for _, s in parts]))

    gu, gus = stack((2 * i, h), h ** -0.5)
    dn, dns = stack((h, i), i ** -0.5)
    return gu, gus, dn, dns


LAYER_TOL = {BF16: 5e-3, F16: 2e-3}


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("t,e,k,shared,h,i", [(1, 4, 2, 0, 128, 128), (1, 1, 1, 0, 16, 16), (7, 8, 2, 1, 256, 144),
                                              (16, 5, 3, 0, 400, 208), (17, 5, 3, 2, 400, 208), (40, 3, 1, 0, 144, 1040),
                                              (300, 8, 2, 0, 512, 384), (700, 6, 6, 1, 128, 48), (130, 64, 4, 0, 64, 80)])
def test_moe_forward_blocks(ops, dtype, t, e, k, shared, h, i):
    gu, gus, dn, dns = layer_weights(e + shared, h, i, seed=t)
    x = randn(t, h, seed=t + 1, dtype=dtype)
    top = randn(t, e, seed=t + 2).topk(k, 1)
    ids, w = top.indices.to(torch.int32), top.values.softmax(1)
    y = ops.moe_forward_blocks(x, gu, gus, dn, dns, topk_ids=ids, topk_weights=w, n_shared=shared)
    ref = ref_layer(x, gu, gus, dn, dns, ids, w, shared)
    close(y, ref, LAYER_TOL[dtype])
    # other index and weight types
    y2 = ops.moe_forward_blocks(x, gu, gus, dn, dns, topk_ids=ids.long(), topk_weights=w, n_shared=shared)
    assert torch.equal(y, y2)
    w16 = w.to(BF16)
    close(ops.moe_forward_blocks(x, gu, gus, dn, dns, topk_ids=ids, topk_weights=w16, n_shared=shared),
          ref_layer(x, gu, gus, dn, dns, ids, w16, shared), LAYER_TOL[dtype])


@pytest.mark.parametrize("t", [5, 16, 200])
def test_moe_forward_blocks_routing_edges(ops, t):
    """All tokens on one expert, an expert named several times by a token, shared experts alone, no tokens."""
    e, h, i = 6, 192, 160
    gu, gus, dn, dns = layer_weights(e, h, i, seed=3)
    x = randn(t, h, seed=4, dtype=BF16)
    w = torch.rand(t, 4, device=DEV)
    for ids in (torch.full((t, 4), 2, dtype=torch.int32, device=DEV),
                torch.tensor([1, 5, 1, 1], dtype=torch.int32, device=DEV).repeat(t, 1)):
        close(ops.moe_forward_blocks(x, gu, gus, dn, dns, topk_ids=ids, topk_weights=w),
              ref_layer(x, gu, gus, dn, dns, ids, w, 0), LAYER_TOL[BF16])
    close(ops.moe_forward_blocks(x, gu[:2], gus[:2], dn[:2], dns[:2], n_shared=2),
          ref_layer(x, gu[:2], gus[:2], dn[:2], dns[:2], None, None, 2), LAYER_TOL[BF16])
    none = ops.moe_forward_blocks(x[:0], gu, gus, dn, dns, topk_ids=ids[:0], topk_weights=w[:0])
    assert none.shape == (0, h)


@pytest.mark.parametrize("t,e,k,shared", [(17, 64, 4, 1), (100, 128, 4, 0), (128, 64, 2, 2), (43, 64, 6, 0), (60, 128, 4, 1)])
@pytest.mark.parametrize("skew", [False, True])
def test_moe_forward_blocks_few_rows_per_expert(ops, t, e, k, shared, skew):
    """More than 16 tokens, few per expert on average; skewed, all slots name one expert (several row tiles)."""
    h, i = 144, 80
    gu, gus, dn, dns = layer_weights(e + shared, h, i, seed=5)
    x = randn(t, h, seed=6, dtype=BF16)
    ids = torch.full((t, k), e - 3, device=DEV, dtype=torch.int32) if skew else \
        randn(t, e, seed=7).topk(k, 1).indices.to(torch.int32)
    w = torch.rand(t, k, generator=torch.Generator(device=DEV).manual_seed(8), device=DEV)
    y = ops.moe_forward_blocks(x, gu, gus, dn, dns, topk_ids=ids, topk_weights=w, n_shared=shared)
    close(y, ref_layer(x, gu, gus, dn, dns, ids, w, shared), LAYER_TOL[BF16])


@pytest.mark.parametrize("t", [3, 150])
def test_moe_forward_blocks_bad_ids_are_dropped_and_reported(ops, t):
    e, h, i = 4, 128, 128
    gu, gus, dn, dns = layer_weights(e, h, i, seed=7)
    x = randn(t, h, seed=8, dtype=BF16)
    ids = torch.randint(0, e, (t, 2), device=DEV, dtype=torch.int32)
    ids[1, 0], ids[2, 1] = e + 3, -1
    w = torch.rand(t, 2, device=DEV)
    y = ops.moe_forward_blocks(x, gu, gus, dn, dns, topk_ids=ids, topk_weights=w)
    assert ops.take_status(x) == 110
    close(y, ref_layer(x, gu, gus, dn, dns, ids, w, 0), LAYER_TOL[BF16])


# ------------------------------------------------------------------ block norm
def norm_inputs(t, h, rd, bd, gate, post, pre, with_y=True, wd=F32, seed=0):
    shape = {"none": None, "channel": (h,), "token": (t, 1), "full": (t, h)}[gate]
    return {
        "y": randn(t, h, seed=seed, scale=0.7, dtype=bd) if with_y else None,
        "r": randn(t, h, seed=seed + 1, dtype=rd),
        "post": (1 + randn(h, seed=seed + 2, scale=0.2)).to(wd) if post else None,
        "gate": None if shape is None else (0.5 + randn(*shape, seed=seed + 3, scale=0.3)).to(wd),
        "pre": (1 + randn(h, seed=seed + 4, scale=0.2)).to(wd) if pre else None,
    }


def ref_norm(v, alpha, eps, grad=None):
    """(r', z or None), and the gradients of y, r, post, gate, pre (None where absent) for grad = (dr', dz)."""
    d = {k: None if t is None else t.detach().double().requires_grad_(grad is not None) for k, t in v.items()}
    rms = lambda a: a * (a.square().mean(-1, keepdim=True) + eps).rsqrt()  # noqa: E731
    new = alpha * d["r"]
    if d["y"] is not None:
        u = d["y"] if d["post"] is None else rms(d["y"]) * d["post"]
        new = new + (u if d["gate"] is None else u * d["gate"])
    z = None if d["pre"] is None else rms(new) * d["pre"]
    if grad is None:
        return new, z
    heads, grads = zip(*[(o, g.double()) for o, g in zip((new, z), grad) if o is not None and g is not None])
    leaves = [k for k in d if d[k] is not None]
    got = torch.autograd.grad(heads, [d[k] for k in leaves], grads, allow_unused=True)
    return new.detach(), None if z is None else z.detach(), dict(zip(leaves, got))


NORM_DTYPES = [(BF16, BF16), (F16, F16), (F32, F32), (F32, BF16), (F32, F16)]
NORM_CASES = [
    # t, h, gate, post, pre, with block rows
    (1, 8, "none", True, True, True), (1, 4096, "channel", True, True, True), (5, 1, "token", True, True, True),
    (3, 40, "full", True, True, True), (2, 257, "channel", False, True, True), (9, 256, "token", False, True, True),
    (4, 264, "none", False, False, True), (311, 264, "channel", True, True, True), (311, 31, "full", True, True, True),
    (320, 1000, "token", True, True, True), (320, 1003, "channel", True, True, True), (300, 2048, "full", True, True, True),
    (7, 4104, "none", True, True, True), (299, 4104, "token", True, True, True), (298, 4099, "channel", True, False, True),
    (5, 8200, "channel", True, True, True), (310, 8200, "none", True, True, True), (3, 16384, "token", True, True, True),
    (305, 16384, "channel", True, True, True), (330, 1536, "none", False, True, False), (2, 24, "none", False, True, False),
]


@pytest.mark.parametrize("rd,bd", NORM_DTYPES)
@pytest.mark.parametrize("t,h,gate,post,pre,with_y", NORM_CASES)
def test_norm_residual_and_gradients(ops, rd, bd, t, h, gate, post, pre, with_y):
    alpha, eps = 0.75, 1e-5
    wd = bd if h % 3 == 0 else F32
    v = norm_inputs(t, h, rd, bd, gate, post, pre, with_y, wd, seed=h)
    if t > 2 and with_y:
        v["y"][1] = 0  # a row of zeros: its norm is 0 / sqrt(eps)
    args = dict(post_weight=v["post"], gate=v["gate"], pre_weight=v["pre"], residual_scale=alpha, eps=eps)
    out = ops.norm_residual(v["y"], v["r"], normed_dtype=bd, **args)
    grads = (randn(t, h, seed=21, dtype=rd), randn(t, h, seed=22, dtype=bd) if pre else None)
    new, z, ref = ref_norm(v, alpha, eps, grads)
    assert out[0].dtype == rd and len(out) == (2 if pre else 1)
    close(out[0], new)
    if pre:
        assert out[1].dtype == bd
        close(out[1], z)
    d = ops.norm_residual_backward(grads[0], grads[1], v["y"], v["r"], **args)
    for got, key in zip(d, ("r", "y", "post", "gate", "pre")):
        assert (got is None) == (v[key] is None)
        if got is not None:
            assert got.dtype == v[key].dtype and got.shape == v[key].shape
            close(got, ref[key])


@pytest.mark.parametrize("t,h", [(4, 512), (400, 512), (6, 33), (350, 5000)])
@pytest.mark.parametrize("which", ["residual", "normed"])
def test_norm_residual_backward_with_one_gradient(ops, t, h, which):
    v = norm_inputs(t, h, F32, F32, "channel", True, True)
    grads = (randn(t, h, seed=31), None) if which == "residual" else (None, randn(t, h, seed=32))
    _, _, ref = ref_norm(v, 1.0, 1e-6, grads)
    d = ops.norm_residual_backward(*grads, v["y"], v["r"], post_weight=v["post"], gate=v["gate"], pre_weight=v["pre"])
    for got, key in zip(d, ("r", "y", "post", "gate", "pre")):
        close(got, torch.zeros_like(got, dtype=torch.float64) if ref[key] is None else ref[key])


@pytest.mark.parametrize("gate", ["channel", "token", "full"])
def test_norm_residual_gradient_against_differences(ops, gate):
    """<gradient, direction> against a central difference of the op's own fp32 outputs (step 1e-2: truncation
    about 1e-4 of the slope, rounding 2^-24 |L| / step about 3e-4)."""
    t, h, step = 3, 40, 1e-2
    v = norm_inputs(t, h, F32, F32, gate, True, True, seed=5)
    gr, gz = randn(t, h, seed=6), randn(t, h, seed=7)

    def loss(u):
        new, z = ops.norm_residual(u["y"], u["r"], post_weight=u["post"], gate=u["gate"], pre_weight=u["pre"],
                                   residual_scale=0.9)
        return float((new.double() * gr).sum() + (z.double() * gz).sum())

    d = dict(zip(("r", "y", "post", "gate", "pre"),
                 ops.norm_residual_backward(gr, gz, v["y"], v["r"], post_weight=v["post"], gate=v["gate"],
                                            pre_weight=v["pre"], residual_scale=0.9)))
    for key in d:
        way = randn(*v[key].shape, seed=8)
        way = way / way.norm()
        slope = (loss({**v, key: v[key] + step * way}) - loss({**v, key: v[key] - step * way})) / (2 * step)
        want = float((d[key].double() * way).sum())
        assert abs(slope - want) <= 5e-3 * max(1.0, float(d[key].norm())), key


def test_norm_residual_autograd(ops):
    t, h = 37, 96
    v = norm_inputs(t, h, F32, BF16, "token", True, True, seed=40)
    leaves = {k: x.clone().requires_grad_(True) for k, x in v.items()}
    new, z = ops.norm_residual(leaves["y"].view(1, t, h), leaves["r"].view(1, t, h), post_weight=leaves["post"],
                               gate=leaves["gate"].view(1, t, 1), pre_weight=leaves["pre"], residual_scale=0.5)
    assert new.shape == (1, t, h) and z.dtype == BF16
    (new.sum() + 2 * z.float().sum()).backward()  # expanded, non-contiguous gradients
    ones = (torch.ones(t, h, device=DEV), torch.full((t, h), 2.0, device=DEV))
    _, _, ref = ref_norm(v, 0.5, 1e-6, ones)
    for k in leaves:
        close(leaves[k].grad, ref[k])
    y = v["y"].clone().requires_grad_(True)
    ops.norm_residual(y, v["r"])[0].sum().backward()  # no norms, no gate: the gradient passes through
    assert (y.grad == 1).all()


@pytest.mark.parametrize("rd,bd", [(BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("t,h", [(1, 4096), (3, 24), (5, 200), (311, 264), (2, 333), (300, 2048), (4, 16384)])
def test_norm_residual_codes(ops, rd, bd, t, h):
    """The codes are those of the fp32 z: each within half a step of e4m3 (2^-4 of the value, 2^-10 of the scale)
    and each scale within fp32 rounding of max|z| / 448."""
    v = norm_inputs(t, h, rd, bd, "channel", True, True, seed=h)
    new, q, s = ops.norm_residual(v["y"], v["r"], post_weight=v["post"], gate=v["gate"], pre_weight=v["pre"],
                                  quantize=True)
    rn, z = ref_norm(v, 1.0, 1e-6)
    close(new, rn)
    assert q.dtype == torch.float8_e4m3fn and s.shape == (t, blocks(h))
    _, rs = ref_codes(z.float(), 1)
    assert float((s - rs).abs().max() / rs.max()) <= 1e-5
    dq = dequant(q, s, 1)
    wide = rs.double().repeat_interleave(128, 1)[:, :h]
    assert ((dq - z).abs() <= z.abs() * (2.0 ** -4 + 1e-4) + wide * 2.0 ** -10 * 1.001).all()
    plain = ops.norm_residual(v["y"], v["r"], post_weight=v["post"], gate=v["gate"], pre_weight=v["pre"])
    assert torch.equal(plain[0], new)


def test_norm_residual_strides_alignment_and_empty(ops):
    t, h = 310, 64
    wide = randn(t, 2 * h + 3, seed=50, dtype=BF16)
    r, y = wide[:, 3:3 + h], wide[:, h + 3:]  # strided views at odd offsets
    w = randn(h + 1, seed=51)[1:]
    out = ops.norm_residual(y, r, post_weight=w, pre_weight=w)
    ref = ref_norm({"y": y, "r": r, "post": w, "gate": None, "pre": w}, 1.0, 1e-6)
    close(out[0], ref[0]), close(out[1], ref[1])
    empty = torch.empty(0, h, device=DEV, dtype=BF16)
    for gate in (w, empty, empty[:, :1]):
        new, z = ops.norm_residual(empty, empty, post_weight=w, gate=gate, pre_weight=w)
        assert new.shape == z.shape == (0, h)
        d = ops.norm_residual_backward(empty, empty, empty, empty, post_weight=w, gate=gate, pre_weight=w)
        assert d[0].shape == (0, h) and d[3].shape == gate.shape and all((g == 0).all() for g in d[2:])


def test_norm_residual_same_bits_every_run(ops):
    v = norm_inputs(2000, 1024, BF16, BF16, "channel", True, True, wd=F32, seed=60)
    g = randn(2000, 1024, seed=61, dtype=BF16), randn(2000, 1024, seed=62, dtype=BF16)
    run = lambda: ops.norm_residual_backward(*g, v["y"], v["r"], post_weight=v["post"], gate=v["gate"],  # noqa: E731
                                             pre_weight=v["pre"])
    first = run()
    for _ in range(3):
        for a, b in zip(first, run()):
            assert torch.equal(a, b)


# ------------------------------------------------------------------ balance loss
def ref_balance(logits, ids, coef, valid, g):
    t, e = logits.shape
    x = logits.detach().double().requires_grad_(True)
    m = torch.ones(t, dtype=torch.bool, device=DEV) if valid is None else valid.bool()
    counts = torch.stack([((ids == j) & m[:, None]).sum() for j in range(e)])
    n = max(1, int(m.sum()))
    p = torch.nan_to_num(torch.softmax(x, 1), nan=0.0) if bool(torch.isneginf(logits).all(1).any()) else torch.softmax(x, 1)
    p = torch.where(m[:, None], p, torch.zeros_like(p))
    loss = coef * e * (counts.double() / (n * ids.shape[1]) * (p.sum(0) / n)).sum()
    grad, = torch.autograd.grad(loss * g, x)
    return loss.detach(), counts, torch.nan_to_num(grad, nan=0.0)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (1, 8, 2), (7, 2, 1), (300, 3, 2), (256, 8, 2), (999, 31, 4), (513, 60, 6),
                                   (1000, 64, 6), (777, 128, 8), (2000, 160, 8), (5000, 256, 8), (20000, 16, 1)])
def test_balance_loss(ops, dtype, t, e, k):
    logits = (randn(t, e, seed=t) + 0.5 * randn(1, e, seed=1)).to(dtype)
    ids = logits.float().topk(k, 1).indices
    for valid, kind in ((None, torch.int32), (torch.rand(t, device=DEV) < 0.7, torch.int64)):
        loss, counts, tokens = ops.balance_loss(logits, ids.to(kind), 0.02, valid=valid)
        ref, rc, rg = ref_balance(logits, ids, 0.02, valid, 1.5)
        assert counts.dtype == torch.int32 and torch.equal(counts.long(), rc)
        assert int(tokens) == (t if valid is None else int(valid.sum()))
        close(loss, ref)
        grad = ops.balance_loss_backward(torch.full((), 1.5, device=DEV), logits, counts, tokens, k, 0.02, valid=valid)
        assert grad.dtype == dtype
        if k == e:  # every expert chosen by every token: no gradient but rounding
            assert float(grad.abs().max()) <= 1e-7
        elif float(rg.norm()) > 0:
            # f16 gradients lie among its subnormals: their step, 2^-24, is the absolute part
            assert float((grad.double() - rg.to(dtype).double()).norm()) <= TOL[dtype] * float(rg.norm()) + \
                (2.0 ** -25 * math.sqrt(t * e) if dtype == F16 else 0.0)


@pytest.mark.parametrize("t,e", [(40, 5), (40, 64), (4000, 200)])
def test_balance_loss_masked_rows(ops, t, e):
    """Experts out of service, a token without any, slots without an expert, and nothing valid at all."""
    logits = randn(t, e, seed=2)
    logits[:, 1] = -math.inf
    logits[3] = -math.inf
    ids = logits.topk(2, 1).indices.to(torch.int32)
    ids[3] = -1
    ids[5, 1] = -1
    loss, counts, tokens = ops.balance_loss(logits, ids, 1.0)
    ref, rc, rg = ref_balance(logits, ids, 1.0, None, 1.0)
    assert torch.equal(counts.long(), rc)
    close(loss, ref)
    grad = ops.balance_loss_backward(torch.ones((), device=DEV), logits, counts, tokens, 2)
    close(grad, rg)
    assert (grad[3] == 0).all() and (grad[:, 1] == 0).all()
    none = torch.zeros(t, dtype=torch.bool, device=DEV)
    loss, counts, tokens = ops.balance_loss(logits, ids, 1.0, valid=none)
    assert float(loss) == 0 and int(tokens) == 0 and (counts == 0).all()
    grad = ops.balance_loss_backward(torch.ones((), device=DEV), logits, counts, tokens, 2, valid=none)
    assert (grad == 0).all()
    logits[7, 2] = math.nan  # is not hidden
    assert ops.balance_loss(logits, ids)[0].isnan()


def test_balance_loss_bad_ids_and_empty(ops):
    logits = randn(50, 8, seed=3)
    ids = logits.topk(2, 1).indices.to(torch.int32)
    ids[4, 0] = 8
    _, counts, _ = ops.balance_loss(logits, ids)
    assert ops.take_status(logits) == 110 and int(counts.sum()) == 99
    loss, counts, tokens = ops.balance_loss(logits[:0], ids[:0])
    assert float(loss) == 0 and int(tokens) == 0 and (counts == 0).all()


def test_balance_loss_autograd_and_differences(ops):
    t, e, k = 30, 12, 3
    logits = randn(t, e, seed=9).requires_grad_(True)
    ids = logits.detach().topk(k, 1).indices.to(torch.int32)
    loss, counts, tokens = ops.balance_loss(logits, ids, 2.0)
    (3 * loss).backward()
    _, _, rg = ref_balance(logits, ids, 2.0, None, 3.0)
    close(logits.grad, rg)
    way = randn(t, e, seed=10)
    way = way / way.norm()
    at = lambda s: float(ops.balance_loss(logits.detach() + s * way, ids, 2.0)[0])  # noqa: E731
    # step 0.1: truncation about (0.1 / sqrt(t e))^2 of the slope, rounding 2^-24 * 2 / 0.1
    slope = 3 * (at(0.1) - at(-0.1)) / 0.2
    want = float((logits.grad.double() * way).sum())
    assert abs(slope - want) <= 1e-2 * float(logits.grad.norm()) + 4e-6
    assert not counts.requires_grad and not tokens.requires_grad


@pytest.mark.parametrize("t,e", [(512, 64), (30000, 256)])
def test_balance_loss_same_bits_every_run(ops, t, e):
    logits = randn(t, e, seed=11)
    ids = logits.topk(4, 1).indices.to(torch.int32)
    first = ops.balance_loss(logits, ids)
    for _ in range(5):
        for a, b in zip(first, ops.balance_loss(logits, ids)):
            assert torch.equal(a, b)


# ------------------------------------------------------------------ refusals, streams, the sublayer
def test_refusals(ops):
    x, xs, w, ws = operands(4, 64, 256)
    cases = [
        (lambda: ops.quantize_e4m3_blocks(torch.zeros(4, 128)), "CUDA"),
        (lambda: ops.quantize_e4m3_blocks(torch.zeros(4, 128, device=DEV, dtype=torch.int32)), "float32"),
        (lambda: ops.quantize_e4m3_blocks(torch.zeros(128, device=DEV), tiles=True), "dims"),
        (lambda: ops.quantize_e4m3_blocks(torch.zeros(4, 128, device=DEV, requires_grad=True)), "gradient"),
        (lambda: ops.block_matmul(x.cpu(), xs, w, ws), "CUDA"),
        (lambda: ops.block_matmul(x.float(), xs, w, ws), "float8_e4m3fn"),
        (lambda: ops.block_matmul(x, xs[:, :1], w, ws), "x_scale"),
        (lambda: ops.block_matmul(x, xs, w, ws.t()), "w_scale"),
        (lambda: ops.block_matmul(x, xs, w[:, :128], ws), r"\[M, K\]"),
        (lambda: ops.block_matmul(x, xs, w, ws, out_dtype=torch.float64), "out_dtype"),
        (lambda: ops.block_matmul(*operands(4, 64, 24)[:3], operands(4, 64, 24)[3]), "multiple of 16"),
    ]
    gu, gus, dn, dns = layer_weights(3, 128, 128)
    h = randn(4, 128, dtype=BF16)
    ids = torch.zeros(4, 2, dtype=torch.int32, device=DEV)
    wt = torch.ones(4, 2, device=DEV)
    layer = lambda **kw: ops.moe_forward_blocks(  # noqa: E731
        kw.get("x", h), kw.get("gu", gu), kw.get("gus", gus), kw.get("dn", dn), kw.get("dns", dns),
        topk_ids=kw.get("ids", ids), topk_weights=kw.get("wt", wt), n_shared=kw.get("n_shared", 0))
    cases += [
        (lambda: layer(x=h.float()), "bfloat16 or float16"),
        (lambda: layer(gu=gu.float()), "float8_e4m3fn"),
        (lambda: layer(gus=gus[:, :1]), "gate_up_scale"),
        (lambda: layer(dn=dn[:2]), "do not match"),
        (lambda: layer(ids=None), "go together"),
        (lambda: layer(ids=ids[:3], wt=wt[:3]), r"\[T, k\]"),
        (lambda: layer(ids=ids.repeat(1, 2), wt=wt.repeat(1, 2)), "min"),
        (lambda: layer(n_shared=4), "n_shared"),
        (lambda: layer(x=h.clone().requires_grad_(True)), "gradient"),
    ]
    r = randn(4, 64, dtype=BF16)
    n = ops.norm_residual
    cases += [
        (lambda: n(r.cpu(), r), "must be on|CUDA"),
        (lambda: n(r.float(), r), "residual"),
        (lambda: n(r[:, :32], r), "shape"),
        (lambda: n(r, r, gate=torch.ones(5, device=DEV)), "gate"),
        (lambda: n(r, r, post_weight=torch.ones(63, device=DEV)), "weight"),
        (lambda: n(None, r, post_weight=torch.ones(64, device=DEV)), "block_out"),
        (lambda: n(r, r, quantize=True), "pre_weight"),
        (lambda: n(r, r, pre_weight=torch.ones(64, device=DEV, dtype=torch.float64)), "float32"),
        (lambda: n(None, torch.zeros(2, 16392, device=DEV), pre_weight=torch.ones(16392, device=DEV)), "16384"),
        (lambda: n(r.clone().requires_grad_(True), r, pre_weight=torch.ones(64, device=DEV), quantize=True), "gradient"),
        (lambda: ops.norm_residual_backward(None, None, r, r), "no gradient"),
        (lambda: ops.norm_residual_backward(r, r, r, r), "pre_weight"),
        (lambda: ops.norm_residual_backward(r.float(), None, r, r), "grad_residual"),
    ]
    lg = randn(4, 8)
    cases += [
        (lambda: ops.balance_loss(lg.cpu(), ids.cpu()), "CUDA"),
        (lambda: ops.balance_loss(randn(4, 300), ids), "256"),
        (lambda: ops.balance_loss(lg, ids[:3]), r"\[T, k\]"),
        (lambda: ops.balance_loss(lg, ids.float()), "ids"),
        (lambda: ops.balance_loss(lg, ids, valid=torch.ones(5, dtype=torch.bool, device=DEV)), "valid"),
        (lambda: ops.balance_loss(lg, ids.repeat(1, 5)), "k="),
        (lambda: ops.balance_loss_backward(torch.ones(2, device=DEV), lg, ids, ids, 2), "grad_loss"),
        (lambda: ops.balance_loss_backward(torch.ones((), device=DEV), lg, ids, ids, 2), "counts"),
    ]
    for call, text in cases:
        with pytest.raises((RuntimeError, ValueError), match=text):
            call()


def test_other_streams_and_graph_capture(ops):
    """Each op runs on the current stream: results produced there are seen, and a captured graph replays them."""
    x = randn(333, 512, seed=70, dtype=BF16)
    w, ws = ref_codes(randn(640, 512, seed=71), 128)
    logits = randn(333, 64, seed=72)
    ids = logits.topk(4, 1).indices.to(torch.int32)
    pre = torch.ones(512, device=DEV)

    def step(src):
        new, q, s = ops.norm_residual(src, src, post_weight=pre, pre_weight=pre, quantize=True)
        y = ops.block_matmul(q, s, w, ws, out_dtype=F32)
        loss, counts, tokens = ops.balance_loss(logits, ids)
        return new, y, loss, ops.balance_loss_backward(loss, logits, counts, tokens, 4)

    want = step(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.zeros_like(x)
        torch.cuda._sleep(2_000_000)
        late.copy_(x)
        got = step(late)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    src = torch.zeros_like(x)
    step(src)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(src)
    src.copy_(x)
    graph.replay()
    for a, b in zip(want, captured):
        assert torch.equal(a, b)


@pytest.mark.parametrize("t", [6, 200])
def test_feed_forward_block(ops, t):
    from stageml_b200.ffn_block import FeedForwardBlock

    e, k, h, i = 8, 2, 256, 160
    block = FeedForwardBlock(randn(e, h, seed=80, scale=h ** -0.5), randn(e + 1, 2 * i, h, seed=81, scale=h ** -0.5, dtype=BF16),
                             randn(e + 1, h, i, seed=82, scale=i ** -0.5, dtype=BF16), k, n_shared=1,
                             pre_weight=1 + randn(h, seed=83, scale=0.1), post_weight=1 + randn(h, seed=84, scale=0.1),
                             gate=randn(h, seed=85, scale=0.3), residual_scale=0.9).to(DEV)
    x = randn(2, t // 2, h, seed=86, dtype=BF16)
    residual, normed = block.start(x)
    new, nxt = block(residual, normed, next_pre_weight=block.pre_weight)
    # the same from the definitions
    rows = x.view(-1, h)
    _, z = ref_norm({"y": None, "r": rows, "post": None, "gate": None, "pre": block.pre_weight}, 1.0, 1e-6)
    close(normed.view(-1, h), z)
    flat = normed.detach().view(-1, h)
    ids, w, _ = ops.route_topk(flat, block.router_w.detach(), k)
    y = ref_layer(flat, block.gate_up, block.gate_up_scale, block.down, block.down_scale, ids, w, 1)
    rn, rz = ref_norm({"y": y, "r": rows, "post": block.post_weight, "gate": block.gate, "pre": block.pre_weight}, 0.9, 1e-6)
    close(new.view(-1, h), rn, LAYER_TOL[BF16])
    close(nxt.view(-1, h), rz, 2 * LAYER_TOL[BF16])
    # training: the norms' weights and the gate from the stream, the router from the balance loss
    (new.float().square().mean() + nxt.float().mean()).backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in (block.post_weight, block.gate, block.pre_weight))
    sgd = torch.optim.SGD([block.router_w], lr=5.0)
    first = None
    for _ in range(60):
        loss, counts, tokens = block.balance(normed.detach())
        assert int(counts.sum()) == k * int(tokens)
        first = float(loss.detach()) if first is None else first
        sgd.zero_grad()
        loss.backward()
        sgd.step()
    assert float(loss.detach()) < first
