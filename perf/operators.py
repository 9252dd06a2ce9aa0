"""Measured cases of the feed-forward sublayer's operators around the MoE layer.

Four operators, each in its plain form (elementary torch operations in 32 bits) and through the
framework's entry points (``own = True``):

``quantize``  e4m3 codes with one fp32 scale per 128 values of a row, or per 128 x 128 tile
              (``ops.quantize_e4m3_blocks``)
``matmul``    y = x w^T on such operands (``ops.block_matmul``)
``experts``   the routed SwiGLU feed-forward layer on such weights (``ops.moe_forward_blocks``)
``norm``      r' = a r + gate * (norm(y) w_post), z = norm(r') w_pre, and the gradients
              (``ops.norm_residual``, ``ops.norm_residual_backward``)
``balance``   the router's balance loss, its counts per expert and the logits' gradient
              (``ops.balance_loss``, ``ops.balance_loss_backward``)

A case is a dict of plain values; ``prepare`` makes what a program has in hand before the call,
``run`` makes one pass, ``work`` counts what a pass cannot do without, and ``exact`` computes the
same outputs from the definitions in 64 bits.
"""

import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


def blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _scale(amax):
    """amax / 448, correctly rounded (a tensor divides by a Python number as a product), 1 for a block of zeros."""
    s = amax / torch.full_like(amax, E4M3_MAX)
    return torch.where(s == 0, torch.ones_like(s), s)


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # the activations of a prefill batch of the Mixtral-shape layer, before its expert products
        {"name": "quantize_rows", "op": "quantize", "rows": 8192, "cols": 4096, "dtype": "bf16", "tiles": False},
        # weights of the fine-grained layer's fused gate/up projection at load time, off the 128 grid
        {"name": "quantize_tiles", "op": "quantize", "rows": 2800, "cols": 2056, "dtype": "bf16", "tiles": True},
        # one token of a decode step through a 4096 x 4096 projection: latency and weight bytes
        {"name": "matmul_token", "op": "matmul", "m": 1, "n": 4096, "k": 4096, "out": "bf16"},
        # a ragged batch of chunked prefill, no dimension on the tile grid
        {"name": "matmul_ragged", "op": "matmul", "m": 333, "n": 2824, "k": 1424, "out": "f16"},
        # a prefill batch through the decoder block's widest projection
        {"name": "matmul_prefill", "op": "matmul", "m": 2048, "n": 11008, "k": 4096, "out": "bf16"},
        # a decode step of eight sequences through the fine-grained layer: most experts see one row
        {"name": "experts_decode", "op": "experts", "t": 8, "e": 64, "top": 6, "shared": 2, "h": 2048, "i": 1408,
         "dtype": "bf16", "skew": 0.0},
        # a prefill batch through the Mixtral-shape layer
        {"name": "experts_prefill", "op": "experts", "t": 2048, "e": 8, "top": 2, "shared": 0, "h": 4096, "i": 14336,
         "dtype": "bf16", "skew": 0.0},
        # one token of a decode step, normalised straight into the codes that the products read
        {"name": "norm_token", "op": "norm", "t": 1, "h": 4096, "resid": "bf16", "block": "bf16", "block_out": True,
         "post": True, "gate": "channel", "pre": True, "codes": True, "backward": False, "weights": "f32"},
        # a ragged training batch with an fp32 residual stream and an odd width, a gate per token
        {"name": "norm_ragged", "op": "norm", "t": 777, "h": 2047, "resid": "f32", "block": "bf16", "block_out": True,
         "post": True, "gate": "token", "pre": True, "codes": False, "backward": True, "weights": "f32"},
        # a training batch at the Mixtral-shape width: forward, then every gradient
        {"name": "norm_train", "op": "norm", "t": 8192, "h": 4096, "resid": "bf16", "block": "bf16",
         "block_out": True, "post": True, "gate": "channel", "pre": True, "codes": False, "backward": True,
         "weights": "bf16"},
        # a small batch on eight experts: launches count
        {"name": "balance_small", "op": "balance", "t": 256, "e": 8, "top": 2, "dtype": "f32", "masked": False},
        # a long packed batch over the most experts that the router takes, padding and a disabled expert in it
        {"name": "balance_large", "op": "balance", "t": 65536, "e": 256, "top": 8, "dtype": "f32", "masked": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _step(rng, lo, hi, step):
    return max(lo, _log(rng, lo, hi) // step * step)


def _cost(case):
    """Roughly how long a pass takes, in bytes moved (the plain products' flops weighed in)."""
    w = work(case)
    return w["bytes"] + w["flops"] / 50.0


def _limit(op):
    return max(_cost(c) for c in listed() if c["op"] == op)


def draw(rng):
    op = rng.choice(["quantize", "matmul", "matmul", "experts", "norm", "norm", "balance"])
    while True:
        if op == "quantize":
            tiles = rng.random() < 0.4
            case = {"op": op, "rows": _log(rng, 1, 16384), "cols": _log(rng, 1, 14336),
                    "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "tiles": tiles}
        elif op == "matmul":
            case = {"op": op, "m": _log(rng, 1, 8192), "n": _log(rng, 1, 14336), "k": _step(rng, 16, 14336, 16),
                    "out": rng.choice(["bf16", "bf16", "f16", "f32"])}
        elif op == "experts":
            e = rng.choice([1, 2, 5, 8, 16, 33, 64])
            case = {"op": op, "t": _log(rng, 1, 8192), "e": e, "top": rng.randint(1, min(e, 8)),
                    "shared": rng.choice([0, 0, 1, 2]), "h": _step(rng, 128, 4096, 16), "i": _step(rng, 128, 14336, 16),
                    "dtype": rng.choice(["bf16", "bf16", "f16"]), "skew": rng.choice([0.0, 0.0, 2.0])}
        elif op == "norm":
            resid = rng.choice(["bf16", "bf16", "f16", "f32"])
            block = resid if resid != "f32" else rng.choice(["f32", "bf16", "f16"])
            backward = rng.random() < 0.6
            block_out = rng.random() < 0.85
            h = _log(rng, 16, 16384)
            h = h if rng.random() < 0.3 else max(16, h // 8 * 8)
            pre = rng.random() < 0.85 or not block_out
            case = {"op": op, "t": _log(rng, 1, 16384), "h": h, "resid": resid, "block": block,
                    "block_out": block_out, "post": block_out and rng.random() < 0.7,
                    "gate": rng.choice(["none", "channel", "token", "full"]) if block_out else "none", "pre": pre,
                    "codes": pre and not backward and rng.random() < 0.4, "backward": backward,
                    "weights": rng.choice(["f32", block])}
        else:
            e = rng.choice([2, 5, 8, 16, 60, 64, 128, 160, 256])
            case = {"op": op, "t": _log(rng, 1, 65536), "e": e, "top": rng.randint(1, min(e, 8)),
                    "dtype": rng.choice(["f32", "f32", "bf16", "f16"]), "masked": rng.random() < 0.5}
        if op == "experts":
            # the plain form pads every expert to the fullest one: keep its batch within the card
            fullest = case["t"] if case["skew"] else min(case["t"], 2 * case["t"] * case["top"] // case["e"] + 32)
            if (case["e"] * fullest + case["t"]) * (2 * case["i"] + case["h"]) * 4 > 12e9:
                continue
        if _cost(case) <= _limit(op):
            return case


# ------------------------------------------------------------------------------ inputs
def _codes(w):
    """Codes and scales of a matrix [rows, cols] in 128 x 128 tiles (weights at load time)."""
    rows, cols = w.shape
    t = torch.nn.functional.pad(w, (0, blocks(cols) * BLOCK - cols, 0, blocks(rows) * BLOCK - rows))
    t = t.view(blocks(rows), BLOCK, blocks(cols), BLOCK)
    s = _scale(t.abs().amax((1, 3)))
    q = (t / s[:, None, :, None]).to(torch.float8_e4m3fn).view(blocks(rows) * BLOCK, blocks(cols) * BLOCK)
    return q[:rows, :cols].contiguous(), s


def _row_codes(x):
    rows, cols = x.shape
    t = torch.nn.functional.pad(x, (0, blocks(cols) * BLOCK - cols)).view(rows, blocks(cols), BLOCK)
    s = _scale(t.abs().amax(2))
    q = (t / s[:, :, None]).to(torch.float8_e4m3fn).view(rows, blocks(cols) * BLOCK)
    return q[:, :cols].contiguous(), s


def _activations(normal, rows, cols):
    """N(0, 1) with a few channels twenty times as large, as the inputs of a trained block have."""
    x = normal(rows, cols)
    scale = torch.ones(cols, device="cuda")
    scale[:: max(1, cols // 8)] = 20.0
    return x * scale


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    state = dict(case)
    if case["op"] == "quantize":
        x = _activations(normal, case["rows"], case["cols"])
        x[:, : min(BLOCK, case["cols"])][(case["rows"] + 1) // 2 :] = 0  # blocks of zeros, as padding leaves
        state["x"] = x.to(DTYPES[case["dtype"]])
    elif case["op"] == "matmul":
        state["x"], state["x_scale"] = _row_codes(_activations(normal, case["m"], case["k"]))
        state["w"], state["w_scale"] = _codes(normal(case["n"], case["k"]) / math.sqrt(case["k"]))
    elif case["op"] == "experts":
        t, e, h, i, n = case["t"], case["e"], case["h"], case["i"], case["e"] + case["shared"]
        state["x"] = normal(t, h).to(DTYPES[case["dtype"]])
        # routing: softmax over the chosen experts; a skewed one favours the first experts
        logits = normal(t, e) - case["skew"] * torch.log(torch.arange(1, e + 1, device="cuda").float())
        top = logits.topk(case["top"], 1)
        state["ids"] = top.indices.to(torch.int32)
        state["weights"] = top.values.softmax(1)
        # the most rows that an expert gets: the plain form's padded batch
        state["cap"] = int(torch.bincount(top.indices.reshape(-1), minlength=e).max())
        gate_up = [_codes(normal(2 * i, h) / math.sqrt(h)) for _ in range(n)]
        state["gate_up"] = torch.stack([q.view(torch.uint8) for q, _ in gate_up]).view(torch.float8_e4m3fn)
        state["gate_up_scale"] = torch.stack([s for _, s in gate_up])
        del gate_up
        down = [_codes(normal(h, i) / math.sqrt(i)) for _ in range(n)]
        state["down"] = torch.stack([q.view(torch.uint8) for q, _ in down]).view(torch.float8_e4m3fn)
        state["down_scale"] = torch.stack([s for _, s in down])
    elif case["op"] == "norm":
        t, h, rd, bd = case["t"], case["h"], DTYPES[case["resid"]], DTYPES[case["block"]]
        wd = DTYPES[case["weights"]]
        state["r"] = _activations(normal, t, h).to(rd)
        state["y"] = (0.5 * normal(t, h)).to(bd) if case["block_out"] else None
        state["w_post"] = (1 + 0.1 * normal(h)).to(wd) if case["post"] else None
        state["w_pre"] = (1 + 0.1 * normal(h)).to(wd) if case["pre"] else None
        shape = {"none": None, "channel": (h,), "token": (t, 1), "full": (t, h)}[case["gate"]]
        state["gate_value"] = None if shape is None else (0.3 + 0.1 * normal(*shape)).to(wd)
        state["alpha"] = 0.875
        state["eps"] = 1e-6
        if case["backward"]:
            state["d_r"] = (1e-3 * normal(t, h)).to(rd)
            state["d_z"] = (1e-3 * normal(t, h)).to(bd) if case["pre"] else None
    else:
        t, e, dt = case["t"], case["e"], DTYPES[case["dtype"]]
        logits = normal(t, e) + 0.5 * normal(1, e)
        state["valid"] = None
        if case["masked"]:
            logits[:, e // 3] = -math.inf  # an expert that is out of service
            state["valid"] = torch.rand(t, generator=g, device="cuda") < 0.9
            if e - 1 < case["top"]:
                logits[:, e // 3] = 0.0
        state["logits"] = logits.to(dt)
        ids = state["logits"].float().topk(case["top"], 1).indices.to(torch.int32)
        if case["masked"]:
            ids[~state["valid"]] = -1
        state["ids"] = ids
        state["coefficient"] = 0.01
        state["d_loss"] = torch.full((), 1.5, device="cuda")
    return state


# ------------------------------------------------------------------------------ plain forms
def _spread(s, n, dim):
    return s.repeat_interleave(BLOCK, dim).narrow(dim, 0, n)


def _plain_quantize(x, tiles):
    x = x.float()
    rows, cols = x.shape
    high = BLOCK if tiles else 1
    t = torch.nn.functional.pad(x, (0, -cols % BLOCK, 0, -rows % high))
    s = _scale(t.view(t.shape[0] // high, high, blocks(cols), BLOCK).abs().amax((1, 3)))
    wide = _spread(s, cols, 1)
    if tiles:
        wide = _spread(wide, rows, 0)
    return (x / wide).to(torch.float8_e4m3fn), s


def _plain_matmul(s):
    x = s["x"].float() * _spread(s["x_scale"], s["k"], 1)
    w = s["w"].float() * _spread(_spread(s["w_scale"], s["k"], 1), s["n"], 0)
    return (x @ w.t()).to(DTYPES[s["out"]])


def _plain_rounded(x):
    """x as its codes and scales hold it."""
    q, s = _plain_quantize(x.reshape(-1, x.shape[-1]), False)
    return (q.float() * _spread(s, x.shape[-1], 1)).view(x.shape)


def _plain_ffn(x, s, first, last):
    """The experts [first, last) on their padded batches x [experts, rows, h] (codes' values)."""
    h, i = s["h"], s["i"]
    up = s["gate_up"][first:last].float() * _spread(_spread(s["gate_up_scale"][first:last], h, 2), 2 * i, 1)
    y = x @ up.transpose(1, 2)
    del up
    gate, up = y[..., :i], y[..., i:]
    act = _plain_rounded(gate / (1 + torch.exp(-gate)) * up)
    down = s["down"][first:last].float() * _spread(_spread(s["down_scale"][first:last], i, 2), h, 1)
    return act @ down.transpose(1, 2)


def _plain_experts(s):
    t, e, k, cap = s["t"], s["e"], s["top"], s["cap"]
    x = _plain_rounded(s["x"].float())
    ids = s["ids"].reshape(-1).long()
    # place of each (token, slot) among its expert's rows
    chosen = ids[:, None] == torch.arange(e, device="cuda")
    place = (chosen.int().cumsum(0) * chosen).sum(1) - 1
    row = ids * cap + place
    padded = torch.zeros(e * cap, s["h"], device="cuda").index_copy(0, row, x.repeat_interleave(k, 0))
    y = _plain_ffn(padded.view(e, cap, -1), s, 0, e).view(e * cap, -1)[row]
    out = (y.view(t, k, -1) * s["weights"][:, :, None]).sum(1)
    if s["shared"]:
        out = out + _plain_ffn(x.expand(s["shared"], t, s["h"]), s, e, e + s["shared"]).sum(0)
    return out.to(DTYPES[s["dtype"]])


def _plain_norm(s):
    r, h = s["r"].float(), s["h"]
    new = s["alpha"] * r
    gate = None if s["gate_value"] is None else s["gate_value"].float()
    y = yh = u = None
    if s["y"] is not None:
        y = s["y"].float()
        yh = u = y
        if s["w_post"] is not None:
            inv_y = torch.rsqrt((y * y).mean(1, keepdim=True) + s["eps"])
            yh = y * inv_y
            u = yh * s["w_post"].float()
        new = new + (u if gate is None else gate * u)
    out = [new.to(s["r"].dtype)]
    if s["w_pre"] is not None:
        inv = torch.rsqrt((new * new).mean(1, keepdim=True) + s["eps"])
        nh = new * inv
        z = nh * s["w_pre"].float()
        out += list(_plain_quantize(z, False)) if s["codes"] else [z.to(DTYPES[s["block"]])]
    if not s["backward"]:
        return out
    d = s["d_r"].float()
    if s["w_pre"] is not None:
        dz = s["d_z"].float()
        dn = dz * s["w_pre"].float()
        d = d + inv * (dn - nh * (dn * nh).mean(1, keepdim=True))
    out.append((s["alpha"] * d).to(s["r"].dtype))
    if y is not None:
        du = d if gate is None else d * gate
        dy = du
        if s["w_post"] is not None:
            dyh = du * s["w_post"].float()
            dy = inv_y * (dyh - yh * (dyh * yh).mean(1, keepdim=True))
        out.append(dy.to(s["y"].dtype))
        if s["w_post"] is not None:
            out.append((du * yh).sum(0).to(s["w_post"].dtype))
        if gate is not None:
            dg = d * u
            dg = {"channel": lambda: dg.sum(0), "token": lambda: dg.sum(1, keepdim=True), "full": lambda: dg}[s["gate"]]()
            out.append(dg.to(s["gate_value"].dtype))
    if s["w_pre"] is not None:
        out.append((dz * nh).sum(0).to(s["w_pre"].dtype))
    return out


def _plain_balance(s):
    x, e, k = s["logits"].float(), s["e"], s["top"]
    valid = torch.ones(s["t"], device="cuda") if s["valid"] is None else s["valid"].float()
    p = torch.exp(x - x.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True) * valid[:, None]
    ids = s["ids"].reshape(-1).long()
    ones = torch.ones_like(ids).masked_fill(ids < 0, 0)
    counts = torch.zeros(e, dtype=torch.int64, device="cuda").index_add(0, ids.clamp(min=0), ones)
    n = valid.sum().clamp(min=1.0)
    share = counts.float() / (n * k)
    loss = s["coefficient"] * e * (share * p.sum(0) / n).sum()
    d = s["d_loss"] * s["coefficient"] * e / n * p * (share - (p * share).sum(1, keepdim=True))
    return loss, counts.to(torch.int32), d.to(s["logits"].dtype)


# ------------------------------------------------------------------------------ one pass
def run(state):
    s = state
    if not own:
        if s["op"] == "quantize":
            return _plain_quantize(s["x"], s["tiles"])
        if s["op"] == "matmul":
            return _plain_matmul(s)
        if s["op"] == "experts":
            return _plain_experts(s)
        return _plain_norm(s) if s["op"] == "norm" else _plain_balance(s)

    from stageml_b200 import ops

    if s["op"] == "quantize":
        return ops.quantize_e4m3_blocks(s["x"], tiles=s["tiles"])
    if s["op"] == "matmul":
        return ops.block_matmul(s["x"], s["x_scale"], s["w"], s["w_scale"], out_dtype=DTYPES[s["out"]])
    if s["op"] == "experts":
        return ops.moe_forward_blocks(s["x"], s["gate_up"], s["gate_up_scale"], s["down"], s["down_scale"],
                                      topk_ids=s["ids"], topk_weights=s["weights"], n_shared=s["shared"])
    if s["op"] == "norm":
        args = {"post_weight": s["w_post"], "gate": s["gate_value"], "pre_weight": s["w_pre"],
                "residual_scale": s["alpha"], "eps": s["eps"]}
        out = ops.norm_residual(s["y"], s["r"], quantize=s["codes"], normed_dtype=DTYPES[s["block"]], **args)
        if s["backward"]:
            out = out + ops.norm_residual_backward(s["d_r"], s["d_z"], s["y"], s["r"], **args)
        return [o for o in out if o is not None]
    loss, counts, tokens = ops.balance_loss(s["logits"], s["ids"], s["coefficient"], valid=s["valid"])
    grad = ops.balance_loss_backward(s["d_loss"], s["logits"], counts, tokens, s["top"], s["coefficient"],
                                     valid=s["valid"])
    return loss, counts, grad


def work(case):
    c = case
    if c["op"] == "quantize":
        scales = blocks(c["rows"]) * blocks(c["cols"]) if c["tiles"] else c["rows"] * blocks(c["cols"])
        n = c["rows"] * c["cols"]
        return {"bytes": n * (SIZES[c["dtype"]] + 1) + 4 * scales, "flops": 3 * n}
    if c["op"] == "matmul":
        m, n, k = c["m"], c["n"], c["k"]
        scales = 4 * (m * blocks(k) + blocks(n) * blocks(k))
        return {"bytes": m * k + n * k + scales + m * n * SIZES[c["out"]], "flops": 2 * m * n * k}
    if c["op"] == "experts":
        t, h, i, e = c["t"], c["h"], c["i"], c["e"]
        # experts that are expected to see a row under even routing; a skewed one reaches no more
        seen = e * (1 - (1 - c["top"] / e) ** t) + c["shared"]
        weights = seen * 3 * i * h * (1 + 4 / BLOCK / BLOCK)
        pairs = t * (c["top"] + c["shared"])
        return {"bytes": int(weights) + 2 * t * h * 2 + t * c["top"] * 8, "flops": 6 * pairs * h * i}
    if c["op"] == "norm":
        n, r, b, w = c["t"] * c["h"], SIZES[c["resid"]], SIZES[c["block"]], SIZES[c["weights"]]
        has_y, pre = c["block_out"], c["pre"]
        gate = {"none": 0, "channel": c["h"], "token": c["t"], "full": n}[c["gate"]] * w
        small = (c["post"] + pre) * c["h"] * w + gate
        z = n + 4 * c["t"] * blocks(c["h"]) if c["codes"] else n * b
        total = n * (2 * r + has_y * b) + pre * z + small
        if c["backward"]:
            total += n * (3 * r + 2 * has_y * b + pre * b) + 2 * small
        return {"bytes": total, "flops": n * (25 if c["backward"] else 10)}
    n, size = c["t"] * c["e"], SIZES[c["dtype"]]
    return {"bytes": 3 * n * size + 4 * c["t"] * c["top"] + (2 * c["t"] if c["masked"] else 0) + 4 * c["e"],
            "flops": 12 * n}


# ------------------------------------------------------------------------------ 64 bits
def _wide64(q, s, rows, cols, high):
    r = torch.arange(rows, device="cuda") // high
    c = torch.arange(cols, device="cuda") // BLOCK
    return q.double() * s.double()[r][:, c]


def _codes64(x, high):
    """Codes and scales of x [rows, cols] (float64) in blocks of high x 128; the scale is an fp32 number."""
    rows, cols = x.shape
    r = torch.arange(rows, device="cuda") // high
    c = torch.arange(cols, device="cuda") // BLOCK
    a = torch.zeros(blocks(rows) if high == BLOCK else rows, blocks(cols), dtype=torch.float64, device="cuda")
    index = (r[:, None] * a.shape[1] + c).reshape(-1)
    a.view(-1).scatter_reduce_(0, index, x.abs().reshape(-1), "amax")
    s = (a / E4M3_MAX).float()
    s[s == 0] = 1.0
    return (x / s.double()[r][:, c]).float().to(torch.float8_e4m3fn), s


def _ffn64(x, s, j):
    h, i = s["h"], s["i"]
    up = _wide64(s["gate_up"][j], s["gate_up_scale"][j], 2 * i, h, BLOCK)
    y = x @ up.t()
    del up
    act = torch.nn.functional.silu(y[:, :i]) * y[:, i:]
    q, sc = _codes64(act, 1)
    return _wide64(q, sc, act.shape[0], i, 1) @ _wide64(s["down"][j], s["down_scale"][j], h, i, BLOCK).t()


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "quantize":
        q, sc = _codes64(s["x"].double(), BLOCK if s["tiles"] else 1)
        return q.double(), sc.double()
    if s["op"] == "matmul":
        return _wide64(s["x"], s["x_scale"], s["m"], s["k"], 1) @ _wide64(s["w"], s["w_scale"], s["n"], s["k"], BLOCK).t()
    if s["op"] == "experts":
        q, sc = _codes64(s["x"].double(), 1)
        x = _wide64(q, sc, s["t"], s["h"], 1)
        out = torch.zeros_like(x)
        for j in range(s["e"]):
            token, slot = (s["ids"] == j).nonzero(as_tuple=True)
            if token.numel():
                out.index_add_(0, token, _ffn64(x[token], s, j) * s["weights"].double()[token, slot][:, None])
        for j in range(s["e"], s["e"] + s["shared"]):
            out += _ffn64(x, s, j)
        return out
    if s["op"] == "norm":
        names = ["r", "y", "w_post", "gate_value", "w_pre"]
        v = {k: None if s[k] is None else s[k].double().requires_grad_(s["backward"]) for k in names}
        rms = lambda a: a / (a.square().mean(1, keepdim=True) + s["eps"]).sqrt()  # noqa: E731
        new = s["alpha"] * v["r"]
        if v["y"] is not None:
            u = v["y"] if v["w_post"] is None else rms(v["y"]) * v["w_post"]
            new = new + (u if v["gate_value"] is None else u * v["gate_value"])
        out = [new.detach()]
        z = None if v["w_pre"] is None else rms(new) * v["w_pre"]
        if z is not None and s["codes"]:
            q, sc = _codes64(z.detach(), 1)
            out += [q.double(), sc.double()]
        elif z is not None:
            out.append(z.detach())
        if s["backward"]:
            heads, grads = [new], [s["d_r"].double()]
            if z is not None:
                heads.append(z)
                grads.append(s["d_z"].double())
            leaves = [v[k] for k in names if v[k] is not None]
            out += list(torch.autograd.grad(heads, leaves, grads))
        return out
    x = s["logits"].double().requires_grad_(True)
    valid = torch.ones(s["t"], dtype=torch.bool, device="cuda") if s["valid"] is None else s["valid"]
    counts = torch.stack([(s["ids"] == j).sum() for j in range(s["e"])])
    n = max(1, int(valid.sum()))
    mean = (torch.softmax(x, 1) * valid[:, None]).sum(0) / n
    loss = s["coefficient"] * s["e"] * (counts.double() / (n * s["top"]) * mean).sum()
    grad, = torch.autograd.grad(loss, x, s["d_loss"].double())
    return loss.detach(), None, grad
