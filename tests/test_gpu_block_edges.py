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
