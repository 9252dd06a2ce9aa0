"""Host-side argument checks of the block-scaled products, the block norm and the balance loss through
the C ABI: bad calls are refused before any GPU work (no GPU needed)."""

import ctypes

import pytest

from stageml_b200 import capi
from stageml_b200._native import load_capi

P = 4096  # a non-null, 16-byte aligned address; never dereferenced


@pytest.mark.parametrize("call,text", [
    (lambda L: L.stageml_quantize_e4m3_blocks(P, capi.I32, 1, 4, 128, 0, P, P, None), "F32, BF16 or F16"),
    (lambda L: L.stageml_quantize_e4m3_blocks(P, capi.F32, 1, -4, 128, 0, P, P, None), "negative"),
    (lambda L: L.stageml_quantize_e4m3_blocks(None, capi.F32, 1, 4, 128, 0, P, P, None), "null"),
    (lambda L: L.stageml_block_matmul(P, P, P, P, 4, 4, 24, capi.BF16, P, None, None), "multiple of 16"),
    (lambda L: L.stageml_block_matmul(P, P, P, P, 4, 4, 32, capi.E4M3, P, None, None), "out_dtype"),
    (lambda L: L.stageml_block_matmul(P, None, P, P, 4, 4, 32, capi.BF16, P, None, None), "null"),
    (lambda L: L.stageml_block_matmul(P + 8, P, P, P, 4, 4, 32, capi.BF16, P, None, None), "aligned"),
    (lambda L: L.stageml_block_matmul(P, P, P, P, -1, 4, 32, capi.BF16, P, None, None), "bad sizes"),
    (lambda L: L.stageml_balance_loss(P, capi.F32, P, capi.I32, None, 4, 300, 2, 1.0, P, P, P, None, None, 0, None), "256"),
    (lambda L: L.stageml_balance_loss(P, capi.F32, P, capi.I32, None, 4, 8, 9, 1.0, P, P, P, None, None, 0, None), "1..8"),
    (lambda L: L.stageml_balance_loss(P, capi.F32, P, capi.F32, None, 4, 8, 2, 1.0, P, P, P, None, None, 0, None), "int32"),
    (lambda L: L.stageml_balance_loss(P, capi.F32, None, capi.I32, None, 4, 8, 2, 1.0, P, P, P, None, None, 0, None), "null"),
    (lambda L: L.stageml_balance_loss_backward(None, P, capi.F32, P, P, None, 4, 8, 2, 1.0, P, None), "null"),
])
def test_bad_calls_are_refused(call, text):
    lib = load_capi()
    assert call(lib) == capi.ERR_INVALID_ARG
    assert text in lib.stageml_last_error().decode()


def test_nothing_to_do_is_ok():
    lib = load_capi()
    assert lib.stageml_quantize_e4m3_blocks(None, capi.F32, 1, 0, 128, 0, None, None, None) == capi.OK
    assert lib.stageml_block_matmul(None, None, None, None, 0, 64, 128, capi.BF16, None, None, None) == capi.OK
    assert lib.stageml_balance_loss_backward(None, None, capi.F32, None, None, None, 0, 8, 2, 1.0, None, None) == capi.OK


def test_moe_blocks_args():
    lib = load_capi()
    a = capi.MoeBlocksArgs(T=64, H=256, I=128, E=8, k=2, n_shared=1, act_dtype=capi.BF16, x=P, topk_ids=P,
                           ids_dtype=capi.I32, topk_weights=P, weights_dtype=capi.F32, gate_up=P, gate_up_scale=P, down=P,
                           down_scale=P, out=P)
    need = lib.stageml_moe_blocks_workspace_bytes(ctypes.byref(a))
    assert need > 64 * 3 * (256 + 128)
    assert lib.stageml_moe_forward_blocks(ctypes.byref(a), P, need - 1, None) == capi.ERR_WORKSPACE
    for field, bad, text in (("H", 250, "multiples of 16"), ("k", 9, "min"), ("act_dtype", capi.F32, "act_dtype"),
                             ("E", 2000, "experts"), ("ids_dtype", capi.F32, "ids"), ("down_scale", None, "null"),
                             ("x", P + 2, "aligned"), ("topk_weights", None, "topk_weights")):
        good = getattr(a, field)
        setattr(a, field, bad)
        assert lib.stageml_moe_forward_blocks(ctypes.byref(a), P, 1 << 40, None) == capi.ERR_INVALID_ARG, field
        assert text in lib.stageml_last_error().decode(), field
        setattr(a, field, good)


def test_norm_args():
    lib = load_capi()
    a = capi.NormArgs(T=8, H=64, resid_dtype=capi.BF16, block_dtype=capi.BF16, residual=P, block_out=P, post_weight=P,
                      post_dtype=capi.F32, gate=P, gate_mode=capi.GATE_CHANNEL, gate_dtype=capi.F32, pre_weight=P,
                      pre_dtype=capi.F32, residual_scale=1.0, eps=1e-6, new_residual=P, normed=P)
    need = lib.stageml_norm_residual_workspace_bytes(ctypes.byref(a), 1)
    assert need > 0 and lib.stageml_norm_residual_workspace_bytes(ctypes.byref(a), 0) == 0
    for field, bad, text in (("H", 20000, "16384"), ("H", 0, "bad sizes"), ("block_dtype", capi.F32, "16-bit residual"),
                             ("gate_mode", 7, "gate"), ("gate_mode", capi.GATE_NONE, "disagree"), ("gate", None, "disagree"),
                             ("block_out", None, "need block_out"), ("pre_dtype", capi.I32, "weights"),
                             ("new_residual", None, "null output"), ("normed", None, "without normed"),
                             ("codes", P, "code_scale")):
        good = getattr(a, field)
        setattr(a, field, bad)
        assert lib.stageml_norm_residual(ctypes.byref(a), None, 0, None) == capi.ERR_INVALID_ARG, field
        assert text in lib.stageml_last_error().decode(), field
        setattr(a, field, good)
    assert lib.stageml_norm_residual_backward(ctypes.byref(a), P, need, None) == capi.ERR_INVALID_ARG
    assert "missing" in lib.stageml_last_error().decode()
    a.d_residual = a.d_block_out = a.d_post = a.d_gate = a.d_pre = P
    assert lib.stageml_norm_residual_backward(ctypes.byref(a), P, need - 1, None) == capi.ERR_WORKSPACE
