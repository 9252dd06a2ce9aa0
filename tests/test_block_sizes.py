"""Sizes of the block-scaled operators through the C ABI, without a GPU: workspaces, and which calls are refused."""

import ctypes

import pytest

from stageml_b200 import capi
from stageml_b200._native import load_capi

P = 4096  # a non-null, 16-byte aligned address; never dereferenced


@pytest.mark.parametrize("t,e,k,shared,streams", [
    (1, 8, 2, 0, True), (16, 8, 2, 0, True), (16, 0, 0, 1, True),  # up to 16 tokens
    (17, 8, 2, 0, False), (64, 64, 2, 0, True), (65, 64, 2, 0, False),  # two rows per expert
    (128, 256, 1, 0, True), (129, 256, 1, 0, False), (32, 128, 4, 0, True), (33, 128, 4, 0, False),  # 128 routed rows
    (17, 0, 0, 1, False), (64, 0, 0, 2, False), (128, 0, 0, 1, False),  # shared experts alone have a row per token
    (24, 64, 2, 1, True), (25, 64, 2, 1, False), (64, 64, 2, 1, False), (128, 256, 2, 1, False),
])
def test_layer_streams_its_weights_for_few_rows_only(t, e, k, shared, streams):
    """Streaming passes over an expert's weights once per 8 or 16 of its rows, tensor-core tiles once. The workspace
    shows which one a call takes: only streaming keeps silu(gate) * up in fp32, 4 bytes per row and column."""
    lib = load_capi()
    i = 8192
    a = capi.MoeBlocksArgs(T=t, H=16, I=i, E=e, k=k, n_shared=shared, act_dtype=capi.BF16, ids_dtype=capi.I32,
                           weights_dtype=capi.F32)
    need = lib.stageml_moe_blocks_workspace_bytes(ctypes.byref(a))
    rows = lib.stageml_plan_rows_cap(t * (k + shared), e + shared)
    assert need > rows * i
    assert (need > 5 * rows * i) == streams


@pytest.mark.parametrize("m,n,k", [(0x7fffffff, 16, 16), (1, 0x7fffffff, 16), (64, 0x7fffff80, 16), (64, 64, 0x7ffffff0),
                                   (1, 16, 0x7fffffff - 4095), (64, 16, 0x7fffffff - 4095)])
def test_products_whose_rounded_sizes_pass_32_bits_are_refused(m, n, k):
    lib = load_capi()
    assert lib.stageml_block_matmul(P, P, P, P, m, n, k, capi.BF16, P, None, None) == capi.ERR_INVALID_ARG
    assert "2^31" in lib.stageml_last_error().decode()
    a = capi.MoeBlocksArgs(T=1, H=0x7fffffff - 4095, I=16, E=1, k=1, act_dtype=capi.BF16, ids_dtype=capi.I32,
                           weights_dtype=capi.F32)
    assert lib.stageml_moe_blocks_workspace_bytes(ctypes.byref(a)) == 0
    assert "2^31" in lib.stageml_last_error().decode()
