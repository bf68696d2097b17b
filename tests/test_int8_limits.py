"""Limits of the int8 and grouped products, on the host: every call here returns
before a launch (there may be no GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from freetoken_amd import _lib, ops

P = ctypes.c_void_p(4096)  # a 16-byte aligned pointer that is never read
INVALID, UNSUPPORTED, WORKSPACE = _lib.FTMOE_ERR_INVALID, _lib.FTMOE_ERR_UNSUPPORTED, _lib.FTMOE_ERR_WORKSPACE


def test_row_type_of_the_expert_layer():
    L = _lib.lib()
    bank = _lib.FtmoeBank(_lib.FMT_INT8, 8, 64, 32, 16, 16, 16, 16)
    bp = ctypes.byref(bank)
    need = {dt: L.ftmoe_experts_int8_rows_workspace(4, 2, bp, None, dt) for dt in (_lib.DTYPE_F32, _lib.DTYPE_BF16)}
    assert need[_lib.DTYPE_BF16] == L.ftmoe_experts_int8_workspace(4, 2, bp, None)
    assert need[_lib.DTYPE_F32] > need[_lib.DTYPE_BF16]

    def call(dt, ws, M=4):
        return L.ftmoe_experts_int8_rows(P, M, 2, P, P, bp, None, 0, dt, P, P, ws, None)

    assert call(2, 1 << 20) == UNSUPPORTED
    assert call(_lib.DTYPE_F32, need[_lib.DTYPE_F32] - 1) == WORKSPACE
    assert call(_lib.DTYPE_F32, need[_lib.DTYPE_BF16]) == WORKSPACE
    assert call(_lib.DTYPE_F32, 0, M=0) == 0
    w, s = torch.zeros((4, 32, 32), dtype=torch.int8), torch.ones((4, 32))
    b = ops.ExpertBank("int8", w, w[:, :, :16].contiguous(), s, s)
    with pytest.raises(ValueError, match="rows are"):
        ops.experts_int8(torch.zeros((2, 32), dtype=torch.bfloat16), torch.ones((2, 1)),
                         torch.zeros((2, 1), dtype=torch.int32), b, route_dtype=torch.float16)


def test_most_features():
    L = _lib.lib()
    n = (1 << 30) + 1
    assert L.ftmoe_matmul_int8(P, P, P, P, 1, n, 16, -1, _lib.DTYPE_BF16, P, None) == UNSUPPORTED
    for fmt in (_lib.FMT_INT8, _lib.FMT_BF16):
        g = _lib.FtmoeGrouped(fmt, 1, n, 16, 4096, 4096, 4096, 4096, 1, 1, 4096, None, None, -1, 4096)
        assert L.ftmoe_grouped_matmul(ctypes.byref(g), None) == UNSUPPORTED


def test_workspace_of_routes_past_32_bits():
    """No size that a caller would allocate: the call refuses."""
    L = _lib.lib()
    bank = _lib.FtmoeBank(_lib.FMT_INT8, 8, 64, 32, 16, 16, 16, 16)
    bp = ctypes.byref(bank)
    for M, k in [(1 << 20, 1 << 12), (1 << 30, 1), (1 << 27, 33), ((1 << 31) - 1, 1)]:
        assert L.ftmoe_experts_int8_workspace(M, k, bp, None) == 0
        assert L.ftmoe_experts_int8(P, M, k, P, P, bp, None, 0, P, P, 1 << 60, None) == INVALID


def test_wrappers_refuse_sizes_past_32_bits():
    """They would reach the library cut to 32 bits: 2^32 + 4 rows as 4."""
    big = (1 << 32) + 16

    def many(*shape, dtype=torch.int8):
        return torch.zeros((1,) * len(shape), dtype=dtype).expand(*shape)

    f32, i32, bf16 = torch.float32, torch.int32, torch.bfloat16
    for call in [
        lambda: ops.act_quant_int8(many(big, 16, dtype=bf16)),
        lambda: ops.act_quant_int8(many(1 << 16, (1 << 16) + 1, 16, dtype=bf16)),
        lambda: ops.act_quant_int8(many(2, big, dtype=bf16)),
        lambda: ops.matmul_int8(many(big, 16), many(big, dtype=f32), many(8, 16), many(8, dtype=f32)),
        lambda: ops.matmul_int8(many(4, 16), many(4, dtype=f32), many(big, 16), many(big, dtype=f32)),
        lambda: ops.matmul_int8(many(4, big), many(4, dtype=f32), many(8, big), many(8, dtype=f32)),
        lambda: ops.group_routes(many(big, dtype=i32), 8),
        lambda: ops.group_routes(many(8, dtype=i32), big),
        lambda: ops.grouped_matmul(many(big, 16, dtype=bf16), many(2, 8, 16, dtype=bf16), many(3, dtype=i32)),
        lambda: ops.grouped_matmul(many(4, 16, dtype=bf16), many(2, big, 16, dtype=bf16), many(3, dtype=i32)),
        lambda: ops.grouped_matmul(many(4, 16, dtype=bf16), many(2, 8, 16, dtype=bf16), many(3, dtype=i32),
                                   order=many(4 << 30, dtype=i32), top_k=1 << 30),
        lambda: ops.grouped_matmul(many(4, big, dtype=bf16), many(2, 8, big, dtype=bf16), many(3, dtype=i32)),
        lambda: ops.experts_int8(many(big, 16, dtype=bf16), many(big, 1, dtype=f32), many(big, 1, dtype=i32),
                                 ops.ExpertBank("int8", many(2, 32, 16), many(2, 16, 16), many(2, 32, dtype=f32),
                                                many(2, 16, dtype=f32))),
        lambda: ops.ExpertBank("int8", many(2, 32, big), many(2, big, 16), many(2, 32, dtype=f32), many(2, big, dtype=f32)),
        lambda: ops.ExpertBank("int8", many(2, 1 << 31, 16), many(2, 16, 1 << 30), many(2, 1 << 31, dtype=f32),
                               many(2, 16, dtype=f32)),
    ]:
        with pytest.raises(ValueError, match="32 bits"):
            call()
