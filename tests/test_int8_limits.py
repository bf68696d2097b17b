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
