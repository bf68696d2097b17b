"""Refusals of the int8 and grouped products, on the host: every call here
returns before a launch (there may be no GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from freetoken_amd import _lib, ops
from freetoken_amd.layers.moe import MoELayer

P = ctypes.c_void_p(4096)  # a 16-byte aligned pointer that is never read
ODD = ctypes.c_void_p(4104)
INVALID, UNSUPPORTED, WORKSPACE = _lib.FTMOE_ERR_INVALID, _lib.FTMOE_ERR_UNSUPPORTED, _lib.FTMOE_ERR_WORKSPACE


def test_act_quant():
    f = _lib.lib().ftmoe_act_quant_int8
    assert f(None, 0, 64, None, None, None) == 0
    assert f(P, -1, 64, P, P, None) == INVALID
    assert f(P, 4, 24, P, P, None) == UNSUPPORTED  # not a multiple of 16
    assert f(P, 4, 0, P, P, None) == UNSUPPORTED
    assert f(None, 4, 64, P, P, None) == INVALID
    assert f(ODD, 4, 64, P, P, None) == UNSUPPORTED
    assert f(P, 4, 64, ODD, P, None) == UNSUPPORTED


def _matmul(M=4, N=32, K=64, act=-1, dt=_lib.DTYPE_BF16, q=P, qs=P, w=P, ws=P, y=P):
    return _lib.lib().ftmoe_matmul_int8(q, qs, w, ws, M, N, K, act, dt, y, None)


def test_matmul_int8():
    assert _matmul(M=0, q=None, qs=None, w=None, ws=None, y=None) == 0
    assert _matmul(M=-1) == INVALID
    assert _matmul(K=72) == UNSUPPORTED
    assert _matmul(K=131072) == UNSUPPORTED  # sums past 32 bits
    assert _matmul(N=0) == UNSUPPORTED
    assert _matmul(act=3) == UNSUPPORTED
    assert _matmul(act=0, N=33) == INVALID  # no halves
    assert _matmul(dt=2) == UNSUPPORTED
    assert _matmul(M=1 << 20, K=2048) == UNSUPPORTED  # x of 2 GiB
    for name in ("q", "qs", "w", "ws", "y"):
        assert _matmul(**{name: None}) == INVALID, name
    for name in ("q", "w", "y"):
        assert _matmul(**{name: ODD}) == UNSUPPORTED, name


def test_group_routes():
    L = _lib.lib()
    need = L.ftmoe_group_routes_workspace(64, 16)
    assert need > 0
    assert L.ftmoe_group_routes(P, -1, 16, P, P, P, need, None) == INVALID
    assert L.ftmoe_group_routes(P, 64, 1024, P, P, P, 1 << 20, None) == UNSUPPORTED
    assert L.ftmoe_group_routes(P, 64, 0, P, P, P, 1 << 20, None) == UNSUPPORTED
    assert L.ftmoe_group_routes(None, 64, 16, P, P, P, need, None) == INVALID
    assert L.ftmoe_group_routes(P, 64, 16, P, None, P, need, None) == INVALID
    assert L.ftmoe_group_routes(P, 64, 16, P, P, P, need - 1, None) == WORKSPACE
    assert L.ftmoe_group_routes(P, 64, 16, P, P, None, need, None) == WORKSPACE


def _grouped(**over):
    v = dict(format=_lib.FMT_INT8, num_experts=8, N=32, K=64, x=P, x_scale=P, w=P, w_scale=P, x_rows=4, top_k=2,
             offsets=P, order=P, row_weight=None, activation=-1, y=P)
    v.update(over)
    g = _lib.FtmoeGrouped(*[v[name] for name, _ in _lib.FtmoeGrouped._fields_])
    return _lib.lib().ftmoe_grouped_matmul(ctypes.byref(g), None)


def test_grouped_matmul():
    assert _lib.lib().ftmoe_grouped_matmul(None, None) == INVALID
    assert _grouped(x_rows=0, x=None, x_scale=None, w=None, w_scale=None, offsets=None, y=None) == 0
    assert _grouped(format=_lib.FMT_FP8_B128) == UNSUPPORTED
    assert _grouped(order=None) == INVALID  # top_k 2 needs an order
    assert _grouped(x_rows=-1) == INVALID
    assert _grouped(top_k=0) == INVALID
    assert _grouped(x_rows=1 << 20, top_k=1 << 12) == INVALID  # rows past 32 bits
    assert _grouped(num_experts=1024) == UNSUPPORTED
    assert _grouped(num_experts=0) == UNSUPPORTED
    assert _grouped(K=24) == UNSUPPORTED
    assert _grouped(K=24, format=_lib.FMT_BF16, x=None) == INVALID  # (24 is fine for bf16)
    assert _grouped(K=20, format=_lib.FMT_BF16) == UNSUPPORTED
    assert _grouped(activation=0, N=31) == INVALID
    for name in ("x", "x_scale", "w", "w_scale", "offsets", "y"):
        assert _grouped(**{name: None}) == INVALID, name
    for name in ("x", "w", "y"):
        assert _grouped(**{name: ODD}) == UNSUPPORTED, name


def _experts(bank=None, shared=None, M=4, k=2, act=0, ws_less=0, x=P, y=P):
    b = bank or _lib.FtmoeBank(_lib.FMT_INT8, 8, 64, 32, 16, 16, 16, 16)
    bp, sp = ctypes.byref(b), ctypes.byref(shared) if shared else None
    L = _lib.lib()
    need = L.ftmoe_experts_int8_workspace(M, k, bp, sp) if M > 0 else 0
    return L.ftmoe_experts_int8(x, M, k, P, P, bp, sp, act, y, P, need - ws_less, None)


def test_experts_int8():
    bank = _lib.FtmoeBank
    i8 = _lib.FMT_INT8
    assert _experts(M=0, x=None, y=None) == 0
    assert _experts(M=-1) == INVALID
    assert _experts(k=0) == INVALID
    assert _experts(act=-1) == UNSUPPORTED
    assert _experts(ws_less=1) == WORKSPACE
    assert _experts(x=None) == INVALID
    assert _experts(y=ODD) == UNSUPPORTED
    assert _experts(bank(_lib.FMT_BF16, 8, 64, 32, 16, None, 16, None)) == UNSUPPORTED
    assert _experts(bank(i8, 8, 72, 32, 16, 16, 16, 16)) == UNSUPPORTED
    assert _experts(bank(i8, 8, 64, 24, 16, 16, 16, 16)) == UNSUPPORTED
    assert _experts(bank(i8, 1024, 64, 32, 16, 16, 16, 16)) == UNSUPPORTED
    assert _experts(bank(i8, 8, 64, 32, 16, None, 16, 16)) == INVALID
    assert _experts(bank(i8, 8, 64, 32, 16, 16, 16, 16, float("nan"))) == INVALID
    assert _experts(bank(i8, 8, 64, 32, 16, 16, 16, 16, 7.0), act=1) == UNSUPPORTED  # the clamp is a silu form
    assert _experts(shared=bank(i8, 2, 64, 32, 16, 16, 16, 16)) == INVALID
    assert _experts(shared=bank(i8, 1, 128, 32, 16, 16, 16, 16)) == INVALID


def test_other_expert_calls_refuse_an_int8_bank():
    L = _lib.lib()
    b = _lib.FtmoeBank(_lib.FMT_INT8, 8, 256, 256, 16, 16, 16, 16)
    assert L.ftmoe_experts_decode(P, 4, 2, P, P, ctypes.byref(b), None, 0, 0, P, P, 1 << 30, None) == UNSUPPORTED
    assert L.ftmoe_experts_prefill(P, 4, 2, P, P, ctypes.byref(b), None, 0, P, P, 1 << 30, None) == UNSUPPORTED


def test_wrappers_refuse():
    q, s = torch.zeros((4, 64), dtype=torch.int8), torch.ones(4)
    w, ws = torch.zeros((32, 64), dtype=torch.int8), torch.ones(32)
    offsets = torch.zeros(9, dtype=torch.int32)
    for call, what in [
        (lambda: ops.act_quant_int8(torch.zeros(2, 64)), "bfloat16"),
        (lambda: ops.act_quant_int8(torch.zeros(2, 64, dtype=torch.bfloat16)), "device"),
        (lambda: ops.matmul_int8(q.float(), s, w, ws), "int8"),
        (lambda: ops.matmul_int8(q, s, w[:, :32], ws), "int8"),
        (lambda: ops.matmul_int8(q, s.double(), w, ws), "float32"),
        (lambda: ops.matmul_int8(q, s[:3], w, ws), "one scale"),
        (lambda: ops.matmul_int8(q, s, w, ws, activation="relu"), "activation"),
        (lambda: ops.matmul_int8(q, s, w, ws), "device"),
        (lambda: ops.group_routes(torch.zeros(4), 8), "int32"),
        (lambda: ops.grouped_matmul(q.float(), w[None], offsets[:2]), "bfloat16"),
        (lambda: ops.grouped_matmul(q, w, offsets), "experts"),
        (lambda: ops.grouped_matmul(q, w[None], offsets), "offsets"),
        (lambda: ops.grouped_matmul(q, w[None], offsets[:2], top_k=2), "order"),
        (lambda: ops.grouped_matmul(q, w[None], offsets[:2], order=torch.zeros(3, dtype=torch.int32)), "order"),
        (lambda: ops.grouped_matmul(q, w[None], offsets[:2]), "x_scale"),
        (lambda: ops.grouped_matmul(q, w[None], offsets[:2], x_scale=s, w_scale=ws), "w_scale"),
        (lambda: ops.grouped_matmul(q, w[None], offsets[:2], x_scale=s, w_scale=ws[None], row_weight=s[:2]), "row_weight"),
        (lambda: ops.ExpertBank("int8", w[None], w[None]), "scales"),
        (lambda: ops.ExpertBank("int8", w[None], w[None], ws[None], ws[None]), "matrices"),
        (lambda: ops.quantize_bank_int8(ops.ExpertBank("mxfp4", w[None], w[None])), "mxfp4"),
    ]:
        with pytest.raises(ValueError, match=what):
            call()


def test_layer_allocates_an_int8_bank():
    layer = MoELayer(4, 2, 64, 32, weight_format="int8", device="cpu")
    bank = layer.bank()
    assert (bank.num_rows, bank.hidden, bank.inter, bank.fmt) == (4, 64, 32, "int8")
    assert bank.host_cstruct().format == _lib.FMT_INT8
