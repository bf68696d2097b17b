"""The int8 and grouped products against plain computations in 64 bits.

Tolerances count roundings.  A rounding to float32 is off by at most 2^-24 of the
value, to bf16 by 2^-8.  An int8 product is an exact integer; its conversion and
the factors (two scales, their product, a router weight) are five roundings to
float32 at most, so (1 + 2^-24)^5 - 1 < 2^-21 of the value, and 2^-8 more for a
bf16 result.  A bf16 product sums K exact products (16 bits of mantissa) in
float32, off by at most K 2^-24 of the sum of their magnitudes.
SwiGLU and the other activations use the hardware exponential and library
functions: within 2^-16 of |gate * up| (the exponential of an argument x is off by
about |x| 2^-24 relative, |x| <= 88 where it matters: 2^-17).
"""

from __future__ import annotations

import ctypes
from pathlib import Path

import numpy as np
import pytest
import torch

from freetoken_amd import ops
from freetoken_amd.layers.moe import MoELayer
from freetoken_amd.moe.fused import fused_topk

from conftest import COS_TOL, MAX_REL_TOL, cosine, max_rel

pytestmark = pytest.mark.gpu

BF16, F32, FUNC = 2.0**-8, 2.0**-21, 2.0**-16


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def int8_rows(dev, g, *shape):
    return torch.randint(-127, 128, shape, generator=g, device=dev, dtype=torch.int8)


def scales(dev, g, *shape):
    return torch.rand(shape, generator=g, device=dev).add_(0.5).mul_(0.01)


def act_ref(kind, gate):
    if kind == "silu":
        return gate * torch.sigmoid(gate)
    return torch.nn.functional.gelu(gate, approximate="tanh" if kind == "gelu_tanh" else "none")


def within(got, ref, err):
    """|got - ref| <= err everywhere, NaN and infinities included as such."""
    got, ref = got.double(), ref.double()
    fine = (got - ref).abs() <= err
    assert bool(fine.all()), float(((got - ref).abs() - err).max())


# ----------------------------------------------------------------------------- quantisation


def quant_ref(x):
    x = x.double().cpu().numpy()
    a = np.abs(x).max(axis=-1, keepdims=True)
    q = np.rint(np.divide(127.0 * x, a, out=np.zeros_like(x), where=a > 0))
    return q.astype(np.int8), (a[..., 0].astype(np.float32) / np.float32(127)).astype(np.float32)


@pytest.mark.parametrize("rows,K", [(1, 16), (3, 48), (5, 2048), (1, 2064), (130, 1536), (7, 7168), (2, 8192), (3, 8208),
                                    (2, 40000)])
def test_quant_exact(dev, rows, K):
    g = gen(dev, rows + K)
    x = torch.randn((rows, K), generator=g, device=dev).mul_(3.0).to(torch.bfloat16)
    x[0, :] = 0
    x[-1, K // 2] = 100.0
    q, s = ops.act_quant_int8(x)
    q_ref, s_ref = quant_ref(x)
    np.testing.assert_array_equal(q.cpu().numpy(), q_ref)
    np.testing.assert_array_equal(s.cpu().numpy(), s_ref)


@pytest.mark.parametrize("shift", [0, 37, 61, 100, 120, -45, -61, -100, -117])
def test_quant_every_mantissa(dev, shift):
    """Every pair of bf16 mantissas: row i has the largest magnitude 1 + i/128
    (times 2^shift), and every smaller one down to 2^-9 of it, both signs: halves
    among them."""
    top = (1 + torch.arange(128, dtype=torch.float64) / 128)[:, None]
    small = torch.cat([(1 + torch.arange(128, dtype=torch.float64) / 128) * 2.0**-e for e in range(0, 10)])[None, :]
    x = torch.cat([top, torch.where(small <= top, small, 0.0), -torch.where(small <= top, small, 0.0)], dim=1)
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % 16)) * 2.0**shift
    b = x.to(torch.bfloat16)
    assert torch.equal(b.double(), x)
    q, s = ops.act_quant_int8(b.to(dev))
    q_ref, s_ref = quant_ref(x)
    np.testing.assert_array_equal(q.cpu().numpy(), q_ref)
    np.testing.assert_array_equal(s.cpu().numpy(), s_ref)
    assert int((np.abs(127 * x.numpy() / np.abs(x.numpy()).max(1, keepdims=True)) % 1 == 0.5).sum()) > 100


def test_quant_extremes(dev):
    """The largest and smallest bf16 numbers, and rows that hold no number."""
    x = torch.zeros((8, 64), dtype=torch.bfloat16)
    big, tiny = torch.finfo(torch.bfloat16).max, 2.0**-133
    x[0, :3] = torch.tensor([big, -big / 2, 1.0], dtype=torch.bfloat16)
    x[1, :3] = torch.tensor([tiny, -tiny, 0.0], dtype=torch.bfloat16)
    x[2, :3] = torch.tensor([3 * tiny, -tiny, 2 * tiny], dtype=torch.bfloat16)
    x[3, 5], x[4, 6], x[5, 7] = float("inf"), float("-inf"), float("nan")
    x[3:6, 9] = 1.0
    x[6, 1] = -0.0
    x[7, 60] = -1.0
    q, s = ops.act_quant_int8(x.to(dev))
    q, s = q.cpu(), s.cpu()
    keep = [0, 1, 2, 6, 7]
    q_ref, s_ref = quant_ref(x[keep])
    np.testing.assert_array_equal(q[keep].numpy(), q_ref)
    np.testing.assert_array_equal(s[keep].numpy(), s_ref)
    assert torch.isnan(s[3:6]).all() and not q[3:6].any()


def test_quant_leading_dimensions_and_empty(dev):
    x = torch.randn((3, 5, 32), generator=gen(dev, 1), device=dev).to(torch.bfloat16)
    q, s = ops.act_quant_int8(x)
    assert q.shape == x.shape and s.shape == (3, 5)
    q2, s2 = ops.act_quant_int8(x.view(15, 32))
    assert torch.equal(q.view(15, 32), q2) and torch.equal(s.view(15), s2)
    q, s = ops.act_quant_int8(x[:, :0])
    assert q.shape == (3, 0, 32) and s.shape == (3, 0)


# ----------------------------------------------------------------------------- the dense product

DENSE = [(1, 16, 16), (1, 4096, 7168), (2, 1, 32), (3, 33, 48), (15, 257, 144), (16, 640, 128), (17, 130, 2064),
         (31, 1000, 112), (48, 768, 2048), (65, 512, 4112), (129, 96, 256), (255, 777, 80), (257, 5120, 1536),
         (300, 300, 304), (513, 264, 1280), (1025, 2056, 640), (2111, 512, 128)]


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("M,N,K", DENSE)
def test_matmul_int8(dev, M, N, K, out_dtype):
    g = gen(dev, M * 7 + N + K)
    q, w = int8_rows(dev, g, M, K), int8_rows(dev, g, N, K)
    s, ws = scales(dev, g, M), scales(dev, g, N)
    y = ops.matmul_int8(q, s, w, ws, out_dtype=out_dtype)
    assert y.dtype == out_dtype and y.shape == (M, N)
    ref = (q.double() @ w.double().T) * s.double()[:, None] * ws.double()
    within(y, ref, ref.abs() * (F32 + (BF16 if out_dtype == torch.bfloat16 else 0)))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("M,N,K", [(1, 2, 16), (3, 66, 144), (20, 1024, 512), (70, 514, 1040), (300, 1536, 768)])
def test_matmul_int8_activation(dev, M, N, K, act):
    g = gen(dev, M + N + K)
    q, w = int8_rows(dev, g, M, K), int8_rows(dev, g, N, K)
    s, ws = scales(dev, g, M), scales(dev, g, N) * (3.0 / K**0.5)
    y = ops.matmul_int8(q, s, w, ws, activation=act, out_dtype=torch.float32)
    assert y.shape == (M, N // 2)
    h = (q.double() @ w.double().T) * s.double()[:, None] * ws.double()
    gate, up = h.chunk(2, dim=1)
    # an input off by F32 moves the activation by at most 1.2 F32 |gate|
    within(y, act_ref(act, gate) * up, (gate * up).abs() * (FUNC + 4 * F32))


def test_matmul_int8_exact_sums(dev):
    """The largest sums: every product of the extreme codes, at the largest K."""
    K = 131056
    q = torch.full((5, K), -128, dtype=torch.int8, device=dev)
    w = torch.full((40, K), 127, dtype=torch.int8, device=dev)
    q[1], w[1], w[2, ::2] = 127, -128, -127
    one = torch.ones(40, device=dev)
    y = ops.matmul_int8(q, one[:5], w, one, out_dtype=torch.float32)
    ref = (q.cpu().long() @ w.cpu().long().T).to(torch.float32)  # rounded to float32 once
    assert torch.equal(y.cpu(), ref)


def test_matmul_int8_out_and_nan_rows(dev):
    g = gen(dev, 9)
    x = torch.randn((6, 256), generator=g, device=dev).to(torch.bfloat16)
    x[2, 3] = float("nan")
    w, ws = int8_rows(dev, g, 100, 256), scales(dev, g, 100)
    q, s = ops.act_quant_int8(x)
    out = torch.empty((6, 100), dtype=torch.float32, device=dev)
    y = ops.matmul_int8(q, s, w, ws, out=out)
    assert y is out
    rows = torch.isnan(y).all(1).cpu()
    assert rows.tolist() == [False, False, True, False, False, False] and not torch.isnan(y[rows.logical_not()]).any()
    assert ops.matmul_int8(q[:0], s[:0], w, ws).shape == (0, 100)


def test_matmul_int8_result_past_32_bits(dev):
    """A result of more than 2^31 values, and a weight row past 2^31 bytes."""
    M, N, K = 262150, 8200, 16
    g = gen(dev, 10)
    q, w = int8_rows(dev, g, M, K), int8_rows(dev, g, N, K)
    s, ws = scales(dev, g, M), scales(dev, g, N)
    y = ops.matmul_int8(q, s, w, ws)
    at = torch.tensor([0, 1, 131071, 261900, M - 2, M - 1], device=dev)
    ref = (q[at].double() @ w.double().T) * s[at].double()[:, None] * ws.double()
    within(y[at], ref, ref.abs() * (BF16 + F32))
    del y
    M, N, K = 3, 17000, 131056
    q, w = int8_rows(dev, g, M, K), int8_rows(dev, g, N, K)
    s, ws = scales(dev, g, M), scales(dev, g, N)
    y = ops.matmul_int8(q, s, w, ws, out_dtype=torch.float32)
    for n in (0, 16390, N - 1):
        ref = (q.double() @ w[n].double()) * s.double() * ws[n].double()
        within(y[:, n], ref, ref.abs() * F32)


# ----------------------------------------------------------------------------- grouping


@pytest.mark.parametrize("numel", [0, 1, 63, 64, 65, 1000, 4096, 4097, 70000])
@pytest.mark.parametrize("E", [1, 16, 1023])
def test_group_routes(dev, numel, E):
    rng = np.random.default_rng(numel + E)
    ids = rng.integers(-2, E + 3, size=numel).astype(np.int32)
    order, offsets = ops.group_routes(torch.from_numpy(ids).to(dev), E)
    got, off = order.cpu().numpy(), offsets.cpu().numpy()
    assert off.shape == (E + 1,) and got.shape == (numel,)
    want = np.concatenate([np.nonzero(ids == e)[0] for e in range(E)]) if numel else np.zeros(0)
    np.testing.assert_array_equal(got[: off[-1]], want)
    np.testing.assert_array_equal(off, np.concatenate([[0], np.cumsum([(ids == e).sum() for e in range(E)])]))


# ----------------------------------------------------------------------------- the grouped product


def grouped_ref(x, w, counts, rows_of, act, weight, x_scale=None, w_scale=None):
    """(result, error bound) in 64 bits; rows_of: (row of y, row of x) of every position."""
    n = w.shape[1] // (2 if act else 1)
    y_rows, x_rows = rows_of
    ref = torch.full((len(y_rows), n), float("nan"), dtype=torch.float64, device=x.device)
    err = torch.zeros_like(ref)
    at = 0
    for e, c in enumerate(counts):
        pos = slice(at, at + c)
        at += c
        xe, we = x[x_rows[pos]].double(), w[e].double()
        h = xe @ we.T
        if x_scale is not None:  # (the sums of int8 codes are exact: scaled afterwards)
            h = h * x_scale[x_rows[pos]].double()[:, None] * w_scale[e].double()
        off = h.abs() * F32 if x_scale is not None else (xe.abs() @ we.abs().T) * (x.shape[1] * 2.0**-24)
        if act:
            g, u = h.chunk(2, dim=1)
            og, ou = off.chunk(2, dim=1)
            h = act_ref(act, g) * u
            off = 1.2 * og * u.abs() + ou * act_ref(act, g).abs() + 1.2 * og * ou + (g * u).abs() * FUNC
        if weight is not None:
            f = weight[y_rows[pos]].double()[:, None]
            h, off = h * f, off * f.abs() + (h * f).abs() * 2.0**-24
        ref[y_rows[pos]] = h
        err[y_rows[pos]] = off + (h.abs() + off) * BF16
    return ref, err


# rows of every expert: empty ones first, last and between; below, at and above the tiles' sizes
COUNTS = [
    [1],
    [0, 3, 0, 1, 16, 0],
    [0, 0, 0],
    [17, 15, 33, 64, 0, 65],
    [130, 0, 1, 256, 257, 5],
    [700, 3, 0, 0, 90],
    [2] * 200 + [0] * 100 + [1] * 30,
]


@pytest.mark.parametrize("act,weigh", [(None, False), (None, True), ("silu", False)])
@pytest.mark.parametrize("N,K", [(96, 128), (258, 144), (512, 1040), (24, 16)])
@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("counts", COUNTS, ids=range(len(COUNTS)))
def test_grouped_laid_out(dev, counts, int8, N, K, act, weigh):
    E, R = len(counts), sum(counts)
    g = gen(dev, E + R + N)
    pad = 3  # rows behind the last group, left as they were
    rows = R + pad
    if int8:
        x, w = int8_rows(dev, g, rows, K), int8_rows(dev, g, E, N, K)
        xs, ws = scales(dev, g, rows), scales(dev, g, E, N)
    else:
        x = torch.randn((rows, K), generator=g, device=dev).to(torch.bfloat16)
        w = torch.randn((E, N, K), generator=g, device=dev).to(torch.bfloat16)
        x[R:] = float("nan")
        xs = ws = None
    weight = torch.rand((rows,), generator=g, device=dev) if weigh else None
    offsets = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device=dev)
    out = torch.full((rows, N // 2 if act else N), 7.0, dtype=torch.bfloat16, device=dev)
    y = ops.grouped_matmul(x, w, offsets, x_scale=xs, w_scale=ws, row_weight=weight, activation=act, out=out)
    assert y is out
    at = torch.arange(R, device=dev)
    ref, err = grouped_ref(x, w, counts, (at, at), act, weight, xs, ws)
    within(y[:R], ref, err)
    assert bool((y[R:] == 7.0).all())


@pytest.mark.parametrize("act,weigh", [(None, True), ("gelu_tanh", False)])
@pytest.mark.parametrize("M,k,E", [(1, 1, 4), (1, 8, 128), (5, 3, 7), (64, 8, 64), (301, 4, 16), (600, 7, 300)])
@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_grouped_routed(dev, M, k, E, int8, act, weigh):
    """Tokens with their top-k ids, some of them of no expert: those rows are left as they were."""
    g, rng = gen(dev, M + k + E), np.random.default_rng(M * k)
    N, K = 136, 272
    ids = rng.integers(0, E, size=(M, k)).astype(np.int32)
    ids[rng.random((M, k)) < 0.1] = -1
    ids[rng.random((M, k)) < 0.05] = E
    if int8:
        x, w = int8_rows(dev, g, M, K), int8_rows(dev, g, E, N, K)
        xs, ws = scales(dev, g, M), scales(dev, g, E, N)
    else:
        x = torch.randn((M, K), generator=g, device=dev).to(torch.bfloat16)
        w = torch.randn((E, N, K), generator=g, device=dev).mul_(0.1).to(torch.bfloat16)
        xs = ws = None
    weight = torch.rand((M * k,), generator=g, device=dev) if weigh else None
    order, offsets = ops.group_routes(torch.from_numpy(ids).to(dev), E)
    out = torch.full((M * k, N // 2 if act else N), 7.0, dtype=torch.bfloat16, device=dev)
    ops.grouped_matmul(x, w, offsets, order=order, top_k=k, x_scale=xs, w_scale=ws, row_weight=weight, activation=act,
                       out=out)
    counts = [int((ids == e).sum()) for e in range(E)]
    listed = order[: sum(counts)].long()
    full = torch.zeros((M * k,), dtype=torch.bool, device=dev)
    full[listed] = True
    y = torch.where(full[:, None], out.double(), float("nan"))
    assert bool((out[~full] == 7.0).all())
    flat = torch.from_numpy(ids.reshape(-1)).to(dev)
    for e in range(E):
        at = torch.nonzero(flat == e)[:, 0]
        if at.numel() == 0:
            continue
        sub = None if weight is None else weight[at]
        place = torch.arange(at.numel(), device=dev)
        ref, err = grouped_ref(x, w[e : e + 1], [at.numel()], (place, at // k), act, sub, xs,
                               None if ws is None else ws[e : e + 1])
        within(y[at], ref, err)


def test_grouped_offsets_are_cut(dev):
    """Offsets outside the rows, or descending, reach no memory outside the tensors: what they name inside is computed."""
    g = gen(dev, 3)
    x = torch.randn((40, 64), generator=g, device=dev).to(torch.bfloat16)
    w = torch.randn((3, 32, 64), generator=g, device=dev).to(torch.bfloat16)
    out = torch.full((40, 32), 7.0, dtype=torch.bfloat16, device=dev)
    offsets = torch.tensor([-5, 10, 4, 1 << 30], dtype=torch.int32, device=dev)  # rows 0-9, none, 4-39
    ops.grouped_matmul(x, w, offsets, out=out)
    ref, err = grouped_ref(x[10:], w[2:], [30], (torch.arange(30, device=dev),) * 2, None, None)
    within(out[10:], ref, err)
    order = torch.arange(40, dtype=torch.int32, device=dev)
    order[7], order[8] = 1 << 30, -3  # not rows: skipped
    out.fill_(7.0)
    ops.grouped_matmul(x, w, torch.tensor([0, 0, 40, 40], dtype=torch.int32, device=dev), order=order, out=out)
    ref, err = grouped_ref(x, w[1:2], [40], (torch.arange(40, device=dev),) * 2, None, None)
    keep = [i for i in range(40) if i not in (7, 8)]
    within(out[keep], ref[keep], err[keep])
    assert bool((out[7:9] == 7.0).all())


@pytest.mark.parametrize("R", [3, 40, 700])
def test_grouped_views(dev, R):
    """Scales, weights, order and offsets that begin 4 bytes into their memory, matrices that begin 16 into theirs."""
    g = gen(dev, R)
    E, N, K, off = 3, 72, 208, 1
    x, w = int8_rows(dev, g, R + off, K)[off:], int8_rows(dev, g, E + off, N, K)[off:]
    xs, ws = scales(dev, g, R + off)[off:], scales(dev, g, E * N + off)[off:].view(E, N)
    weight = torch.rand((R + off,), generator=g, device=dev)[off:]
    order = torch.randperm(R, generator=g, device=dev).to(torch.int32)
    order = torch.cat([order[:1], order])[off:]
    counts = [R // 3, 0, R - R // 3]
    offsets = torch.tensor([0, 0] + list(np.cumsum(counts)), dtype=torch.int32, device=dev)[off:]
    y = ops.grouped_matmul(x, w, offsets, order=order, x_scale=xs, w_scale=ws, row_weight=weight)
    at = order.long()
    ref, err = grouped_ref(x, w, counts, (at, at), None, weight, xs, ws)
    within(y, ref, err)


def test_grouped_nan_stays_in_its_row(dev):
    """A token's infinity or NaN reaches its own rows only; zeros beside NaN weights of other experts do not."""
    g = gen(dev, 4)
    x = torch.randn((30, 80), generator=g, device=dev).to(torch.bfloat16)
    w = torch.randn((2, 48, 80), generator=g, device=dev).to(torch.bfloat16)
    x[3, 7], x[20, 0] = float("nan"), float("inf")
    w[1, 5] = float("nan")
    offsets = torch.tensor([0, 17, 30], dtype=torch.int32, device=dev)
    y = ops.grouped_matmul(x, w, offsets)
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[3], want[20], want[17:, 5] = True, True, True
    assert torch.equal(bad, want)


def test_grouped_weights_past_32_bits(dev):
    """The last expert's matrix lies 4 GiB behind the first."""
    g = gen(dev, 5)
    E, N, K = 66, 8192, 8192
    w = torch.zeros((E, N, K), dtype=torch.int8, device=dev)
    w[-1] = int8_rows(dev, g, N, K)
    for R in (4, 200):
        x, xs, ws = int8_rows(dev, g, R, K), scales(dev, g, R), scales(dev, g, E, N)
        offsets = torch.zeros(E + 1, dtype=torch.int32, device=dev)
        offsets[-1] = R
        y = ops.grouped_matmul(x, w, offsets, x_scale=xs, w_scale=ws)
        at = torch.arange(R, device=dev)
        ref, err = grouped_ref(x, w[-1:], [R], (at, at), None, None, xs, ws[-1:])
        within(y, ref, err)


# ----------------------------------------------------------------------------- every form

FORMS_HELPER = Path(__file__).resolve().parent / "gpu_helpers" / "libmatmulforms.so"
FORMS = ["split", "whole", "wide", "128x64", "128x64 once", "256x128", "256x128 once", "256x256"]


class FormArgs(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("x", "xs", "w", "ws", "offsets", "order", "ids", "row_weight",
                                                "extra_w", "extra_ws", "y")]
                + [(n, ctypes.c_int) for n in ("int8", "E", "N", "K", "rows", "x_rows", "top_k", "act", "extra",
                                               "extra_x", "quantise", "out_f32")]
                + [("limit", ctypes.c_float), ("extra_limit", ctypes.c_float)])


def run_form(form, **args):
    if not FORMS_HELPER.exists():
        from tests.gpu_helpers import build_helpers  # built by __graft_entry__.build(); rebuilt if absent

        build_helpers.build()
    fn = ctypes.CDLL(str(FORMS_HELPER)).ftmoe_test_matmul_form
    fn.argtypes = [ctypes.POINTER(FormArgs), ctypes.c_int, ctypes.c_void_p]
    ptr = {k: v.data_ptr() if isinstance(v, torch.Tensor) else v for k, v in args.items()}
    assert fn(ctypes.byref(FormArgs(**ptr)), FORMS.index(form), torch.cuda.current_stream().cuda_stream) == 0


@pytest.mark.parametrize("gate", [False, True], ids=["plain", "gated"])
@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("form", FORMS)
def test_forms(dev, form, int8, gate):
    """Every form at the same ragged problem, whatever the rule would take: empty groups, blocks of one row to several,
    rows in a routed order with several routes per token, one more group with a matrix and rows of its own behind."""
    counts, k = [1, 0, 33, 5, 0, 270, 64, 129, 16], 2
    E, R, extra = len(counts), sum(counts), 37
    x_rows = R // k
    for N, K in [(530, 1168), (40, 16), (1030, 384)]:
        g = gen(dev, N)
        if int8:
            x, w = int8_rows(dev, g, x_rows + extra, K), int8_rows(dev, g, E + 1, N, K)
            xs, ws = scales(dev, g, x_rows + extra), scales(dev, g, E + 1, N)
        else:
            x = torch.randn((x_rows + extra, K), generator=g, device=dev).to(torch.bfloat16)
            w = torch.randn((E + 1, N, K), generator=g, device=dev).to(torch.bfloat16)
            xs = ws = None
        more = w[E].clone(), None if ws is None else ws[E].clone()
        weight = None if gate else torch.rand((R,), generator=g, device=dev)
        order = torch.randperm(R, generator=g, device=dev).to(torch.int32)
        offsets = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device=dev)
        n_out = N // 2 if gate else N
        guard = torch.full((R + extra + 1, n_out), 7.0, dtype=torch.bfloat16, device=dev)
        run_form(form, x=x, xs=xs, w=w, ws=ws, offsets=offsets, order=order, ids=None, row_weight=weight, extra_w=more[0],
                 extra_ws=more[1], y=guard, int8=int(int8), E=E, N=N, K=K, rows=R, x_rows=x_rows + extra, top_k=k,
                 act=0 if gate else -1, extra=extra, extra_x=x_rows, quantise=0, out_f32=0, limit=0.0, extra_limit=0.0)
        at = order.long()
        act = "silu" if gate else None
        ref, err = grouped_ref(x, w, counts, (at, at // k), act, weight, xs, ws)
        within(guard[:R], ref, err)
        at = torch.arange(extra, device=dev)
        ref, err = grouped_ref(x[x_rows:], w[E:], [extra], (at, at), act, None, None if xs is None else xs[x_rows:],
                               None if ws is None else ws[E:])
        within(guard[R : R + extra], ref, err)
        assert bool((guard[-1] == 7.0).all())


@pytest.mark.parametrize("form", FORMS)
def test_forms_dense_f32(dev, form):
    """One group without offsets and order, float32 results."""
    M, N, K = 301, 517, 1808
    g = gen(dev, 11)
    x, w, xs, ws = int8_rows(dev, g, M, K), int8_rows(dev, g, N, K), scales(dev, g, M), scales(dev, g, N)
    y = torch.full((M + 1, N), 7.0, device=dev)
    run_form(form, x=x, xs=xs, w=w, ws=ws, offsets=None, order=None, ids=None, row_weight=None, extra_w=None,
             extra_ws=None, y=y, int8=1, E=1, N=N, K=K, rows=M, x_rows=M, top_k=1, act=-1, extra=0, extra_x=0, quantise=0, out_f32=1,
             limit=0.0, extra_limit=0.0)
    ref = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    within(y[:M], ref, ref.abs() * F32)
    assert bool((y[M] == 7.0).all())


@pytest.mark.parametrize("K", [16, 768, 2032, 2048])
@pytest.mark.parametrize("form", ["split", "whole"])
def test_forms_that_quantise(dev, form, K):
    """bf16 rows quantised inside the product: the codes and scales of act_quant_int8, so the very results."""
    counts = [3, 0, 1, 20]
    E, R, N = len(counts), sum(counts), 200
    g = gen(dev, K)
    x = torch.randn((R, K), generator=g, device=dev).to(torch.bfloat16)
    x[1] = 0
    w, ws = int8_rows(dev, g, E, N, K), scales(dev, g, E, N)
    offsets = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device=dev)
    q, s = ops.act_quant_int8(x)
    y = torch.full((2, R + 1, N), 7.0, dtype=torch.bfloat16, device=dev)
    y[:, :R] = float("nan")
    for i, (rows, xs) in enumerate([(x, None), (q, s)]):
        run_form(form, x=rows, xs=xs, w=w, ws=ws, offsets=offsets, order=None, ids=None, row_weight=None, extra_w=None,
                 extra_ws=None, y=y[i], int8=1, E=E, N=N, K=K, rows=R, x_rows=R, top_k=1, act=-1, extra=0, extra_x=0,
                 quantise=1 - i, out_f32=0, limit=0.0, extra_limit=0.0)
    assert torch.equal(y[0], y[1]) and bool((y[:, R] == 7.0).all())


@pytest.mark.parametrize("rows,k,E,extra", [(1, 1, 1, 0), (8, 8, 128, 1), (32, 8, 3, 4), (64, 2, 16, 33), (64, 1, 1, 0),
                                            (20, 4, 1023, 0), (6, 3, 5, 2)])
@pytest.mark.parametrize("gate", [False, True], ids=["plain", "gated"])
@pytest.mark.parametrize("form", ["split", "whole"])
def test_forms_by_id(dev, form, gate, rows, k, E, extra):
    """Groups found from the rows' ids (some of no group): the very results of listed groups on quantised rows."""
    N, K, tokens = 74, 592, rows // k
    g, rng = gen(dev, rows + E), np.random.default_rng(rows + E)
    x = torch.randn((tokens + extra, K), generator=g, device=dev).to(torch.bfloat16)
    w, ws = int8_rows(dev, g, E + 1, N, K), scales(dev, g, E + 1, N)
    flat = rng.integers(0, E, size=rows).astype(np.int32)
    flat[rng.random(rows) < 0.15] = -1
    flat[rng.random(rows) < 0.1] = E
    ids = torch.from_numpy(flat).to(dev)
    weight = None if gate else torch.rand((rows,), generator=g, device=dev)
    order, offsets = ops.group_routes(ids, E)
    q, s = ops.act_quant_int8(x)
    more = w[E].clone(), ws[E].clone()
    y = torch.full((2, rows + extra + 1, N // 2 if gate else N), 7.0, dtype=torch.bfloat16, device=dev)
    for i, rows_of in enumerate([dict(x=x, xs=None, offsets=None, order=None, ids=ids),
                                 dict(x=q, xs=s, offsets=offsets, order=order, ids=None)]):
        run_form(form, w=w, ws=ws, row_weight=weight, extra_w=more[0], extra_ws=more[1], y=y[i], int8=1, E=E, N=N, K=K,
                 rows=rows, x_rows=tokens + extra, top_k=k, act=0 if gate else -1, extra=extra, extra_x=tokens,
                 quantise=1 - i, out_f32=0, limit=0.0, extra_limit=0.0, **rows_of)
    skipped = torch.from_numpy((flat < 0) | (flat >= E)).to(dev)
    assert torch.equal(y[0], y[1]) and bool((y[0, :rows][skipped] == 7.0).all()) and bool((y[0, -1] == 7.0).all())


# ----------------------------------------------------------------------------- the layer


def make_bank(dev, g, E, H, I):
    def one(n, k):
        return ops.act_quant_int8(torch.randn((E, n, k), generator=g, device=dev).mul_(k**-0.5).to(torch.bfloat16))

    (gu, gs), (dn, ds) = one(2 * I, H), one(H, I)
    return ops.ExpertBank("int8", gu, dn, gs, ds)


def routing(dev, g, M, k, E):
    top = torch.topk(torch.randn((M, E), generator=g, device=dev), k, dim=1)
    return torch.softmax(top.values, 1).contiguous(), top.indices.to(torch.int32).contiguous()


def values(x):
    """What the int8 codes of x's rows stand for."""
    x = x.double()
    a = x.abs().amax(-1, keepdim=True)
    return torch.where(a > 0, (127 * x / torch.where(a > 0, a, 1.0)).round() * (a / 127), 0.0)


def layer_ref(x, tw, ids, bank, shared, act):
    def mlp(rows, b, e):
        limit = b.swiglu_limit
        h = rows @ (b.gate_up[e].double() * b.gate_up_scale[e].double()[:, None]).T
        gate, up = h.chunk(2, dim=1)
        if limit > 0:
            gate, up = gate.clamp_max(limit), up.clamp(-limit, limit)
        a = (act_ref(act, gate) * up).to(torch.bfloat16)
        return values(a) @ (b.down[e].double() * b.down_scale[e].double()[:, None]).T

    xv = values(x)
    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for e in range(bank.num_rows):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if t.numel():
            y.index_add_(0, t, mlp(xv[t], bank, e) * tw[t, j].double()[:, None])
    return y if shared is None else y + mlp(xv, shared, 0)


LAYER = [  # M, k, E, H, I, shared inter, activation, limit
    (1, 2, 16, 256, 128, 0, "silu", 0.0),
    (4, 2, 16, 1024, 512, 0, "silu", 0.0),
    (7, 8, 128, 336, 112, 48, "silu", 0.0),
    (64, 8, 64, 512, 256, 256, "gelu", 0.0),
    (130, 4, 8, 272, 400, 16, "silu", 0.75),
    (40, 2, 24, 272, 144, 144, "silu", 0.75),
    (700, 6, 32, 640, 384, 384, "gelu_tanh", 0.0),
    (1500, 8, 16, 512, 256, 0, "silu", 0.0),
]


@pytest.mark.parametrize("case", LAYER, ids=lambda c: "x".join(map(str, c[:6])))
def test_experts_int8(dev, case):
    M, k, E, H, I, Is, act, limit = case
    g = gen(dev, M + E)
    x = torch.randn((M, H), generator=g, device=dev).to(torch.bfloat16)
    bank = make_bank(dev, g, E, H, I)
    shared = make_bank(dev, g, 1, H, Is) if Is else None
    bank.swiglu_limit = limit
    if shared:
        shared.swiglu_limit = 2 * limit
    tw, ids = routing(dev, g, M, k, E)
    if M > 2:  # padded places: no expert
        ids[M // 2 :: 3] = -1
        ids[0, 0] = E
    y = ops.experts_int8(x, tw, ids, bank, shared=shared, activation=act)
    ref = layer_ref(x, tw, ids, bank, shared, act)
    got, want = y.double().cpu().numpy(), ref.cpu().numpy()
    assert max_rel(got, want) <= MAX_REL_TOL and cosine(got, want) >= COS_TOL, (max_rel(got, want), cosine(got, want))
    if shared is None and M > 2:
        assert not y[M // 2].any()  # a token without experts
    # the same result from the operators one by one, exactly, the routes summed in order
    q, s = ops.act_quant_int8(x)
    order, offsets = ops.group_routes(ids, E)

    if limit:  # the clamp is the layer's own: the products alone have none
        return
    h = torch.zeros((M * k, I), dtype=torch.bfloat16, device=dev)
    ops.grouped_matmul(q, bank.gate_up, offsets, order=order, top_k=k, x_scale=s, w_scale=bank.gate_up_scale,
                       activation=act, out=h)
    hq, hs = ops.act_quant_int8(h)
    o = torch.zeros((M * k, H), dtype=torch.bfloat16, device=dev)
    ops.grouped_matmul(hq, bank.down, offsets, order=order, x_scale=hs, w_scale=bank.down_scale,
                       row_weight=tw.view(-1), out=o)
    total = torch.zeros((M, H), device=dev)
    for j in range(k):
        total = total + o.view(M, k, H)[:, j].float()
    if shared is not None:
        sq, ss = ops.act_quant_int8(ops.matmul_int8(q, s, shared.gate_up[0], shared.gate_up_scale[0], activation=act))
        total = total + ops.matmul_int8(sq, ss, shared.down[0], shared.down_scale[0]).float()
    assert torch.equal(y, total.to(torch.bfloat16))


def test_layer_module(dev):
    """MoELayer with int8 weights: forward from logits and routed_forward, decode and prefill sizes, from a bf16 bank."""
    g = gen(dev, 21)
    E, H, I, k = 16, 512, 256, 4
    bf = ops.ExpertBank("bf16", torch.randn((E, 2 * I, H), generator=g, device=dev).mul_(H**-0.5).to(torch.bfloat16),
                        torch.randn((E, H, I), generator=g, device=dev).mul_(I**-0.5).to(torch.bfloat16))
    bank = ops.quantize_bank_int8(bf)
    assert (bank.gate_up.float() * bank.gate_up_scale[..., None] - bf.gate_up.float()).abs().max() \
        <= bank.gate_up_scale.max() * 0.5001
    layer = MoELayer(E, k, H, I, weight_format="int8", device=dev)
    for name in ("gate_up", "down"):
        getattr(layer, name + "_proj").copy_(getattr(bank, name))
        getattr(layer, name + "_scale").copy_(getattr(bank, name + "_scale"))
    for M in (1, 5, 40, 1100):
        x = torch.randn((M, H), generator=g, device=dev).to(torch.bfloat16)
        logits = torch.randn((M, E), generator=g, device=dev)
        y = layer.forward(x, logits)
        tw, ids = fused_topk(x, logits, k, True)
        assert torch.equal(y, layer.routed_forward(x, tw, ids))
        ref = layer_ref(x, tw, ids, bank, None, "silu").cpu().numpy()
        got = y.double().cpu().numpy()
        assert max_rel(got, ref) <= MAX_REL_TOL and cosine(got, ref) >= COS_TOL
        # and near the bf16 layer that it was made from: rounding to 8 bits, four times
        full = ops.experts_decode(x, tw, ids, bf).double().cpu().numpy()
        assert cosine(got, full) >= 0.999
    assert layer.forward(x[:0], logits[:0]).shape == (0, H)


# ----------------------------------------------------------------------------- graphs and streams


@pytest.mark.parametrize("M", [1, 24, 300])
def test_graph_replays_equal_eager(dev, M):
    """Two captured steps of the layer (and of its products alone) that replay in
    turn, with new inputs and eager calls in between, equal the eager calls."""
    g = gen(dev, M)
    E, H, I, k = 32, 512, 256, 4
    bank, shared = make_bank(dev, g, E, H, I), make_bank(dev, g, 1, H, I)
    w = torch.randn((E, 96, H), generator=g, device=dev).to(torch.bfloat16)

    def step(x, tw, ids):
        order, offsets = ops.group_routes(ids, E)
        z = torch.zeros((M * k, 96), dtype=torch.bfloat16, device=dev)
        ops.grouped_matmul(x, w, offsets, order=order, top_k=k, row_weight=tw.view(-1), out=z)
        q, s = ops.act_quant_int8(x)
        return (ops.experts_int8(x, tw, ids, bank, shared=shared), z,
                ops.matmul_int8(q, s, bank.gate_up[3], bank.gate_up_scale[3], out_dtype=torch.float32))

    def inputs():
        return (torch.randn((M, H), generator=g, device=dev).to(torch.bfloat16), *routing(dev, g, M, k, E))

    step(*inputs())
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        bufs = inputs()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*bufs)
        graphs.append((graph, bufs, out))
    for _ in range(3):
        want = []
        for graph, bufs, out in graphs:
            for b, v in zip(bufs, inputs()):
                b.copy_(v)
            want.append(step(*[b.clone() for b in bufs]))
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, _, out), ref in zip(graphs, want):
            for a, b in zip(out, ref):
                assert torch.equal(a, b)


def test_two_streams_at_once(dev):
    """Calls on two streams at the same time do not share scratch memory."""
    g = gen(dev, 77)
    E, H, I, k, M = 16, 512, 256, 4, 128
    bank = make_bank(dev, g, E, H, I)
    ins = [(torch.randn((M, H), generator=g, device=dev).to(torch.bfloat16), *routing(dev, g, M, k, E)) for _ in range(2)]
    want = [ops.experts_int8(*v, bank) for v in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    for _ in range(5):
        got = []
        for st, v in zip(streams, ins):
            with torch.cuda.stream(st):
                got.append(ops.experts_int8(*v, bank))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("shared", [False, True], ids=["routed", "shared"])
@pytest.mark.parametrize("H,I,E,k", [(1024, 512, 16, 2), (2048, 768, 128, 8), (2064, 528, 12, 3)])
def test_layer_does_not_depend_on_the_batch(dev, H, I, E, k, shared):
    """Integer sums and one order of roundings in every form: a token's result is the same alone, in a step of a few
    and in a batch of hundreds."""
    g = gen(dev, H + E)
    bank = make_bank(dev, g, E, H, I)
    sb = make_bank(dev, g, 1, H, I) if shared else None
    x = torch.randn((600, H), generator=g, device=dev).to(torch.bfloat16)
    tw, ids = routing(dev, g, 600, k, E)
    whole = ops.experts_int8(x, tw, ids, bank, shared=sb)
    for first, n in [(0, 1), (1, 2), (7, 4), (30, 9), (64, 40), (300, 299)]:
        part = slice(first, first + n)
        assert torch.equal(ops.experts_int8(x[part], tw[part], ids[part], bank, shared=sb), whole[part]), n


@pytest.mark.parametrize("M", [3, 4, 90])
def test_layer_odd_tokens(dev, M):
    """A token of no expert is zero, one with an infinity or a NaN is NaN in its own row alone; the result may be
    written over the tokens; a step in which no token has an expert."""
    g = gen(dev, M)
    E, H, I, k = 24, 512, 384, 4
    bank = make_bank(dev, g, E, H, I)
    x = torch.randn((M, H), generator=g, device=dev).to(torch.bfloat16)
    tw, ids = routing(dev, g, M, k, E)
    fine = ops.experts_int8(x, tw, ids, bank)
    assert bool(torch.isfinite(fine).all())
    bad = x.clone()
    bad[1, 5], bad[2, 0] = float("nan"), float("-inf")
    ids[0] = -1
    y = ops.experts_int8(bad, tw, ids, bank)
    assert not y[0].any() and bool(torch.isnan(y[1:3]).all()) and torch.equal(y[3:], fine[3:])
    ids[0] = E + 5
    assert ops.experts_int8(x, tw, ids, bank, out=x) is x
    assert not x[0].any() and torch.equal(x[1:], fine[1:])
    assert not ops.experts_int8(x, tw, torch.full_like(ids, E), bank).any()


def test_layer_with_a_limit_in_a_small_step(dev):
    """Clamped SwiGLU, the shared expert's limit its own, the same in a small step as in a batch."""
    g = gen(dev, 21)
    E, H, I, k = 16, 1024, 512, 2
    bank, shared = make_bank(dev, g, E, H, I), make_bank(dev, g, 1, H, I)
    bank.swiglu_limit, shared.swiglu_limit = 0.75, 7.0
    x = torch.randn((400, H), generator=g, device=dev).to(torch.bfloat16)
    tw, ids = routing(dev, g, 400, k, E)
    whole = ops.experts_int8(x, tw, ids, bank, shared=shared)
    for part in (slice(0, 1), slice(1, 12), slice(100, 400)):
        assert torch.equal(ops.experts_int8(x[part], tw[part], ids[part], bank, shared=shared), whole[part])
    bank.swiglu_limit = shared.swiglu_limit = 0.0
    assert not torch.equal(ops.experts_int8(x, tw, ids, bank, shared=shared), whole)
