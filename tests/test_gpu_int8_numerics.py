"""Numerics of the int8 products and the int8 expert layer at their edges, against
64 bits.

Roundings: to float32 at most 2^-24 of the value, to bf16 2^-8.  A product's row is
an exact integer converted to float32 and multiplied by its factors: five roundings
at most, below 2^-21.  A sum of n float32 values in order is off by at most n 2^-24
of the sum of their magnitudes.
"""

from __future__ import annotations

import pytest
import torch

from freetoken_amd import ops
from freetoken_amd.layers.moe import MoELayer
from freetoken_amd.moe.fused_int8 import fused_experts_int8

from test_gpu_int8 import BF16, F32, gen, grouped_ref, int8_rows, make_bank, routing, scales, within

pytestmark = pytest.mark.gpu


def activations(x, ids, bank, act="silu"):
    """Codes and scales of the routes' activations between the two products, from the operators one by one."""
    M, k = ids.shape
    q, s = ops.act_quant_int8(x)
    order, offsets = ops.group_routes(ids, bank.num_rows)
    h = torch.zeros((M * k, bank.inter), dtype=torch.bfloat16, device=x.device)
    ops.grouped_matmul(q, bank.gate_up, offsets, order=order, top_k=k, x_scale=s, w_scale=bank.gate_up_scale,
                       activation=act, out=h)
    return ops.act_quant_int8(h)


def down_rows(hq, hs, ids, bank, tw):
    """The routes' weighted rows in 64 bits, [M, k, H]; zeros where a route has no expert."""
    flat = ids.view(-1)
    rows = torch.zeros((flat.numel(), bank.hidden), dtype=torch.float64, device=hq.device)
    for e in range(bank.num_rows):
        at = torch.nonzero(flat == e)[:, 0]
        if at.numel():
            rows[at] = (hq[at].double() @ bank.down[e].double().T) * hs[at].double()[:, None] * bank.down_scale[e].double()
    return (rows * tw.double().view(-1, 1)).view(*ids.shape, -1)


@pytest.mark.parametrize("M,k,E,H,I,Is", [(1, 2, 16, 1024, 512, 0), (1, 8, 128, 2048, 768, 768), (3, 9, 12, 272, 144, 48),
                                          (40, 4, 8, 2064, 400, 400), (300, 8, 16, 640, 384, 16),
                                          (1500, 6, 16, 512, 256, 256)])
def test_float32_rows_are_rounded_once(dev, M, k, E, H, I, Is):
    """With float32 rows nothing between the down products and the result is rounded to fewer bits: the error is that
    of one rounding to bf16, however far the routes cancel."""
    g = gen(dev, M + H)
    bank, shared = make_bank(dev, g, E, H, I), make_bank(dev, g, 1, H, Is) if Is else None
    x = torch.randn((M, H), generator=g, device=dev).to(torch.bfloat16)
    tw, ids = routing(dev, g, M, k, E)
    if M > 2:
        ids[1::3] = -1
        ids[0, 0] = E
    y = ops.experts_int8(x, tw, ids, bank, shared=shared, route_dtype=torch.float32)
    rows = down_rows(*activations(x, ids, bank), ids, bank, tw)
    if shared is not None:
        one = torch.zeros((M, 1), dtype=torch.int32, device=dev)
        rows = torch.cat([rows, down_rows(*activations(x, one, shared), one, shared, torch.ones((M, 1), device=dev))], 1)
    ref, size = rows.sum(1), rows.abs().sum(1)
    off = size * (F32 + (k + 1) * 2.0**-24)
    within(y, ref, off + (ref.abs() + off) * BF16)
    # (rows rounded to bf16 first are not within it)
    y = ops.experts_int8(x, tw, ids, bank, shared=shared)
    assert not bool(((y.double() - ref).abs() <= off + (ref.abs() + off) * BF16).all())


def test_layer_module_keeps_float32_rows(dev):
    """MoELayer sums the routes from float32 rows, in small steps and batches, with a shared expert and without."""
    g = gen(dev, 31)
    E, H, I, k = 16, 512, 256, 4
    bank, shared = make_bank(dev, g, E, H, I), make_bank(dev, g, 1, H, I)
    layer = MoELayer(E, k, H, I, weight_format="int8", device=dev)
    for name in ("gate_up", "down"):
        getattr(layer, name + "_proj").copy_(getattr(bank, name))
        getattr(layer, name + "_scale").copy_(getattr(bank, name + "_scale"))
    for M in (1, 7, 500):
        x = torch.randn((M, H), generator=g, device=dev).to(torch.bfloat16)
        tw, ids = routing(dev, g, M, k, E)
        for layer.shared_expert in (None, shared):
            want = ops.experts_int8(x, tw, ids, bank, shared=layer.shared_expert, route_dtype=torch.float32)
            assert torch.equal(layer.routed_forward(x, tw, ids), want)


def test_float32_rows_do_not_depend_on_the_batch(dev):
    g = gen(dev, 32)
    E, H, I, k = 128, 2048, 768, 8
    bank, shared = make_bank(dev, g, E, H, I), make_bank(dev, g, 1, H, I)
    x = torch.randn((600, H), generator=g, device=dev).to(torch.bfloat16)
    tw, ids = routing(dev, g, 600, k, E)
    whole = ops.experts_int8(x, tw, ids, bank, shared=shared, route_dtype=torch.float32)
    for first, n in [(0, 1), (1, 2), (7, 4), (64, 40), (300, 299)]:
        part = slice(first, first + n)
        y = ops.experts_int8(x[part], tw[part], ids[part], bank, shared=shared, route_dtype=torch.float32)
        assert torch.equal(y, whole[part]), n


@pytest.mark.parametrize("M", [2, 200])
def test_float32_rows_in_a_replayed_graph(dev, M):
    """A captured layer replayed with new inputs, eager calls in between."""
    g = gen(dev, M)
    E, H, I, k = 32, 512, 256, 4
    bank, shared = make_bank(dev, g, E, H, I), make_bank(dev, g, 1, H, I)

    def inputs():
        return (torch.randn((M, H), generator=g, device=dev).to(torch.bfloat16), *routing(dev, g, M, k, E))

    def step(x, tw, ids):
        return ops.experts_int8(x, tw, ids, bank, shared=shared, route_dtype=torch.float32)

    step(*inputs())
    torch.cuda.synchronize()
    bufs, graph = inputs(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*bufs)
    for _ in range(3):
        for b, v in zip(bufs, inputs()):
            b.copy_(v)
        want = step(*[b.clone() for b in bufs])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("shared", [False, True], ids=["routed", "shared"])
@pytest.mark.parametrize("M,H,I", [(3, 512, 256), (4, 2048, 768), (6, 2064, 528), (90, 512, 384), (400, 1024, 512)])
def test_clamped_swiglu_keeps_nan(dev, M, H, I, shared):
    """With a limit too, a token with an infinity or a NaN is NaN in its own row alone, whatever the step's size."""
    g = gen(dev, M + H)
    E, k = 24, 4
    bank, sb = make_bank(dev, g, E, H, I), make_bank(dev, g, 1, H, I) if shared else None
    for b in (bank, sb) if shared else (bank,):
        b.swiglu_limit = 0.75
    x = torch.randn((M, H), generator=g, device=dev).to(torch.bfloat16)
    tw, ids = routing(dev, g, M, k, E)
    fine = ops.experts_int8(x, tw, ids, bank, shared=sb)
    assert bool(torch.isfinite(fine).all())
    x[1, 5], x[2, 0] = float("nan"), float("-inf")
    y = ops.experts_int8(x, tw, ids, bank, shared=sb)
    assert bool(torch.isnan(y[1:3]).all())
    keep = [i for i in range(M) if i not in (1, 2)]
    assert torch.equal(y[keep], fine[keep])


def test_clamped_swiglu_of_finite_values(dev):
    """The clamp at its borders: gates and ups beyond, at and within the limit, and infinite products of finite rows."""
    H = I = 16
    one, more = torch.ones((1, 2 * I), device=dev), torch.ones((1, H), device=dev)
    bank = ops.ExpertBank("int8", torch.zeros((1, 2 * I, H), dtype=torch.int8, device=dev),
                          torch.zeros((1, H, I), dtype=torch.int8, device=dev), one, more, swiglu_limit=2.0)
    bank.gate_up[0, :I, 0] = torch.tensor([0, 1, -1, 2, 3, 127, -127, 4, 2, 2, 2, 2, 2, 2, 2, 2], device=dev)
    bank.gate_up[0, I:, 0] = torch.tensor([5, 1, -1, 2, -2, 3, -3, 127, -127, 2, 0, 1, 4, -4, 1, 1], device=dev)
    bank.gate_up_scale[0, 14] = float("inf")  # an infinite gate is capped, an infinite up clamped
    bank.gate_up_scale[0, I + 15] = float("inf")
    bank.down[0, torch.arange(I), torch.arange(I)] = 127
    for M in (1, 40, 400):
        x = torch.zeros((M, H), dtype=torch.bfloat16, device=dev)
        x[:, 0] = 1.0  # codes 127 of 1/127: one
        ids = torch.zeros((M, 1), dtype=torch.int32, device=dev)
        tw = torch.ones((M, 1), device=dev)
        y = ops.experts_int8(x, tw, ids, bank, route_dtype=torch.float32)
        h = (bank.gate_up[0, :, 0].double() * bank.gate_up_scale[0].double()).clamp(max=1e30)
        gate, up = h[:I].clamp(max=2.0), h[I:].clamp(-2.0, 2.0)
        a = (gate * torch.sigmoid(gate) * up).to(torch.bfloat16).double()
        want = (127 * a / a.abs().max()).round() * a.abs().max()
        within(y, want.expand(M, -1), want.abs() * (BF16 + F32))


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("M", [1, 40, 300])
def test_silu_relative_to_its_result(dev, M, out_dtype):
    """silu(gate) up over gates from -88 to 88, the smallest results among normal numbers, relative to the result: the
    exponential of x is off by about |x| 2^-24 and 2^-22 relative, the other operations by 2^-21 together: below 2^-16."""
    g = gen(dev, M)
    K, n = 16, 1760
    gate = (torch.arange(n, device=dev) - n / 2 + 0.5).mul_(0.1)
    q = torch.zeros((M, K), dtype=torch.int8, device=dev)
    q[:, 0] = 1
    w = torch.zeros((2 * n, K), dtype=torch.int8, device=dev)
    w[:, 0] = 1
    ws = torch.cat([gate, torch.rand(n, generator=g, device=dev) + 1.0])  # (a channel's scale may be any number)
    y = ops.matmul_int8(q, torch.ones(M, device=dev), w, ws, activation="silu", out_dtype=out_dtype)
    ref = (gate.double() * torch.sigmoid(gate.double()) * ws[n:].double()).expand(M, -1)
    assert float(ref.abs().min()) > 2.0**-126
    within(y, ref, ref.abs() * (2.0**-16 + (BF16 if out_dtype == torch.bfloat16 else 0)))


# (largest magnitudes of the rows, of the weights), so that a product of scales leaves the normal numbers on the way
FAR = [(2.0**-117, 2.0**-4), (2.0**-120, 2.0**-3), (2.0**-60, 2.0**-62), (2.0**126, 2.0**-110), (2.0**127, 2.0**-126),
       (2.0**-126, 2.0**120), (2.0**64, 2.0**50), (2.0**100, 2.0**-40)]


@pytest.mark.parametrize("top,wtop", FAR, ids=range(len(FAR)))
@pytest.mark.parametrize("M", [1, 40, 300])
def test_far_scales(dev, M, top, wtop):
    """Rows and weights far from 1: the exact sum times its factors, right wherever the result and each scale are
    normal float32 numbers; a sum of zero is zero."""
    g = gen(dev, M)
    N, K = 200, 272
    x = torch.randint(-128, 129, (M, K), generator=g, device=dev).double().mul_(2.0**-8)
    x[:, 3] = 1.0
    q, s = ops.act_quant_int8((x * top).to(torch.bfloat16))
    w, ws = int8_rows(dev, g, N, K), (torch.rand(N, generator=g, device=dev) + 1.0).mul_(wtop / 254)
    w[7] = 0
    sums = q.double() @ w.double().T
    ref = sums * s.double()[:, None] * ws.double()
    # scales below the normal numbers hold fewer bits themselves, and are compared as they are
    normal = (ref.abs() >= 2.0**-126) & (ref.abs() < 2.0**127) | (sums == 0)
    assert int(normal.sum()) >= normal.numel() // 2
    y = ops.matmul_int8(q, s, w, ws, out_dtype=torch.float32)
    within(torch.where(normal, y.double(), 0.0), torch.where(normal, ref, 0.0), ref.abs() * F32)
    assert torch.equal(ops.matmul_int8(q, -s, w, ws, out_dtype=torch.float32), -y)  # a scale's sign is its own
    offsets = torch.tensor([0, M], dtype=torch.int32, device=dev)
    weight = torch.rand(M, generator=g, device=dev)
    y = ops.grouped_matmul(q, w[None], offsets, x_scale=s, w_scale=ws[None], row_weight=weight)
    ref = ref * weight.double()[:, None]
    normal &= (ref.abs() >= 2.0**-126) | (sums == 0)
    within(torch.where(normal, y.double(), 0.0), torch.where(normal, ref, 0.0), ref.abs() * (F32 + BF16))


@pytest.mark.parametrize("M", [2, 300])
def test_fused_experts_int8(dev, M):
    """The functional form and MoELayer are ops.experts_int8 with float32 rows, the clamp of a model with clamped SwiGLU
    among their arguments."""
    g = gen(dev, M)
    E, H, I, k = 16, 512, 256, 4
    bank, shared = make_bank(dev, g, E, H, I), make_bank(dev, g, 1, H, I)
    x = torch.randn((M, H), generator=g, device=dev).to(torch.bfloat16)
    tw, ids = routing(dev, g, M, k, E)
    layer = MoELayer(E, k, H, I, weight_format="int8", device=dev)
    for name in ("gate_up", "down"):
        getattr(layer, name + "_proj").copy_(getattr(bank, name))
        getattr(layer, name + "_scale").copy_(getattr(bank, name + "_scale"))
    arrays = (bank.gate_up, bank.gate_up_scale, bank.down, bank.down_scale)
    results = []
    for limit in (None, 0.0, 0.5):
        for sb in (None, shared):
            bank.swiglu_limit = limit or 0.0
            want = ops.experts_int8(x, tw, ids, bank, shared=sb, route_dtype=torch.float32)
            assert torch.equal(fused_experts_int8(x, *arrays, tw, ids, shared=sb, swiglu_limit=limit), want)
            layer.swiglu_limit, layer.shared_expert = limit, sb
            assert torch.equal(layer.routed_forward(x, tw, ids), want)
            results.append(want)
    assert torch.equal(results[0], results[2]) and not torch.equal(results[2], results[4])
    assert torch.equal(fused_experts_int8(x, *arrays, tw, ids), results[0])
    gelu = fused_experts_int8(x, *arrays, tw, ids, activation="gelu")
    bank.swiglu_limit = 0.0
    assert torch.equal(gelu, ops.experts_int8(x, tw, ids, bank, activation="gelu", route_dtype=torch.float32))
    with pytest.raises(ValueError, match="silu"):
        fused_experts_int8(x, *arrays, tw, ids, activation="gelu", swiglu_limit=0.5)
    with pytest.raises(ValueError, match="swiglu_limit"):
        fused_experts_int8(x, *arrays, tw, ids, swiglu_limit=float("nan"))


def test_most_features(dev):
    """As many output channels as a product takes: their scales and results past 2^31 bytes."""
    g = gen(dev, 41)
    K = 16
    for N in (1 << 30, (1 << 29) + 24, (1 << 28) + 40):
        q, s = int8_rows(dev, g, 2, K), scales(dev, g, 2)
        w, ws = int8_rows(dev, g, N, K), scales(dev, g, N)
        at = torch.cat([torch.arange(300, device=dev), torch.randint(0, N, (3000,), generator=g, device=dev),
                        N - 1 - torch.arange(300, device=dev), (N // 2 + torch.arange(-150, 150, device=dev))])
        ref = (q.double() @ w[at].double().T) * s.double()[:, None] * ws[at].double()
        y = ops.matmul_int8(q, s, w, ws)
        within(y[:, at], ref, ref.abs() * (F32 + BF16))
        offsets = torch.tensor([0, 2], dtype=torch.int32, device=dev)
        y = ops.grouped_matmul(q, w[None], offsets, x_scale=s, w_scale=ws[None])
        within(y[:, at], ref, ref.abs() * (F32 + BF16))
        del y, w, ws


@pytest.mark.parametrize("rows,K", [((1 << 26) + 5, 16), ((1 << 24) + 3, 2064)])
def test_quant_more_rows_than_a_launch(dev, rows, K):
    """More rows than one launch has threads for: the codes and scales of the rows alone."""
    x = torch.empty((rows, K), dtype=torch.bfloat16, device=dev).normal_(generator=gen(dev, K))
    q, s = ops.act_quant_int8(x)
    for first in (0, (1 << 23) - 50, (1 << 24) - 50, rows - 100):
        part = slice(max(0, first), min(rows, first + 100))
        qp, sp = ops.act_quant_int8(x[part])
        assert torch.equal(q[part], qp) and torch.equal(s[part], sp)
    top = torch.stack([x[i : i + (1 << 22)].abs().amax(1).float().sum(dtype=torch.float64) for i in range(0, rows, 1 << 22)])
    assert abs(float(s.sum(dtype=torch.float64) * 127 / top.sum()) - 1) < 1e-6


def test_layer_of_more_tokens_than_a_launch(dev):
    """An expert layer of more (short) tokens than the grouping's launch can quantise beside it."""
    M, H, I, E = (1 << 24) + 7, 16, 16, 3
    g = gen(dev, 51)
    bank = make_bank(dev, g, E, H, I)
    x = torch.empty((M, H), dtype=torch.bfloat16, device=dev).normal_(generator=g)
    ids = torch.randint(0, E, (M, 1), generator=g, device=dev, dtype=torch.int32)
    tw = torch.rand((M, 1), generator=g, device=dev)
    y = ops.experts_int8(x, tw, ids, bank, route_dtype=torch.float32)
    for first in (0, (1 << 23) - 50, M - 100):
        part = slice(first, first + 100)
        assert torch.equal(y[part], ops.experts_int8(x[part], tw[part], ids[part], bank, route_dtype=torch.float32))


@pytest.mark.parametrize("E", [1, 16, 1023])
@pytest.mark.parametrize("numel", [2048 * 63 + 1, 2048 * 64 - 1, 2048 * 65, 1_200_001, 2048 * 1025 + 3, 30_000_000])
def test_group_routes_long(dev, numel, E):
    """Long lists of routes: stable, with ids of no expert left out and the tail filled."""
    ids = torch.randint(-2, E + 3, (numel,), generator=gen(dev, numel + E), device=dev, dtype=torch.int32)
    if E > 1:
        ids[numel // 3 : numel // 2] = E // 2  # a long run of one expert
    order, offsets = ops.group_routes(ids, E)
    key = torch.where((ids < 0) | (ids > E), E + 1, ids)
    counts = torch.bincount(key, minlength=E + 2)
    assert torch.equal(offsets.long(), torch.cat([counts.new_zeros(1), counts[:E].cumsum(0)]))
    listed = int(counts[: E + 1].sum())
    assert torch.equal(order[:listed].long(), torch.sort(key, stable=True).indices[:listed])
    assert bool((order[listed:] == numel).all())


def test_group_routes_longest(dev):
    """The most routes that 32 bits count, few of them of an expert: the places near both ends."""
    numel, E = (1 << 31) - 1, 5
    ids = torch.full((numel,), -1, dtype=torch.int32, device=dev)
    at = torch.tensor([0, 2047, 2048, 1 << 30, numel - 2049, numel - 2, numel - 1], device=dev)
    ids[at] = torch.tensor([3, 0, 3, 4, 0, 3, 0], dtype=torch.int32, device=dev)
    order, offsets = ops.group_routes(ids, E)
    assert offsets.tolist() == [0, 3, 3, 3, 6, 7]
    assert order[:7].tolist() == [2047, numel - 2049, numel - 1, 0, 2048, numel - 2, 1 << 30]
    assert all(bool((part == numel).all()) for part in order[7:].split(1 << 28))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("counts", [[3, 0, 1], [70, 5, 0, 129], [300, 700]], ids=range(3))
@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_grouped_activation_with_weights(dev, counts, int8, act):
    """An activation and row weights together, in a routed order: row_weight * act(gate) * up."""
    E, R, N, K = len(counts), sum(counts), 140, 272
    g = gen(dev, R)
    if int8:
        x, w, xs, ws = int8_rows(dev, g, R, K), int8_rows(dev, g, E, N, K), scales(dev, g, R), scales(dev, g, E, N)
    else:
        x = torch.randn((R, K), generator=g, device=dev).to(torch.bfloat16)
        w, xs, ws = torch.randn((E, N, K), generator=g, device=dev).mul_(0.1).to(torch.bfloat16), None, None
    weight = torch.randn(R, generator=g, device=dev)
    order = torch.randperm(R, generator=g, device=dev).to(torch.int32)
    offsets = torch.tensor([0] + counts, dtype=torch.int32, device=dev).cumsum(0, dtype=torch.int32)
    y = ops.grouped_matmul(x, w, offsets, order=order, x_scale=xs, w_scale=ws, row_weight=weight, activation=act)
    at = order.long()
    ref, err = grouped_ref(x, w, counts, (at, at), act, weight, xs, ws)
    within(y, ref, err)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("M,k,E,H,I", [(1, 8, 128, 2048, 768), (4, 2, 16, 1024, 512), (2, 4, 16, 4096, 512)])
def test_small_steps_with_every_activation(dev, M, k, E, H, I, act):
    """Steps that quantise inside the products give the operators' results one by one, whatever the activation."""
    g = gen(dev, M + H)
    bank = make_bank(dev, g, E, H, I)
    x = torch.randn((M, H), generator=g, device=dev).to(torch.bfloat16)
    tw, ids = routing(dev, g, M, k, E)
    y = ops.experts_int8(x, tw, ids, bank, activation=act, route_dtype=torch.float32)
    rows = down_rows(*activations(x, ids, bank, act), ids, bank, tw)
    ref, off = rows.sum(1), rows.abs().sum(1) * (F32 + (k + 1) * 2.0**-24)
    within(y, ref, off + (ref.abs() + off) * BF16)
