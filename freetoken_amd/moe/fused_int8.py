"""8-bit integer (W8A8) routed experts: int8 weights with one float32 scale per
output channel, tokens quantised with one scale each, for decode and prefill
alike.  No counterpart in the reference; the signature is that of
``fused_fp8_block.py``.  ``topk_ids`` index bank rows, ids outside them are
skipped.  ``swiglu_limit`` > 0 clamps the SwiGLU inputs as in ``fused_ds_fp4.py``
(silu only); 0 (or None) leaves them unclamped.  A token's rows are summed in
float32 unrounded."""

from __future__ import annotations

import torch

from .. import ops


def fused_experts_int8(
    hidden_states, gate_up, gate_up_scale, down, down_scale,
    topk_weights, topk_ids, activation="silu",
    apply_router_weight_on_input=False, shared: ops.ExpertBank | None = None,
    swiglu_limit: float | None = 0.0,
):
    assert not apply_router_weight_on_input
    bank = ops.ExpertBank("int8", gate_up, down, gate_up_scale, down_scale, swiglu_limit=float(swiglu_limit or 0.0))
    return ops.experts_int8(hidden_states, topk_weights, topk_ids, bank, shared=shared, activation=activation,
                            route_dtype=torch.float32)


__all__ = ["fused_experts_int8"]
