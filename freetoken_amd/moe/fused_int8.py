"""8-bit integer (W8A8) routed experts: int8 weights with one float32 scale per
output channel, tokens quantised with one scale each, for decode and prefill
alike.  No counterpart in the reference; the signature is that of
``fused_fp8_block.py``.  ``topk_ids`` index bank rows, ids outside them are
skipped."""

from __future__ import annotations

from .. import ops


def fused_experts_int8(
    hidden_states, gate_up, gate_up_scale, down, down_scale,
    topk_weights, topk_ids, activation="silu",
    apply_router_weight_on_input=False, shared: ops.ExpertBank | None = None,
):
    assert not apply_router_weight_on_input
    bank = ops.ExpertBank("int8", gate_up, down, gate_up_scale, down_scale)
    return ops.experts_int8(hidden_states, topk_weights, topk_ids, bank, shared=shared, activation=activation)


__all__ = ["fused_experts_int8"]
