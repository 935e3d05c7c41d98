"""What an SGLang-on-ROCm build calls to run its fused-MoE layers through this operator.

The reference wires itself into SGLang with a patch (extra/sglang.patch: the weight loader interleaves ``w13`` and
its block scales once both halves of an expert have arrived, lines 46-98; ``fused_experts_impl`` is short-circuited
into quantise -> align -> operator, lines 1-44).  ``extra/sglang_rocm.patch`` of this repository is the same wiring
for a ROCm build, and keeps the logic here so that it can be exercised without SGLang:

* :class:`W13Interleaver` - the weight-loader bookkeeping;
* :func:`fused_experts`   - the forward path, with this library's own HIP quantiser and aligner in place of SGLang's
  helpers and the storing variant of the operator in place of zero-fill + add;
* :func:`norm_moe`, :func:`norm_dense_mlp` - the feed-forward halves of a decoder layer from the residual addition on, an
  expert layer and a dense one, on this library's norm, router and block-scaled product (the reference has no part of
  these; its callers take them from SGLang);
* :func:`norm_sorted_moe` - an expert layer whose experts are spread over GPUs or whose weights the fused operator does not take,
  on sorted tokens and one product for all experts.
"""
import os
from typing import NamedTuple, Optional, Tuple

import torch

from .utils import get_best_config, interleave_tensor


class W13Interleaver:
    """Counts the gate (``w1``) and up (``w3``) shards an expert's fused ``w13`` slot has received and, once both are
    there, rewrites the slot in the operator's interleaved row order - chunks of 8 rows for weights, of 1 row for
    128x128 block scales (reference extra/sglang.patch:71-78,87-94)."""

    def __init__(self, num_experts: int, rep: int):
        self.rep = rep
        self.halves_loaded = [0] * num_experts

    def shard_loaded(self, expert_data: torch.Tensor, expert_id: int, shard_id: str) -> bool:
        """Call after the loader has copied ``shard_id`` into ``expert_data`` (the expert's ``[N, K]`` slot of the
        parameter).  Returns True when this call interleaved the slot."""
        if shard_id not in ("w1", "w3", "w13"):
            return False
        self.halves_loaded[expert_id] += 2 if shard_id == "w13" else 1
        if self.halves_loaded[expert_id] != 2:
            return False
        expert_data.copy_(interleave_tensor(expert_data.unsqueeze(0), self.rep)[0])
        return True


def fused_experts(hidden_states: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, topk_weights: torch.Tensor,
                  topk_ids: torch.Tensor, w13_scale: torch.Tensor, w2_scale: torch.Tensor,
                  routed_scaling_factor: Optional[float] = None, config_path: Optional[str] = None,
                  group_size: int = 128) -> torch.Tensor:
    """The body ``fused_experts_impl`` is replaced with (reference extra/sglang.patch:18-41): tuning knobs from the
    table ``ALPHA_MOE_CONFIG`` names, per-token-group FP8 quantisation of ``hidden_states``, block alignment of the
    routing, the fused operator.  ``hidden_states`` ``[M, K]`` bf16 is overwritten with the result and returned, as in
    the reference (which zero-fills it and adds; the storing variant needs no zero-fill)."""
    import alpha_moe  # noqa: F401  registers the operators

    config_path = config_path or os.environ["ALPHA_MOE_CONFIG"]
    cfg = get_best_config(config_path, hidden_states.shape[0])
    if topk_ids.dtype != torch.int32:
        topk_ids = topk_ids.to(torch.int32)
    torch.ops.alpha_moe.fused_experts(
        hidden_states, topk_ids.contiguous(), w13, w13_scale, w2, w2_scale, topk_weights.to(torch.float32), group_size,
        cfg["block_m"], cfg["block_n"], cfg["warp_n"], cfg["stages"], routed_scaling_factor or 1.0)
    return hidden_states


def norm_moe(hidden_states: torch.Tensor, residual: torch.Tensor, norm_weight: torch.Tensor, gate_weight: torch.Tensor,
             w13: torch.Tensor, w2: torch.Tensor, w13_scale: torch.Tensor, w2_scale: torch.Tensor, top_k: int,
             scoring: str = "softmax", correction_bias: Optional[torch.Tensor] = None, num_groups: int = 1, top_groups: int = 1,
             renormalize: bool = True, routed_scaling_factor: Optional[float] = None, eps: float = 1e-6,
             config_path: Optional[str] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """An expert layer from the residual addition on: ``(output, residual)``, both ``[M, K]`` bf16.

    ``residual + hidden_states`` is normalised and quantised in one kernel, the bf16 row goes through the gate (a plain
    product in ``gate_weight``'s type, ``[E_routed, K]``), the router picks ``top_k`` experts (``route_topk``), and the fused
    operator reads the codes.  ``w13 [E, N, K]`` and its scales are interleaved as for :func:`fused_experts`.  Experts that
    ``w13`` has beyond the gate's are shared ones: every token visits them, with a weight of 1 after the operator's
    ``routed_scaling_factor``.  The aligner is a launch of its own at any number of tokens (:func:`fused_experts`
    does without up to 16), and a ``correction_bias`` that is not fp32 is converted in every call."""
    from .layer_hip import rms_norm_quant_fp8, route_topk
    from .prep_hip import moe_align_block_size

    experts = w13.shape[0]
    shared = experts - gate_weight.shape[0]
    if shared < 0:
        raise ValueError(f"the gate has {gate_weight.shape[0]} experts, w13 only {experts}")
    scaling = routed_scaling_factor or 1.0
    bias = None if correction_bias is None else correction_bias.to(torch.float32)
    cfg = get_best_config(config_path or os.environ["ALPHA_MOE_CONFIG"], hidden_states.shape[0])
    x = rms_norm_quant_fp8(hidden_states, norm_weight, eps, residual=residual, keep_norm=True)
    out = torch.empty_like(hidden_states)
    if hidden_states.shape[0] == 0:
        return out, x.residual
    logits = torch.nn.functional.linear(x.norm.to(gate_weight.dtype), gate_weight)
    weights, ids = route_topk(logits, top_k, scoring=scoring, bias=bias, num_groups=num_groups, top_groups=top_groups,
                              renormalize=renormalize, shared_experts=shared, shared_weight=1.0 / scaling)
    aligned = moe_align_block_size(ids, cfg["block_m"], experts)
    torch.ops.alpha_moe.fused_moe_w8a8_up_down_store(
        x.q, x.scale, w13, w13_scale, w2, w2_scale, *aligned, weights, out, top_k + shared, cfg["block_m"], cfg["block_n"],
        cfg["warp_n"], cfg["stages"], scaling)
    return out, x.residual


def norm_sorted_moe(hidden_states: torch.Tensor, residual: torch.Tensor, norm_weight: torch.Tensor, gate_weight: torch.Tensor,
                    w13: torch.Tensor, w2: torch.Tensor, w13_scale: torch.Tensor, w2_scale: torch.Tensor, top_k: int,
                    scoring: str = "softmax", correction_bias: Optional[torch.Tensor] = None, num_groups: int = 1,
                    top_groups: int = 1, renormalize: bool = True, routed_scaling_factor: Optional[float] = None,
                    eps: float = 1e-6, first_expert: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """An expert layer from the residual addition on, of which this GPU holds the experts ``first_expert, first_expert + 1, ...``:
    ``(output, residual)``, both ``[M, K]`` bf16; the outputs of all GPUs add up to the layer's.

    ``w13 [E, 2 I, K]`` and ``w2 [E, K, I]`` are in checkpoint order (the gate's rows, then the up projection's, NOT interleaved) with
    scales per 128 x 128 block; ``gate_weight`` has the rows of all GPUs' experts.  Every token is routed; the slots of this GPU's experts
    are sorted by expert as FP8 codes, go through both products, and come back as weighted sums.  Where the whole
    layer's experts are here and interleaved, :func:`norm_moe` is the faster way."""
    from .layer_hip import (combine_tokens, grouped_block_scaled_mm, rms_norm_quant_fp8, route_topk, sort_tokens,
                            swiglu_quant_fp8)

    experts = w13.shape[0]
    if first_expert < 0 or first_expert + experts > gate_weight.shape[0]:
        raise ValueError(f"experts {first_expert} to {first_expert + experts - 1} are not all of the gate's {gate_weight.shape[0]}")
    bias = None if correction_bias is None else correction_bias.to(torch.float32)
    x = rms_norm_quant_fp8(hidden_states, norm_weight, eps, residual=residual, keep_norm=True)
    logits = torch.nn.functional.linear(x.norm.to(gate_weight.dtype), gate_weight)
    weights, ids = route_topk(logits, top_k, scoring=scoring, bias=bias, num_groups=num_groups, top_groups=top_groups,
                              renormalize=renormalize)
    if first_expert:
        ids = ids - first_expert
    s = sort_tokens(x.q, ids, experts, x_scale=x.scale)
    q, scale = swiglu_quant_fp8(grouped_block_scaled_mm(s.rows, s.scale, s.offsets, w13, w13_scale))
    rows = grouped_block_scaled_mm(q, scale, s.offsets, w2, w2_scale)
    return combine_tokens(rows, s.row_of_slot, weights, 1.0 if routed_scaling_factor is None else routed_scaling_factor), x.residual


class Adapters(NamedTuple):
    """Low-rank adapters of a dense layer's two products, and which of them each token has (``layer_hip.add_adapters``)."""
    a13: torch.Tensor
    b13: torch.Tensor
    a2: torch.Tensor
    b2: torch.Tensor
    ids: torch.Tensor
    scale: Optional[torch.Tensor] = None


def norm_dense_mlp(hidden_states: torch.Tensor, residual: torch.Tensor, norm_weight: torch.Tensor, w13: torch.Tensor,
                   w2: torch.Tensor, w13_scale: torch.Tensor, w2_scale: torch.Tensor, eps: float = 1e-6,
                   adapters: Optional[Adapters] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """A dense layer (or an unfused shared expert) from the residual addition on: ``(output, residual)``, both ``[M, K]`` bf16.

    ``w13 [2 I, K]`` holds the gate's rows, then the up projection's, as checkpoints do (NOT interleaved), ``w2 [K, I]``; scales
    are per 128 x 128 block.  Four kernels: norm, product, SwiGLU, product.  With ``adapters`` (``a13 [L, rank, K]``, ``b13 [L, 2 I, rank]``,
    ``a2 [L, rank, I]``, ``b2 [L, K, rank]``) two more behind each product, which read the codes that it reads."""
    from .layer_hip import add_adapters, block_scaled_mm, rms_norm_quant_fp8, swiglu_quant_fp8

    x = rms_norm_quant_fp8(hidden_states, norm_weight, eps, residual=residual)
    gate_up = block_scaled_mm(x.q, x.scale, w13, w13_scale)
    if adapters is not None:
        gate_up = add_adapters(gate_up, x.q, adapters.a13, adapters.b13, adapters.ids, adapters.scale, x.scale)
    q, scale = swiglu_quant_fp8(gate_up)
    out = block_scaled_mm(q, scale, w2, w2_scale)
    if adapters is not None:
        out = add_adapters(out, q, adapters.a2, adapters.b2, adapters.ids, adapters.scale, scale)
    return out, x.residual
