"""The operators around the fused experts: what a decoder layer runs in front of ``fused_moe_w8a8_up_down``, and the FP8
products of its dense layers.  Callers of the reference take these from their serving engine.

* :func:`rms_norm_quant_fp8` - residual addition, RMS norm and per-token-group FP8 quantisation in one kernel;
* :func:`route_topk`         - the router's selection, in the form ``moe_align_block_size`` and the fused operator take;
* :func:`block_scaled_mm`    - FP8 matrix product with the layer's scales (1 x 128 for tokens, 128 x 128 for weights);
* :func:`swiglu_quant_fp8`   - SwiGLU and quantisation between the two products of a dense layer.

HIP kernels on the current stream of the inputs' device; nothing is kept between calls, so they may be captured into HIP graphs
and run on several streams at once.  Inputs are contiguous.  Inference only: inputs that require gradients are refused while
gradients are recorded, and inputs that carry a forward-mode tangent wherever tangents are, in a trace too.
"""
from typing import NamedTuple, Optional, Tuple

import torch

import alpha_moe  # noqa: F401  (registers the operators; fails if the libraries are not built)

# (the overloads themselves: the lookup of one by name is a microsecond of a call on a few tokens)
_norm = torch.ops.alpha_moe.rms_norm_quant_fp8.default
_norm_keep = torch.ops.alpha_moe.rms_norm_quant_fp8.keep_norm
_add_norm = torch.ops.alpha_moe.add_rms_norm_quant_fp8.default
_add_norm_keep = torch.ops.alpha_moe.add_rms_norm_quant_fp8.keep_norm
_swiglu_quant_fp8 = torch.ops.alpha_moe.swiglu_quant_fp8.default
_block_scaled_mm = torch.ops.alpha_moe.block_scaled_mm.default
_route_topk = torch.ops.alpha_moe.route_topk.default


class NormQuant(NamedTuple):
    """Result of :func:`rms_norm_quant_fp8`; ``residual`` and ``norm`` are None where they were not asked for."""
    q: torch.Tensor
    scale: torch.Tensor
    residual: Optional[torch.Tensor]
    norm: Optional[torch.Tensor]


def rms_norm_quant_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None,
                       keep_norm: bool = False, group_size: int = 128) -> NormQuant:
    """``h = x + residual``; ``y = h / sqrt(mean(h^2) + eps) * weight`` in fp32; ``y`` quantised per token and 128 columns.

    x ``[M, K]`` bf16 or fp32, K a multiple of 128 up to 65536; weight ``[K]`` bf16 or fp32; residual None or like x.  Returns
    ``q [M, K]`` float8_e4m3fn and ``scale [M, K/128]`` float32 of ``y`` (as ``per_token_group_quant_fp8`` defines them, but NaN
    in a group that holds one; a row whose squares add up to more than fp32 holds becomes 0, one whose squares are all below its
    numbers is not a number if ``eps`` is 0), ``residual`` = ``h`` in x's dtype (a new tensor), and with ``keep_norm`` ``norm`` =
    ``y`` in x's dtype, which a router or a bf16 product reads.
    """
    if residual is None:
        if not keep_norm:
            return NormQuant(*_norm(x, weight, eps, group_size), None, None)
        q, scale, norm = _norm_keep(x, weight, eps, group_size)
        return NormQuant(q, scale, None, norm)
    if not keep_norm:
        return NormQuant(*_add_norm(x, residual, weight, eps, group_size), None)
    return NormQuant(*_add_norm_keep(x, residual, weight, eps, group_size))


def swiglu_quant_fp8(gate_up: torch.Tensor, group_size: int = 128) -> Tuple[torch.Tensor, torch.Tensor]:
    """``gate_up [M, 2 I]`` bf16 or fp32, the gate in the first half of the columns (checkpoint order, not interleaved) ->
    ``(q [M, I] float8_e4m3fn, scale [M, I/128] float32)`` of ``silu(gate) * up``, computed in fp32 (where the silu of a gate below
    -88.7 is -0)."""
    return _swiglu_quant_fp8(gate_up, group_size)


def block_scaled_mm(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor) -> torch.Tensor:
    """``out [M, N] = (x * x_scale) (w * w_scale)^T``, rounded once to bfloat16.

    x ``[M, K]`` float8_e4m3fn with x_scale ``[M, K/128]``; w ``[N, K]`` float8_e4m3fn with w_scale ``[ceil(N/128), K/128]``.
    N is of any size, K a multiple of 128 up to 65536.  The product of two scales is taken first, in fp32, and has to be one of its
    normal numbers or 0.  Bit for bit the same from run to run.
    """
    return _block_scaled_mm(x, x_scale, w, w_scale)


def route_topk(logits: torch.Tensor, top_k: int, scoring: str = "softmax", bias: Optional[torch.Tensor] = None,
               num_groups: int = 1, top_groups: int = 1, renormalize: bool = True, shared_experts: int = 0,
               shared_weight: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(topk_weights float32, topk_ids int32)``, both ``[M, top_k + shared_experts]``, from ``logits [M, E]`` bf16 or fp32.

    Scores are ``softmax`` or ``sigmoid`` of the logits.  Experts are chosen by score + ``bias`` (``[E]`` float32, compared in 64
    bits; weights are free of it) or, without one, by logit; equal ones by ascending index.  With ``num_groups`` > 1 only
    the experts of the ``top_groups`` best groups (runs of ``E / num_groups`` experts, ranked by their two best choices' sum, or by their
    best one without a bias) take part.  ``renormalize`` divides a token's weights by their sum.  The last ``shared_experts`` columns
    name the experts E, E + 1, ... fused behind the routed ones, with ``shared_weight`` (1 / routed scaling factor
    where the fused operator scales everything).  E is at most 4096, top_k and num_groups at most 64.

    A NaN ranks last and makes its row's weights NaN (and so does +inf in a softmax); a row whose chosen scores are all 0 (every
    logit -inf) has weights of 0.  Ids are valid whatever the logits hold.  Scores up to e^-700 are 0; above, renormalised weights
    keep their ratio where all chosen scores are too small for fp32 (beside larger ones, and with ``renormalize=False``, one below
    2^-126 may count as 0).
    """
    if scoring not in ("softmax", "sigmoid"):
        raise ValueError(f"scoring must be 'softmax' or 'sigmoid', got {scoring!r}")
    return _route_topk(logits, bias, top_k, scoring == "sigmoid", num_groups, top_groups, renormalize, shared_experts,
                       shared_weight)
