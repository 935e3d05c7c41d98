"""The operators around the fused experts: what a decoder layer runs in front of ``fused_moe_w8a8_up_down``, the FP8 products of
its dense layers, and what brings tokens to weights of their own outside the fused call.  Callers of the reference take these from
their serving engine.

* :func:`rms_norm_quant_fp8` - residual addition, RMS norm and per-token-group FP8 quantisation in one kernel;
* :func:`route_topk`         - the router's selection, in the form ``moe_align_block_size`` and the fused operator take;
* :func:`block_scaled_mm`    - FP8 matrix product with the layer's scales (1 x 128 for tokens, 128 x 128 for weights);
* :func:`swiglu_quant_fp8`   - SwiGLU and quantisation between the two products of a dense layer;
* :func:`sort_tokens`, :func:`combine_tokens` - the tokens of all routing slots sorted by expert, and their weighted sums back;
* :func:`grouped_block_scaled_mm` - the block-scaled product of sorted tokens with each expert's weights;
* :func:`add_adapters`       - low-rank adapters of many requests beside a shared projection.

HIP kernels on the current stream of the inputs' device; nothing is kept between calls, so they may be captured into HIP graphs
and run on several streams at once.  Inputs are contiguous.  :func:`sort_tokens` and :func:`combine_tokens` are differentiable (once:
what has no second derivative says so), capture forward and backward pass together, and hold no eager graph of the same
leaves while a backward pass is captured.  The others are for inference only: inputs that require gradients are refused while gradients
are recorded, and inputs that carry a forward-mode tangent wherever tangents are, by all of them, in a trace too.
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
_sort_tokens = torch.ops.alpha_moe.sort_tokens.default
_sort_tokens_scaled = torch.ops.alpha_moe.sort_tokens.scaled
_combine_tokens = torch.ops.alpha_moe.combine_tokens.default
_add_adapters = torch.ops.alpha_moe.add_adapters.default
_grouped_block_scaled_mm = torch.ops.alpha_moe.grouped_block_scaled_mm.default


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


class SortedTokens(NamedTuple):
    """Result of :func:`sort_tokens`; ``scale`` is None where there were no scales."""
    rows: torch.Tensor
    scale: Optional[torch.Tensor]
    offsets: torch.Tensor
    row_of_slot: torch.Tensor


def sort_tokens(x: torch.Tensor, topk_ids: torch.Tensor, num_experts: int, x_scale: Optional[torch.Tensor] = None) -> SortedTokens:
    """The tokens of all routing slots, sorted by expert: what a product with each expert's weights reads.

    x ``[M, K]`` bf16, fp32 or float8_e4m3fn codes (K a multiple of 128) with or without ``x_scale [M, K/128]`` float32; topk_ids
    ``[M, top_k]`` int32, top_k at most 64, at most 4096 experts, M below 2^24 - 1, rows of at most 2^27 bytes.
    Returns ``rows [M * top_k, K]``: x's row of every slot by ascending expert, equal experts by ascending slot, and behind them
    a row of zeros for each slot whose id is outside ``[0, num_experts)`` (a padded batch, experts of another GPU); ``scale`` in
    the same order; ``offsets [num_experts + 1]`` int32, the first row of each expert, the last one the number of slots that
    have one; ``row_of_slot [M, top_k]`` int32, the slot's row r, or ``~r`` (negative) where that is one of the zeros. Nothing
    of it depends on anything but the inputs.

    Differentiable in x where there is no x_scale: a token's gradient is its slots' sum, in fp32, rounded once; what the rows of
    zeros are given counts for nothing.
    """
    if x_scale is None:
        rows, offsets, row_of_slot = _sort_tokens(x, topk_ids, num_experts)
        return SortedTokens(rows, None, offsets, row_of_slot)
    return SortedTokens(*_sort_tokens_scaled(x, x_scale, topk_ids, num_experts))


def combine_tokens(rows: torch.Tensor, row_of_slot: torch.Tensor, topk_weights: Optional[torch.Tensor] = None,
                   scaling_factor: float = 1.0) -> torch.Tensor:
    """``out[t] = scaling_factor * sum over s of topk_weights[t, s] * rows[row_of_slot[t, s]]``, the way back from :func:`sort_tokens`.

    rows ``[M * top_k, K]`` bf16 or fp32, row_of_slot as :func:`sort_tokens` returns it, topk_weights ``[M, top_k]`` float32 or None (all 1).
    Summed in fp32 by ascending s and rounded once, to rows' dtype.  Slots with a negative entry take no part, whatever their row and
    weight hold; a token without any others is 0.

    Differentiable in rows and topk_weights.  (row_of_slot names every row once; if it does not, sums are as written above, and
    gradients of rows that it names twice or not at all are undefined.)
    """
    return _combine_tokens(rows, row_of_slot, topk_weights, scaling_factor)


def grouped_block_scaled_mm(x: torch.Tensor, x_scale: torch.Tensor, offsets: torch.Tensor, w: torch.Tensor,
                            w_scale: torch.Tensor) -> torch.Tensor:
    """The product of :func:`block_scaled_mm` for tokens sorted by expert: ``out[r] = (x[r] * x_scale[r]) (w[e] * w_scale[e])^T`` for the rows
    ``offsets[e] <= r < offsets[e + 1]``, rounded once to bfloat16.

    x ``[R, K]`` float8_e4m3fn, x_scale ``[R, K/128]`` and offsets ``[E + 1]`` int32 as :func:`sort_tokens` returns them (ascending, from 0
    on; rows behind the last become 0; with other offsets rows may be wrong or not written, and nothing beside them is touched);
    w ``[E, N, K]`` float8_e4m3fn in checkpoint order, w_scale ``[E, ceil(N/128), K/128]``. N is of any size, K a multiple of
    128 up to 65536, E at most 4096. Bit for bit the same from run to run.
    """
    return _grouped_block_scaled_mm(x, x_scale, offsets, w, w_scale)


def add_adapters(base: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, adapter_ids: torch.Tensor,
                 scale: Optional[torch.Tensor] = None, x_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Low-rank adapters of many requests beside a shared projection: ``base[m] + scale[l] * (x[m] a[l]^T) b[l]^T`` with
    ``l = adapter_ids[m]``; ``base[m]`` where l is outside ``[0, L)``.  A new tensor like base.

    base ``[M, N]`` bf16 is the projection's result (of :func:`block_scaled_mm`, say), x ``[M, K]`` its input: bf16, or float8_e4m3fn codes
    with ``x_scale [M, K/128]`` float32.  a ``[L, rank, K]`` and b ``[L, N, rank]`` bf16 (adapters of smaller rank padded with zeros),
    scale ``[L]`` float32 or None (all 1), adapter_ids ``[M]`` int32 in any order (neighbours of one adapter share its reading).  K a multiple of
    128 up to 65536, N at most 2^24, rank a multiple of 8 up to 128, M at most 1048560.

    Sums and the ``rank`` values between the two products are fp32, sums in an order that depends on the sizes alone; one rounding at
    the end.  Another request's adapter or activations, whatever they hold, change nothing of a token's result.
    What an infinity in b meets is infinite or NaN.
    """
    return _add_adapters(base, x, x_scale, a, b, adapter_ids, scale)
