"""Rows on which the router and the norm can lose what their definitions keep: choices that only 64 bits tell apart behind a long sum,
scores below fp32's normal numbers, infinities, and a row beside lost ones.  Against the float64 oracle, as in test_gpu_layer.py."""
import math

import pytest
import torch

from oracle import layer_oracle as L
from test_gpu_layer import DEV, NORM, U, activations, assert_codes, assert_route, assert_within, half_step

pytestmark = pytest.mark.gpu


# ---- a softmax's sum over many experts ---------------------------------------------------------------------
@pytest.mark.parametrize("E,small,second", [(4096, 63, 100), (2048, 63, 2047), (1025, 63, 1024), (1500, 63, 64), (1024, 15, 100),
                                            (512, 7, 8), (256, 3, 255)])
@pytest.mark.parametrize("gap", [2, 10, 40, 59, 60, 62])
def test_softmax_with_a_bias_of_one_loud_expert_and_many_faint_ones(E, small, second, gap):
    """One score near 1 and, behind it in the same lane, scores of 0.999 * 2^-24, each of which a sum near 1 may drop when they are
    added one by one; a second expert's bias is `gap` * 2^-24 behind the first one's score as such a sum has it."""
    print(f"case loud softmax E={E} small={small} second={second} gap={gap}", flush=True)
    logits = torch.full((1, E), -math.inf)
    logits[0, 0] = 0.0
    logits[0, 1:small + 1] = math.log(0.999 * U)
    bias = torch.full((E,), -0.6)
    bias[0], bias[second] = -0.5, 0.5 - gap * U
    for top_k in (1, 2, 8):
        assert_route(logits, top_k, bias=bias)
        assert_route(logits, top_k, bias=bias, renormalize=False)
        for groups in (4, 8):
            if E % groups == 0:
                assert_route(logits, top_k, bias=bias, num_groups=groups, top_groups=2)


# ---- scores below fp32's normal numbers --------------------------------------------------------------------
def assert_far_route(logits, top_k, **kw):
    """As assert_route, for weights far from 1.  A weight w is exp of some |x| <= -ln w below the largest chosen logit: the
    subtraction is off by |x| u in the exponent, x log2(e) by 1.25 |x| u, the exponential 2 u; the sum of at most 64 of them by
    its terms' errors, weighted, (2.25 ln 64 + 2) u < 12 u, and 6 additions; the division u: (2.25 |ln w| + 21) u, and 8 u for
    the factor 1 + exp(l) that scores below 2^-24 leave out.  A score below 2^-126 may be 0 where the chosen ones' sum is not below 2^-24."""
    from alpha_moe_python import layer_hip
    dev = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    w, ids = layer_hip.route_topk(logits.to(DEV), top_k, **dev)
    want, want_ids = L.route_topk(logits, top_k, **kw)
    assert torch.equal(ids.cpu().long(), want_ids)
    rel = (2.25 * want.clamp_min(2.0 ** -126).log().abs() + 32) * U
    assert_within(w, want, rel * want + 2.0 ** -102, "weights")
    return w


FAR = [[-99.0] + [-100.0] * 15, [-88.0, -88.5, -89.0, -90.0] * 4, [-87.0, -88.0] + [-600.0] * 14, [-699.0 + i / 4 for i in range(16)],
       [-17.0, -30.0, -60.0, -120.0] * 4, [-16.0, -16.5, -17.5, -18.0] * 4, [-650.0] + [-720.0] * 15, [-300.0] * 16,
       [-103.0, -math.inf] * 8, [-200.0 + 13 * i for i in range(16)], [-15.0, -95.0] * 8]


@pytest.mark.parametrize("E", [16, 64, 100, 256, 600, 1100, 4096])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("biased", [False, True])
def test_sigmoid_weights_of_far_logits_keep_their_ratio(E, dtype, biased):
    """every chosen logit below -88, where a sigmoid is no fp32 number any more; the weights' ratio is"""
    print(f"case far sigmoid E={E} {dtype} {biased}", flush=True)
    g = torch.Generator().manual_seed(E)
    logits = torch.full((len(FAR), E), -math.inf)
    for m, row in enumerate(FAR):
        logits[m, torch.randperm(E, generator=g)[:16]] = torch.tensor(row)
    logits = logits.to(dtype)
    bias = 0.1 * torch.randn(E, generator=g) if biased else None
    groups = dict(num_groups=4, top_groups=2) if E % 4 == 0 else {}
    for top_k in (1, 4, 8):
        assert_far_route(logits, top_k, scoring="sigmoid", bias=bias)
        assert_far_route(logits, top_k, scoring="sigmoid", bias=bias, shared_experts=1, shared_weight=0.4, **groups)
    if bias is None:
        w = assert_far_route(logits, 4, scoring="sigmoid")
        assert bool(((w.sum(1) - 1).abs() < 8 * U).all())


@pytest.mark.parametrize("E", [16, 64, 100, 256, 600, 1100, 4096])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_softmax_weights_of_experts_far_below_the_largest_keep_their_ratio(E, dtype):
    """a bias keeps the row's largest logit out: what is chosen lies further below it than fp32 reaches"""
    print(f"case far softmax E={E} {dtype}", flush=True)
    g = torch.Generator().manual_seed(E)
    logits = torch.full((len(FAR), E), -math.inf)
    bias = torch.full((E,), -2.0)
    for m, row in enumerate(FAR):
        at = torch.randperm(E - 1, generator=g)[:15] + 1
        logits[m, at] = torch.tensor(row[:15]) + 3.0
    logits[:, 0] = 3.0
    logits = logits.to(dtype)
    bias[0] = -math.inf
    bias[1:] += torch.randperm(E - 1, generator=g) / E
    for top_k in (1, 4, 8):
        assert_far_route(logits, top_k, bias=bias)
        if E % 4 == 0:
            assert_far_route(logits, top_k, bias=bias, num_groups=4, top_groups=3)
    best = logits.float()[:, 1:].amax(1)             # the experts with the largest logits behind it, and nobody else
    for m in range(len(FAR)):
        one = torch.full((E,), -math.inf)
        which = (logits[m].float() == best[m]).nonzero().flatten()
        one[which] = 0.5
        assert_far_route(logits[m:m + 1], min(8, which.numel()), bias=one)


@pytest.mark.parametrize("E", [16, 256, 1100])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_scores_up_to_e_to_the_minus_700_are_equal(E, scoring):
    """a bias of zeros, so that the scores alone decide, in 64 bits: down to e^-700 the larger one is first, below the lower index"""
    logits = torch.full((3, E), -math.inf)
    logits[:, :16] = torch.tensor([-720.0, -701, -650, -699, -698, -710, -600, -705] * 2)
    logits[1] = logits[1].flip(0)
    if scoring == "softmax":
        logits[2, 8] = 0.0                           # (in the rows before, the largest is -600 itself)
    for top_k in (1, 8, 16):
        assert_far_route(logits, top_k, scoring=scoring, bias=torch.zeros(E))


# ---- infinities --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("E", [16, 64, 256, 1100])
@pytest.mark.parametrize("renormalize", [True, False])
def test_softmax_rows_with_an_infinite_logit_have_no_weights(E, renormalize):
    """infinity minus infinity: the row's weights are NaN, whichever experts a bias or the masked others make it visit"""
    from alpha_moe_python import layer_hip
    logits = torch.randn((4, E), generator=torch.Generator().manual_seed(E))
    logits[0, 2:] = -math.inf
    logits[0, 1] = math.inf
    logits[1, 5] = math.inf
    logits[2, 3:] = -math.inf
    bias = 0.1 * torch.randn(E, generator=torch.Generator().manual_seed(E + 1))
    for b in (None, bias.to(DEV)):
        for top_k in (1, 8):
            w, ids = layer_hip.route_topk(logits.to(DEV), top_k, bias=b, renormalize=renormalize, shared_experts=1, shared_weight=0.5)
            assert bool(w[:2, :top_k].isnan().all()) and bool(w[2:].isfinite().all()) and bool((w[:, top_k] == 0.5).all())
            ids = ids.cpu()
            assert bool(((ids[:, :top_k] >= 0) & (ids[:, :top_k] < E)).all()) and all(len(set(r.tolist())) == top_k + 1 for r in ids)


# ---- norm --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [512, 4224])
def test_norm_of_an_ordinary_row_beside_lost_ones(K, dtype):
    """a NaN in one group of the weight, and rows that hold NaN, infinities and values whose squares pass fp32: the other groups of an
    ordinary row are those of the whole row"""
    from alpha_moe_python import layer_hip
    x = activations(5, K, 3, dtype)
    x[0, 5], x[1, 200], x[3, 300] = float("nan"), float("inf"), 2.0 ** 100
    w = 1 + 0.3 * torch.randn(K, generator=torch.Generator().manual_seed(K))
    w[130] = float("nan")
    r = layer_hip.rms_norm_quant_fp8(x.to(DEV), w.to(DEV), keep_norm=True)
    plain = w.clone()
    plain[130] = 1.0                                 # (the row's length does not depend on the weight)
    rows, cols = [2, 4], [c for c in range(K) if not 128 <= c < 256]
    y, _ = L.rms_norm(x[rows], plain, 1e-6)
    assert_codes(r.q[rows][:, cols], r.scale[rows][:, [0] + list(range(2, K // 128))], y[:, cols], NORM)
    cols += [c for c in range(128, 256) if c != 130]
    assert_within(r.norm[rows][:, cols], y[:, cols], (half_step(dtype) + NORM) * y[:, cols].abs(), "norm")
    lost = r.q.float().cpu()[rows][:, 128:256]
    assert bool(lost.isnan().all()) and bool(r.scale.cpu()[rows][:, 1].isnan().all()) and bool(r.norm[rows][:, 130].isnan().all())
