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
