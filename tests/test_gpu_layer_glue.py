"""The feed-forward halves of a decoder layer (sglang_glue.norm_moe, norm_dense_mlp): the operators around the fused experts
run together, eagerly and from a graph.  They equal the operators called one by one bit for bit, and each step is held to the
float64 oracle on the step's own inputs.  (From end to end no bar holds: where the bf16 product between two steps falls on the other
side of a rounding boundary, and the element is its group's largest, the group's scale moves by up to 2^-7 and all its 128 codes
may round anew.)"""
import json
import os

import pytest
import torch

from alpha_moe_python import layer_hip
from alpha_moe_python.prep import block_quant_fp8
from alpha_moe_python.sglang_glue import norm_dense_mlp, norm_moe
from alpha_moe_python.utils import interleave_tensor
from gpu_util import assert_parity_rows
from oracle import layer_oracle as L
from oracle import moe_oracle as O
from test_gpu_layer import NORM, U, assert_codes, assert_mm, assert_route

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("M,K,I", [(1, 512, 256), (7, 1024, 384), (64, 512, 768), (300, 1152, 256), (1000, 512, 1024)])
def test_dense_layer(M, K, I):
    print(f"case dense M={M} K={K} I={I}", flush=True)
    g = torch.Generator().manual_seed(M + K)
    hidden, residual = (torch.randn((M, K), generator=g).to(torch.bfloat16) for _ in range(2))
    norm = (1 + 0.2 * torch.randn(K, generator=g)).to(torch.bfloat16)
    w13, s13 = block_quant_fp8(torch.randn((2 * I, K), generator=g) * 0.1)
    w2, s2 = block_quant_fp8(torch.randn((K, I), generator=g) * 0.1)
    args = [t.to(DEV) for t in (hidden, residual, norm, w13, w2, s13, s2)]
    out, total = norm_dense_mlp(*args)
    x = layer_hip.rms_norm_quant_fp8(args[0], args[2], 1e-6, residual=args[1])
    assert torch.equal(total, x.residual)
    assert torch.equal(total.cpu(), (hidden.float() + residual.float()).to(torch.bfloat16))
    assert_codes(x.q, x.scale, L.rms_norm(hidden, norm, 1e-6, residual)[0], NORM)
    gu = layer_hip.block_scaled_mm(x.q, x.scale, args[3], args[5])
    assert_mm(gu, x.q.cpu(), x.scale.cpu(), w13, s13)
    q, s = layer_hip.swiglu_quant_fp8(gu)
    gate = gu.cpu()[:, :I].double().abs()
    assert_codes(q, s, L.swiglu(gu.cpu()), (gate.max().item() + 16) * U)
    assert_mm(out, q.cpu(), s.cpu(), w2, s2)
    assert torch.equal(out, layer_hip.block_scaled_mm(q, s, args[4], args[6]))

    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        again = norm_dense_mlp(*args)
    for step in range(3):
        args[0].copy_(torch.randn((M, K), generator=g).to(torch.bfloat16))
        want = norm_dense_mlp(*args)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(again, want)), step


@pytest.mark.parametrize("shared", [0, 1])
@pytest.mark.parametrize("M,E,top_k,kw", [
    (1, 16, 4, dict()), (5, 16, 4, dict(scoring="sigmoid", groups=(4, 2), bias=True)), (40, 32, 6, dict(scoring="sigmoid")),
    (300, 16, 2, dict(groups=(4, 2), renormalize=False))])
def test_expert_layer(M, E, top_k, kw, shared, tmp_path):
    print(f"case experts M={M} E={E} top_k={top_k} {kw} shared={shared}", flush=True)
    K, I, scaling = 512, 256, 2.5 if shared else 1.0
    g = torch.Generator().manual_seed(M + E)
    table = os.path.join(tmp_path, "table.json")
    with open(table, "w") as fh:
        json.dump({"1": {"block_m": 16, "block_n": 32, "warp_n": 8, "stages": 4},
                   "64": {"block_m": 16, "block_n": 64, "warp_n": 4, "stages": 3},
                   "512": {"block_m": 64, "block_n": 64, "warp_n": 4, "stages": 3}}, fh)
    hidden, residual = (torch.randn((M, K), generator=g).to(torch.bfloat16) for _ in range(2))
    norm = (1 + 0.2 * torch.randn(K, generator=g)).to(torch.bfloat16)
    gate = torch.randn((E, K), generator=g) * 0.05
    bias = 0.1 * torch.randn(E, generator=g) if kw.get("bias") else None
    w13, s13 = block_quant_fp8(torch.randn((E + shared, 2 * I, K), generator=g) * 0.05)
    w2, s2 = block_quant_fp8(torch.randn((E + shared, K, I), generator=g) * 0.05)
    w13, s13 = interleave_tensor(w13, 8), interleave_tensor(s13, 1)
    groups, top_groups = kw.get("groups", (1, 1))
    route = dict(scoring=kw.get("scoring", "softmax"), num_groups=groups, top_groups=top_groups,
                 renormalize=kw.get("renormalize", True))
    args = [t.to(DEV) for t in (hidden, residual, norm, gate, w13, w2, s13, s2)]

    def call():
        return norm_moe(*args, top_k, correction_bias=None if bias is None else bias.to(DEV), routed_scaling_factor=scaling,
                        config_path=table, **route)
    out, total = call()
    assert torch.equal(total.cpu(), (hidden.float() + residual.float()).to(torch.bfloat16))
    x = layer_hip.rms_norm_quant_fp8(args[0], args[2], 1e-6, residual=args[1], keep_norm=True)
    assert torch.equal(total, x.residual)
    assert_codes(x.q, x.scale, L.rms_norm(hidden, norm, 1e-6, residual)[0], NORM)
    logits = torch.nn.functional.linear(x.norm.float(), args[3])        # the gate: a library's product
    weights, ids = assert_route(logits.cpu(), top_k, bias=bias, shared_experts=shared, shared_weight=1.0 / scaling, **route)
    aligned = O.align_reference(ids.cpu(), 16, E + shared)
    refs = [O.fused_moe_oracle(x.q.cpu(), x.scale.cpu(), w13, s13, w2, s2, *aligned, weights.cpu(),
                               torch.zeros((M, K), dtype=torch.bfloat16), top_k + shared, 16, scaling, up_nudge=nudge)
            for nudge in (0.0, 1e-5, -1e-5)]
    assert_parity_rows(out, refs, "experts")
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(call(), (out, total)))


def expert_layer(M, tmp_path):
    K, I, E = 512, 256, 16
    table = os.path.join(tmp_path, "table.json")
    with open(table, "w") as fh:
        json.dump({"1": {"block_m": 16, "block_n": 32, "warp_n": 8, "stages": 4},
                   "512": {"block_m": 64, "block_n": 64, "warp_n": 4, "stages": 3}}, fh)
    g = torch.Generator().manual_seed(M)
    hidden, residual = (torch.randn((M, K), generator=g).to(torch.bfloat16) for _ in range(2))
    gate, bias = torch.randn((E, K), generator=g) * 0.05, (0.1 * torch.randn(E, generator=g)).to(torch.bfloat16)
    w13, s13 = block_quant_fp8(torch.randn((E + 1, 2 * I, K), generator=g) * 0.05)
    w2, s2 = block_quant_fp8(torch.randn((E + 1, K, I), generator=g) * 0.05)
    args = [t.to(DEV) for t in (hidden, residual, torch.ones(K), gate, interleave_tensor(w13, 8), w2, interleave_tensor(s13, 1), s2)]
    return g, args, bias.to(DEV), dict(scoring="sigmoid", num_groups=4, top_groups=2, config_path=table)


def test_expert_layer_with_a_bf16_bias_and_no_scaling(tmp_path):
    _, args, bias, kw = expert_layer(7, tmp_path)
    a = norm_moe(*args, 4, correction_bias=bias, routed_scaling_factor=None, **kw)
    b = norm_moe(*args, 4, correction_bias=bias.float(), routed_scaling_factor=1.0, **kw)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and bool(a[0].isfinite().all())


@pytest.mark.parametrize("M", [1, 20, 600])
def test_expert_layer_captured_and_replayed(M, tmp_path):
    print(f"case captured experts M={M}", flush=True)
    g, args, bias, kw = expert_layer(M, tmp_path)

    def call():
        return norm_moe(*args, 4, correction_bias=bias, routed_scaling_factor=2.5, **kw)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        call()                                  # the fused operator's scratch memory of this stream
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        again = call()
    for step in range(4):
        args[0].copy_(torch.randn(args[0].shape, generator=g).to(torch.bfloat16))
        want = call()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(again, want)), step


def test_no_tokens_and_refusals(tmp_path):
    table = os.path.join(tmp_path, "table.json")
    with open(table, "w") as fh:
        json.dump({"1": {"block_m": 16, "block_n": 32, "warp_n": 8, "stages": 4}}, fh)
    K, I, E = 256, 128, 4
    empty = torch.empty((0, K), dtype=torch.bfloat16, device=DEV)
    norm, gate = torch.ones(K, device=DEV), torch.ones((E, K), device=DEV)
    w13, s13 = (t.to(DEV) for t in block_quant_fp8(torch.ones((E, 2 * I, K))))
    w2, s2 = (t.to(DEV) for t in block_quant_fp8(torch.ones((E, K, I))))
    out, total = norm_moe(empty, empty, norm, gate, w13, w2, s13, s2, 2, config_path=table)
    assert out.shape == total.shape == (0, K)
    out, total = norm_dense_mlp(empty, empty, norm, w13[0], w2[0], s13[0], s2[0])
    assert out.shape == total.shape == (0, K)
    x = torch.ones((1, K), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):
        norm_moe(x, x, norm, torch.ones((E + 1, K), device=DEV), w13, w2, s13, s2, 2, config_path=table)
    with pytest.raises(RuntimeError):
        norm_dense_mlp(x, x.float(), norm, w13[0], w2[0], s13[0], s2[0])
    with pytest.raises(RuntimeError):
        norm_dense_mlp(x, x, norm, w13[0], w2[0], s13[0], s2[0][:, :0])
