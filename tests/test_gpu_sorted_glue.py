"""An expert layer on sorted tokens and a dense layer with adapters (sglang_glue.norm_sorted_moe, norm_dense_mlp): the operators run
together, eagerly and from a graph, equal to the operators called one by one bit for bit, each step held to the float64 oracle on its own
inputs; and the sorted path in training, with the products between the sort and the combination in torch."""
import pytest
import torch

from alpha_moe_python import layer_hip
from alpha_moe_python.prep import block_quant_fp8
from alpha_moe_python.sglang_glue import Adapters, norm_dense_mlp, norm_sorted_moe
from oracle import layer_oracle as L
from test_gpu_adapters import check as check_adapters
from test_gpu_grouped import check as check_grouped
from test_gpu_layer import DEV, NORM, U, assert_codes, assert_mm, assert_route, assert_within
from test_gpu_sort import check_sort

pytestmark = pytest.mark.gpu


def layer(E, K, I, gate_experts, seed):
    g = torch.Generator().manual_seed(seed)
    w13, s13 = block_quant_fp8(torch.randn((E, 2 * I, K), generator=g) * 0.05)
    w2, s2 = block_quant_fp8(torch.randn((E, K, I), generator=g) * 0.05)
    norm = (1 + 0.2 * torch.randn(K, generator=g)).to(torch.bfloat16)
    return norm, torch.randn((gate_experts, K), generator=g) * 0.05, w13, w2, s13, s2


@pytest.mark.parametrize("M,E,gate_experts,first,top_k,I,scaling", [
    (1, 16, 16, 0, 4, 256, 1.0), (7, 8, 32, 8, 6, 128, 2.5), (61, 24, 24, 0, 8, 384, 1.5), (300, 4, 16, 12, 3, 128, 1.0),
    (1000, 16, 16, 0, 2, 256, 2.5)])
def test_expert_layer_on_sorted_tokens(M, E, gate_experts, first, top_k, I, scaling):
    print(f"case sorted experts M={M} E={E} of {gate_experts} from {first} top_k={top_k}", flush=True)
    K = 512
    g = torch.Generator().manual_seed(M)
    hidden, residual = (torch.randn((M, K), generator=g).to(torch.bfloat16) for _ in range(2))
    norm, gate, w13, w2, s13, s2 = layer(E, K, I, gate_experts, M)
    args = [t.to(DEV) for t in (hidden, residual, norm, gate, w13, w2, s13, s2)]
    kw = dict(top_k=top_k, routed_scaling_factor=scaling, first_expert=first)
    out, total = norm_sorted_moe(*args, **kw)
    x = layer_hip.rms_norm_quant_fp8(args[0], args[2], 1e-6, residual=args[1], keep_norm=True)
    assert torch.equal(total, x.residual)
    assert_codes(x.q, x.scale, L.rms_norm(hidden, norm, 1e-6, residual)[0], NORM)
    logits = torch.nn.functional.linear(x.norm.float(), args[3])
    assert_route(logits.cpu(), top_k)
    weights, ids = layer_hip.route_topk(logits, top_k)
    ids = ids - first
    s = check_sort(x.q.cpu(), ids.cpu(), E, x.scale.cpu())
    gate_up = layer_hip.grouped_block_scaled_mm(s.rows, s.scale, s.offsets, args[4], args[6])
    check_grouped(s.rows.cpu(), s.scale.cpu(), s.offsets.cpu(), w13, s13, gate_up)
    q, scale = layer_hip.swiglu_quant_fp8(gate_up)
    assert_codes(q, scale, L.swiglu(gate_up.cpu()), (gate_up[:, :I].abs().max().item() + 16) * U)
    rows = layer_hip.grouped_block_scaled_mm(q, scale, s.offsets, args[5], args[7])
    check_grouped(q.cpu(), scale.cpu(), s.offsets.cpu(), w2, s2, rows)
    assert torch.equal(out, layer_hip.combine_tokens(rows, s.row_of_slot, weights, scaling))
    want, size = L.combine_tokens(rows.cpu(), s.row_of_slot.cpu(), weights.cpu(), scaling)
    assert_within(out, want, 2.0 ** -8 * want.abs() + (top_k + 2) * U * size, "combined")

    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        again = norm_sorted_moe(*args, **kw)
    for step in range(3):
        args[0].copy_(torch.randn((M, K), generator=g).to(torch.bfloat16))
        want = norm_sorted_moe(*args, **kw)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(again, want)), step


def test_parts_of_the_experts_add_up():
    """two GPUs' halves of the experts, one after the other: what each slot adds is added once"""
    M, K, I, E, top_k = 50, 512, 128, 12, 4
    norm, gate, w13, w2, s13, s2 = (t.to(DEV) for t in layer(E, K, I, E, 3))
    g = torch.Generator().manual_seed(4)
    hidden, residual = (torch.randn((M, K), generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    parts = [norm_sorted_moe(hidden, residual, norm, gate, w13[a:b].contiguous(), w2[a:b].contiguous(), s13[a:b].contiguous(),
                             s2[a:b].contiguous(), top_k, first_expert=a)[0].double() for a, b in ((0, 5), (5, 12))]
    whole, _ = norm_sorted_moe(hidden, residual, norm, gate, w13, w2, s13, s2, top_k)
    # each of the three is rounded to bf16 once; a row's own values do not depend on its neighbours, but its product's tile may differ
    size = sum(p.abs() for p in parts) + whole.double().abs()
    assert bool(((parts[0] + parts[1] - whole.double()).abs() <= 2.0 ** -6 * size + 1e-3 * size.max()).all())
    with pytest.raises(ValueError):
        norm_sorted_moe(hidden, residual, norm, gate, w13, w2, s13, s2, top_k, first_expert=1)


@pytest.mark.parametrize("M,rank,adapters", [(1, 16, 2), (33, 8, 20), (200, 64, 5), (1500, 16, 9), (2300, 24, 6)])
def test_dense_layer_with_adapters(M, rank, adapters):
    print(f"case dense with adapters M={M} rank={rank} of {adapters}", flush=True)
    K, I = 512, 384
    g = torch.Generator().manual_seed(M)
    hidden, residual = (torch.randn((M, K), generator=g).to(torch.bfloat16) for _ in range(2))
    norm = (1 + 0.2 * torch.randn(K, generator=g)).to(torch.bfloat16)
    w13, s13 = block_quant_fp8(torch.randn((2 * I, K), generator=g) * 0.1)
    w2, s2 = block_quant_fp8(torch.randn((K, I), generator=g) * 0.1)
    low = lambda *shape: (torch.randn(shape, generator=g) * 0.1).to(torch.bfloat16)
    ad = Adapters(low(adapters, rank, K), low(adapters, 2 * I, rank), low(adapters, rank, I), low(adapters, K, rank),
                  torch.randint(-1, adapters, (M,), generator=g, dtype=torch.int32), 0.5 + torch.rand(adapters, generator=g))
    args, on = [t.to(DEV) for t in (hidden, residual, norm, w13, w2, s13, s2)], Adapters(*(t.to(DEV) for t in ad))
    out, total = norm_dense_mlp(*args, adapters=on)
    x = layer_hip.rms_norm_quant_fp8(args[0], args[2], 1e-6, residual=args[1])
    assert torch.equal(total, x.residual)
    base = layer_hip.block_scaled_mm(x.q, x.scale, args[3], args[5])
    gate_up = layer_hip.add_adapters(base, x.q, on.a13, on.b13, on.ids, on.scale, x.scale)
    cpu = lambda t: t.cpu()
    check_adapters(dict(base=cpu(base), x=cpu(x.q), a=ad.a13, b=ad.b13, adapter_ids=ad.ids, scale=ad.scale, x_scale=cpu(x.scale)), gate_up)
    q, scale = layer_hip.swiglu_quant_fp8(gate_up)
    base = layer_hip.block_scaled_mm(q, scale, args[4], args[6])
    assert_mm(base, q.cpu(), scale.cpu(), w2, s2)
    check_adapters(dict(base=cpu(base), x=cpu(q), a=ad.a2, b=ad.b2, adapter_ids=ad.ids, scale=ad.scale, x_scale=cpu(scale)), out)
    assert torch.equal(out, layer_hip.add_adapters(base, q, on.a2, on.b2, on.ids, on.scale, scale))
    none = ad.ids < 0
    plain, _ = norm_dense_mlp(*args)
    assert torch.equal(out.cpu()[none], plain.cpu()[none])


def test_a_training_step_on_sorted_tokens():
    """sort, each expert's own products in torch, weighted sums: gradients of the tokens, of the router's weights and of the experts'
    weights against the same layer written slot by slot in float64"""
    M, K, E, top_k = 40, 48, 6, 3
    g = torch.Generator().manual_seed(1)
    x0, w0 = torch.randn((M, K), generator=g), torch.randn((E, K, K), generator=g) / K ** 0.5
    p0, c = torch.rand((M, top_k), generator=g), torch.randn((M, K), generator=g)
    ids = torch.randint(-1, E, (M, top_k), generator=g, dtype=torch.int32)
    x, w, p = (t.to(DEV).requires_grad_() for t in (x0, w0, p0))
    s = layer_hip.sort_tokens(x, ids.to(DEV), E)
    bounds = s.offsets.tolist()
    parts = [torch.tanh(s.rows[lo:hi] @ w[e]) for e, (lo, hi) in enumerate(zip(bounds, bounds[1:]))]
    rows = torch.cat(parts + [s.rows[bounds[-1]:] * float("nan")])               # (behind the last expert: anything)
    out = layer_hip.combine_tokens(rows, s.row_of_slot, p, 0.5)
    got = torch.autograd.grad((out * c.to(DEV)).sum(), (x, w, p))
    xd, wd, pd = (t.double().requires_grad_() for t in (x0, w0, p0))
    total = torch.zeros((), dtype=torch.float64)
    want_out = torch.zeros((M, K), dtype=torch.float64)
    for t in range(M):
        for j in range(top_k):
            e = int(ids[t, j])
            if e >= 0:
                y = torch.tanh(xd[t] @ wd[e]) * pd[t, j] * 0.5
                want_out[t] += y.detach()
                total = total + (y * c[t].double()).sum()
    want = torch.autograd.grad(total, (xd, wd, pd))
    # a tanh's argument is a sum of K products of fp32 numbers (K u of the sum over magnitudes, some 8 here), tanh a few u, and the
    # chain behind it some 3 K additions: 1e-4 of the largest value is ten times that
    assert_within(out, want_out, torch.full_like(want_out, 1e-4 * want_out.abs().max().item()), "output")
    for a, b, name in zip(got, want, ("tokens", "experts' weights", "router's weights")):
        assert_within(a, b, torch.full_like(b, 1e-4 * b.abs().max().item()), name)


def test_layers_without_tokens():
    """a batch of nothing: results of no rows, gradients of zeros"""
    K, I, E, top_k, L_ = 512, 128, 4, 2, 3
    norm, gate, w13, w2, s13, s2 = (t.to(DEV) for t in layer(E, K, I, E, 3))
    nothing = torch.empty((0, K), dtype=torch.bfloat16, device=DEV)
    for t in norm_sorted_moe(nothing, nothing, norm, gate, w13, w2, s13, s2, top_k):
        assert t.shape == (0, K) and t.dtype == torch.bfloat16
    low = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
    ad = Adapters(low(L_, 8, K), low(L_, 2 * I, 8), low(L_, 8, I), low(L_, K, 8), torch.empty(0, dtype=torch.int32, device=DEV))
    for t in norm_dense_mlp(nothing, nothing, norm, w13[0].contiguous(), w2[0].contiguous(), s13[0].contiguous(), s2[0].contiguous(), adapters=ad):
        assert t.shape == (0, K) and t.dtype == torch.bfloat16
    x = nothing.clone().requires_grad_()
    w = torch.empty((0, top_k), device=DEV, requires_grad=True)
    s = layer_hip.sort_tokens(x, torch.empty((0, top_k), dtype=torch.int32, device=DEV), E)
    assert s.offsets.tolist() == [0] * (E + 1)
    gx, gw = torch.autograd.grad(layer_hip.combine_tokens(s.rows, s.row_of_slot, w).sum(), (x, w))
    assert gx.shape == (0, K) and gw.shape == (0, top_k)


def test_more_experts_than_offsets_in_flight():
    """above 256 experts their offsets are looked through twice: every expert's rows, the last one's and those behind it"""
    E, K, N = 700, 128, 128
    g = torch.Generator().manual_seed(11)
    w, ws = block_quant_fp8(torch.randn((E, N, K), generator=g))
    for mean in (1, 40):
        ids = torch.randint(-1, E, (mean * E // 2, 2), generator=g, dtype=torch.int32)
        ids[0, 0] = E - 1
        x = torch.randn((ids.shape[0], K), generator=g).to(DEV)
        q = layer_hip.rms_norm_quant_fp8(x, torch.ones(K, device=DEV))
        s = layer_hip.sort_tokens(q.q, ids.to(DEV), E, x_scale=q.scale)
        out = layer_hip.grouped_block_scaled_mm(s.rows, s.scale, s.offsets, w.to(DEV), ws.to(DEV))
        check_grouped(s.rows.cpu(), s.scale.cpu(), s.offsets.cpu(), w, ws, out)
