"""Tokens sorted by expert and back without a GPU: what the C ABI refuses, the fake implementations with their gradients, and the
oracle by hand."""
import pytest
import torch

import alpha_moe
import alpha_moe_ops  # noqa: F401  (fake implementations)
from alpha_moe_python import layer_hip
from oracle import layer_oracle as L

OK, NULL, SHAPE, WORKSPACE, ALIGN = 0, 1, 2, 7, 10
A = alpha_moe.c_abi


def sort(x=4096, size=2, scale_in=None, ids=4096, rows=4096, scale=None, offsets=4096, row_of_slot=4096, M=4, K=8, top_k=2, E=8, ws=None, nws=0):
    return A.alpha_moe_sort_tokens(x, size, scale_in, ids, rows, scale, offsets, row_of_slot, M, K, top_k, E, ws, nws, None)


def test_sort_refusals():
    for kw in (dict(size=3), dict(size=8), dict(M=-1), dict(M=2 ** 24), dict(K=0), dict(top_k=0), dict(top_k=65), dict(E=0), dict(E=4097),
               dict(size=1, K=64), dict(K=2 ** 27),
               dict(size=2, scale_in=4096, scale=4096)):
        assert sort(**kw) == SHAPE, kw
    for name in ("x", "ids", "rows", "offsets", "row_of_slot"):
        assert sort(**{name: None}) == NULL, name
    assert sort(size=1, K=128, scale_in=4096) == NULL and sort(size=1, K=128, scale=4096) == NULL      # both or neither
    assert sort(x=4097) == ALIGN and sort(rows=4099) == ALIGN and sort(size=4, x=4098) == ALIGN and sort(size=1, K=128, x=4104) == ALIGN
    big = dict(M=40000, top_k=8, E=256)
    need = A.alpha_moe_sort_workspace_bytes(40000, 8, 256)
    assert need > 0 and sort(**big) == WORKSPACE and sort(**big, ws=4096, nws=need - 1) == WORKSPACE and sort(**big, nws=need) == WORKSPACE
    assert A.alpha_moe_sort_workspace_bytes(8, 8, 256) == 0 and A.alpha_moe_sort_workspace_bytes(-1, 8, 8) == 0
    assert A.alpha_moe_sort_workspace_bytes(40000, 8, 0) == 0 and A.alpha_moe_sort_workspace_bytes(40000, 65, 8) == 0


def test_combine_refusals():
    def call(rows=4096, at=4096, weights=4096, out=4096, M=4, K=8, top_k=2):
        return A.alpha_moe_combine_tokens(rows, 0, at, weights, out, M, K, top_k, 1.0, None)
    assert call(M=0) == OK and call(M=-1) == SHAPE and call(K=0) == SHAPE and call(top_k=0) == SHAPE and call(top_k=65) == SHAPE
    assert call(M=2 ** 24) == SHAPE and call(K=2 ** 26 + 1) == SHAPE
    assert call(rows=None) == NULL and call(at=None) == NULL and call(out=None) == NULL
    assert call(rows=4097) == ALIGN and call(out=4103) == ALIGN

    def grad(g=4096, rows=4096, at=4096, weights=4096, grad_rows=4096, grad_weights=4096, M=4, K=8, top_k=2):
        return A.alpha_moe_combine_tokens_grad(g, rows, 0, at, weights, grad_rows, grad_weights, M, K, top_k, 1.0, None)
    assert grad(M=0) == OK and grad(grad_rows=None, grad_weights=None) == OK
    assert grad(M=-1) == SHAPE and grad(K=0) == SHAPE and grad(top_k=65) == SHAPE
    assert grad(g=None) == NULL and grad(at=None) == NULL and grad(rows=None) == NULL
    for name in ("g", "rows", "grad_rows"):
        assert grad(**{name: 4097}) == ALIGN, name


def meta(shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_fake_implementations_and_their_gradients():
    ids = meta((3, 2), torch.int32)
    s = layer_hip.sort_tokens(meta((3, 256), torch.float8_e4m3fn), ids, 9, x_scale=meta((3, 2)))
    assert s.rows.shape == (6, 256) and s.rows.dtype == torch.float8_e4m3fn and s.scale.shape == (6, 2)
    assert s.offsets.shape == (10,) and s.row_of_slot.shape == (3, 2) and s.offsets.dtype == s.row_of_slot.dtype == torch.int32
    x, w = meta((3, 7), torch.bfloat16).requires_grad_(), meta((3, 2)).requires_grad_()
    s = layer_hip.sort_tokens(x, ids, 9)
    assert s.scale is None and s.rows.requires_grad and not s.offsets.requires_grad and not s.row_of_slot.requires_grad
    out = layer_hip.combine_tokens(s.rows, s.row_of_slot, w, 2.0)
    assert out.shape == (3, 7) and out.dtype == torch.bfloat16
    gx, gw = torch.autograd.grad(out, (x, w), meta((3, 7), torch.bfloat16))
    assert gx.shape == (3, 7) and gx.dtype == torch.bfloat16 and gw.shape == (3, 2) and gw.dtype == torch.float32
    with torch.no_grad():
        assert not layer_hip.combine_tokens(layer_hip.sort_tokens(x, ids, 9).rows, s.row_of_slot, w).requires_grad


def test_derivatives_that_do_not_exist_are_refused():
    import torch.autograd.forward_ad as fwd
    ids, at = meta((3, 2), torch.int32), meta((3, 2), torch.int32)
    x, rows, w = meta((3, 8)), meta((6, 8)), meta((3, 2))
    codes, scale = meta((3, 128), torch.float8_e4m3fn), meta((3, 1))
    with pytest.raises(RuntimeError, match="x requires a gradient"):
        layer_hip.sort_tokens(codes.detach().requires_grad_(), ids, 4)
    with pytest.raises(RuntimeError, match="x_scale requires a gradient"):
        layer_hip.sort_tokens(codes, ids, 4, x_scale=scale.detach().requires_grad_())
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.empty_like(t))
        for call, name in ((lambda: layer_hip.sort_tokens(dual(x), ids, 4), "x"),
                           (lambda: layer_hip.combine_tokens(dual(rows), at, w), "rows"),
                           (lambda: layer_hip.combine_tokens(rows, at, dual(w)), "topk_weights")):
            with pytest.raises(RuntimeError, match=f"{name} carries a tangent"):
                call()
    r, v = rows.detach().requires_grad_(), w.detach().requires_grad_()
    out = layer_hip.combine_tokens(r, at, v)
    with pytest.raises(RuntimeError, match="requires a gradient"):
        torch.autograd.grad(out, (r, v), meta((3, 8)).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: layer_hip.combine_tokens(t, at, w).sum())(rows)


def test_cpu_tensors_are_refused():
    x, ids = torch.zeros((2, 8)), torch.zeros((2, 2), dtype=torch.int32)
    for call in (lambda: layer_hip.sort_tokens(x, ids, 4), lambda: layer_hip.combine_tokens(torch.zeros((4, 8)), ids)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


def test_oracle_by_hand():
    ids = torch.tensor([[2, 0], [-1, 2], [0, 3]], dtype=torch.int32)
    slots, offsets, at = L.sort_slots(ids, 3)
    assert slots.tolist() == [1, 4, 0, 3, 2, 5] and offsets.tolist() == [0, 2, 2, 4] and at.tolist() == [[2, 0], [~4, 3], [1, ~5]]
    rows = torch.arange(1.0, 7.0)[:, None]
    w = torch.tensor([[1.0, 2.0], [float("nan"), 3.0], [4.0, float("nan")]])
    out, size = L.combine_tokens(rows, at, w, 2.0)
    assert out.flatten().tolist() == [10.0, 24.0, 16.0] == size.flatten().tolist()
    gr, gw, _ = L.combine_tokens_grad(torch.tensor([[1.0], [-1.0], [0.5]]), rows, at, w, 2.0)
    assert gr.flatten().tolist() == [4.0, 4.0, 2.0, -6.0, 0.0, 0.0] and gw.tolist() == [[6.0, 2.0], [0.0, -8.0], [2.0, 0.0]]


def test_grouped_refusals_and_shapes():
    def call(x=4096, xs=4096, off=4096, w=4096, ws=4096, out=4096, M=4, N=100, K=256, E=8):
        return A.alpha_moe_grouped_block_scaled_mm(x, xs, off, w, ws, out, M, N, K, E, None)
    assert call(M=0) == OK and call(M=-1) == SHAPE and call(N=0) == SHAPE and call(K=0) == SHAPE and call(K=64) == SHAPE
    assert call(K=65536 + 128) == SHAPE and call(E=0) == SHAPE and call(E=4097) == SHAPE
    for name in ("x", "xs", "off", "w", "ws", "out"):
        assert call(**{name: None}) == NULL, name
    for name in ("x", "w", "out"):
        assert call(**{name: 4104}) == ALIGN, name
    for M, N, E in ((2 ** 31 - 1, 8, 8), (8, 2 ** 31 - 1, 8), (2 ** 30, 2 ** 30, 4096), (2 ** 31 - 300, 40, 1), (8, 2 ** 31 - 300, 8)):
        assert call(M=M, N=N, E=E) == SHAPE, (M, N, E)
    x, xs = meta((6, 256), torch.float8_e4m3fn), meta((6, 2))
    out = layer_hip.grouped_block_scaled_mm(x, xs, meta((5,), torch.int32), meta((4, 100, 256), torch.float8_e4m3fn), meta((4, 1, 2)))
    assert out.shape == (6, 100) and out.dtype == torch.bfloat16
    with pytest.raises(RuntimeError, match="x_scale requires a gradient"):
        layer_hip.grouped_block_scaled_mm(x, xs.requires_grad_(), meta((5,), torch.int32), meta((4, 100, 256), torch.float8_e4m3fn), meta((4, 1, 2)))


def test_adapter_refusals_and_shapes():
    def call(base=4096, x=4096, xs=None, a=4096, b=4096, ids=4096, scale=None, out=4096, M=4, N=100, K=256, rank=16, L=8, ws=4096, nws=1 << 40):
        return A.alpha_moe_add_adapters(base, x, xs, a, b, ids, scale, out, M, N, K, rank, L, ws, nws, None)
    assert call(M=0) == OK and call(M=-1) == SHAPE and call(N=0) == SHAPE and call(K=0) == SHAPE and call(K=64) == SHAPE
    assert call(K=65536 + 128) == SHAPE and call(L=0) == SHAPE and call(M=1048561) == SHAPE and call(N=2 ** 31 - 1) == SHAPE
    assert call(N=2 ** 24 + 1) == SHAPE and call(M=1048560, N=2 ** 24) == SHAPE       # (more threads than a launch has)
    for rank in (0, -8, 4, 12, 136):
        assert call(rank=rank) == SHAPE, rank
    for name in ("base", "x", "a", "b", "ids", "out"):
        assert call(**{name: None}) == NULL, name
    for name in ("base", "x", "a", "b", "out"):
        assert call(**{name: 4104}) == ALIGN, name
    need = A.alpha_moe_adapters_workspace_bytes(4, 100, 256, 16, 8)
    assert need >= 4 * 16 * 4 and call(ws=None) == WORKSPACE and call(ws=4104) == WORKSPACE and call(nws=need - 1) == WORKSPACE
    assert A.alpha_moe_adapters_workspace_bytes(0, 100, 256, 16, 8) == 0 and A.alpha_moe_adapters_workspace_bytes(4, 100, 256, 15, 8) == 0
    base, x, ids = meta((6, 100), torch.bfloat16), meta((6, 256), torch.bfloat16), meta((6,), torch.int32)
    a, b = meta((3, 16, 256), torch.bfloat16), meta((3, 100, 16), torch.bfloat16)
    out = layer_hip.add_adapters(base, x, a, b, ids, scale=meta((3,)))
    assert out.shape == (6, 100) and out.dtype == torch.bfloat16
    for i, name in enumerate(("base", "x", "a", "b")):
        args = [base, x, a, b]
        args[i] = args[i].detach().requires_grad_()
        with pytest.raises(RuntimeError, match=f"{name} requires a gradient"):
            layer_hip.add_adapters(*args, ids)


def test_oracle_of_adapters_by_hand():
    base, x = torch.ones((3, 2)), torch.zeros((3, 128))
    x[:, 0] = torch.tensor([1.0, 2.0, -3.0])
    a, b = torch.zeros((2, 8, 128)), torch.zeros((2, 2, 8))
    a[0, 0, 0], a[1, 3, 0] = 2.0, 1.0
    b[0, :, 0], b[1, :, 3] = torch.tensor([1.0, -1.0]), torch.tensor([0.5, 4.0])
    out, inner, outer = L.add_adapters(base, x, a, b, torch.tensor([0, 5, 1]), torch.tensor([10.0, -1.0]))
    assert out.tolist() == [[21.0, -19.0], [1.0, 1.0], [2.5, 13.0]]
    assert inner.tolist() == [[20.0, 20.0], [0.0, 0.0], [1.5, 12.0]] == outer.tolist()


@pytest.mark.parametrize("factor,applied", [(None, 1.0), (1.0, 1.0), (2.5, 2.5), (0.0, 0.0), (-1.0, -1.0)])
def test_expert_layer_applies_the_factor_it_is_given(factor, applied, monkeypatch):
    """a factor of 0 is one, too"""
    from alpha_moe_python.sglang_glue import norm_sorted_moe
    seen, combine = [], layer_hip.combine_tokens
    monkeypatch.setattr(layer_hip, "combine_tokens", lambda rows, at, w, c: seen.append(c) or combine(rows, at, w, c))
    M, K, I, E, f8, bf = 3, 256, 128, 4, torch.float8_e4m3fn, torch.bfloat16
    out, residual = norm_sorted_moe(meta((M, K), bf), meta((M, K), bf), meta((K,), bf), meta((E, K), bf), meta((E, 2 * I, K), f8),
                                    meta((E, K, I), f8), meta((E, 2, 2)), meta((E, 2, 1)), 2, routed_scaling_factor=factor)
    assert out.shape == residual.shape == (M, K) and seen == [applied]


def test_every_kernel_of_the_adapters_has_a_case():
    """the cases of the test on the GPU are of the tiles that they name; each kind of rank, tile and codes is among them"""
    from test_gpu_adapters import TILES, plan_of
    first, second, runs = set(), set(), set()
    for tiles, M, N, K, rank, adapters, fp8 in TILES:
        assert plan_of(M, N, K, rank, adapters) == tiles
        kind = 16 if rank <= 16 else 32 if rank <= 32 else 64 if rank <= 64 else 128
        first.add((tiles[0], min(kind, 64 if tiles[0] == 64 else 32), fp8))          # (of more ranks, workgroups take a part)
        second.add((tiles[1], kind))
        runs.add((tiles[1], tiles[2]))
    assert first == {(t, k, f) for t, ks in ((16, (16, 32)), (64, (16, 32, 64))) for k in ks for f in (False, True)}
    assert second == {(16, 16), (16, 32), (16, 64), (16, 128), (64, 16), (64, 32), (64, 64), (32, 128)}
    assert runs == {(16, 1), (64, 1), (64, 2), (64, 3), (64, 4), (32, 1), (32, 2), (32, 4)}


def test_every_tile_of_the_grouped_product_has_a_case():
    """the cases of the test on the GPU are of the tiles that they name, and leave none out"""
    import ctypes
    from test_gpu_grouped import TILES
    plan = (ctypes.c_int * 2)()
    for tile, counts, tail, N, K in TILES:
        assert A.alpha_moe_grouped_mm_plan(sum(counts) + tail, N, K, len(counts), plan) == OK and tuple(plan) == tile, (tile, N, K, tuple(plan))
    reached = set()
    for M in (1, 8, 61, 300, 1000, 3000, 10000, 70000):
        for E in (1, 8, 60, 256, 700):
            for N in (17, 512, 2049, 7168):
                for K in (128, 640, 1024, 2048, 7168):
                    assert A.alpha_moe_grouped_mm_plan(M, N, K, E, plan) == OK
                    reached.add(tuple(plan))
    assert reached == {t[0] for t in TILES}
    for M, N, K, E in ((0, 8, 128, 1), (8, 8, 64, 1), (8, 8, 128, 4097), (8, 0, 128, 1)):
        assert A.alpha_moe_grouped_mm_plan(M, N, K, E, plan) == SHAPE
