"""The operators around the fused experts without a GPU: what the C ABI and the torch operators refuse, their fake
implementations, and the float64 oracle they are held to."""
import ctypes
import math

import pytest
import torch

import alpha_moe
import alpha_moe_ops  # noqa: F401  (fake implementations)
from alpha_moe_python import layer_hip
from oracle import layer_oracle as L

OK, NULL, SHAPE, ALIGN = 0, 1, 2, 10
P, I, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_float


def c(name, argtypes, *args, restype=ctypes.c_int):
    fn = getattr(alpha_moe.c_abi, name)
    fn.restype, fn.argtypes = restype, argtypes
    return fn(*args)


def norm(x=4096, residual=None, weight=4096, q=4096, scale=4096, residual_out=None, norm_out=None, M=4, K=256):
    return c("alpha_moe_rms_norm_quant_fp8", [P, P, P, I, I, F, P, P, P, P, I, I, P], x, residual, weight, 0, 0, 1e-6, q, scale,
             residual_out, norm_out, M, K, None)


def test_norm_refusals():
    assert norm(M=0) == OK and norm(M=0, x=None) == OK          # nothing to do, nothing launched
    assert norm(M=-1) == SHAPE and norm(K=0) == SHAPE and norm(K=200) == SHAPE and norm(K=65536 + 128) == SHAPE
    assert norm(x=None) == NULL and norm(weight=None) == NULL and norm(q=None) == NULL and norm(scale=None) == NULL
    assert norm(residual=4096) == NULL and norm(residual_out=4096) == NULL    # both or neither
    for name in ("x", "weight", "q", "norm_out"):
        assert norm(**{name: 4096 + 8}) == ALIGN, name
    assert norm(residual=4100, residual_out=4096) == ALIGN and norm(residual=4096, residual_out=4100) == ALIGN


def test_swiglu_refusals():
    def call(x=4096, q=4096, scale=4096, M=4, width=256):
        return c("alpha_moe_swiglu_quant_fp8", [P, I, P, P, I, I, P], x, 0, q, scale, M, width, None)
    assert call(M=0) == OK and call(M=-1) == SHAPE and call(width=0) == SHAPE and call(width=192) == SHAPE
    assert call(x=None) == NULL and call(q=None) == NULL and call(scale=None) == NULL
    assert call(x=4104) == ALIGN and call(q=4104) == ALIGN


def test_mm_refusals():
    def call(x=4096, xs=4096, w=4096, ws=4096, out=4096, M=4, N=100, K=256):
        return c("alpha_moe_block_scaled_mm", [P, P, P, P, P, I, I, I, P], x, xs, w, ws, out, M, N, K, None)
    assert call(M=0) == OK and call(M=-1) == SHAPE and call(N=0) == SHAPE and call(K=0) == SHAPE and call(K=64) == SHAPE
    assert call(K=65536 + 128) == SHAPE
    for name in ("x", "xs", "w", "ws", "out"):
        assert call(**{name: None}) == NULL, name
    for name in ("x", "w", "out"):
        assert call(**{name: 4104}) == ALIGN, name
    assert call(M=2 ** 31 - 1) == SHAPE and call(N=2 ** 31 - 1) == SHAPE and call(M=2 ** 30, N=2 ** 30) == SHAPE


def test_route_refusals():
    def call(logits=4096, weights=4096, ids=4096, M=4, E=64, top_k=4, groups=1, top_groups=1, shared=0):
        return c("alpha_moe_route_topk", [P, I, P, P, P] + [I] * 8 + [F, P], logits, 1, None, weights, ids, M, E, top_k, 0, groups,
                 top_groups, 1, shared, 1.0, None)
    assert call(M=0) == OK and call(M=-1) == SHAPE and call(E=0) == SHAPE and call(E=4097) == SHAPE
    assert call(top_k=0) == SHAPE and call(top_k=65, E=128) == SHAPE and call(top_k=5, E=4) == SHAPE
    assert call(groups=0) == SHAPE and call(groups=3) == SHAPE and call(E=130, groups=65) == SHAPE
    assert call(groups=4, top_groups=5) == SHAPE and call(groups=4, top_groups=0) == SHAPE
    assert call(groups=32, top_groups=1, top_k=3) == SHAPE      # two experts a group
    assert call(shared=-1) == SHAPE
    assert call(logits=None) == NULL and call(weights=None) == NULL and call(ids=None) == NULL


def test_more_rows_than_a_launch_has_threads_for_are_refused():
    assert norm(M=2 ** 22) == SHAPE
    assert c("alpha_moe_route_topk", [P, I, P, P, P] + [I] * 8 + [F, P], 4096, 1, None, 4096, 4096, 2 ** 26, 8, 2, 0, 1, 1, 1, 0, 1.0, None) == SHAPE
    for M, N in ((1, 2 ** 31 - 300), (2 ** 31 - 300, 1), (2 ** 24, 2 ** 24), (8, 2 ** 30)):
        assert c("alpha_moe_block_scaled_mm", [P] * 5 + [I] * 3 + [P], 4096, 4096, 4096, 4096, 4096, M, N, 128, None) == SHAPE, (M, N)


def test_cpu_tensors_and_unknown_scoring_are_refused():
    x = torch.zeros((2, 128), dtype=torch.bfloat16)
    q, s = x.to(torch.float8_e4m3fn), torch.ones((2, 1))
    for call in (lambda: layer_hip.rms_norm_quant_fp8(x, x[0]), lambda: layer_hip.swiglu_quant_fp8(torch.zeros((2, 256))),
                 lambda: layer_hip.block_scaled_mm(q, s, q, s[:1]), lambda: layer_hip.route_topk(torch.zeros((2, 8)), 2)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
    with pytest.raises(ValueError):
        layer_hip.route_topk(torch.zeros((2, 8)), 2, scoring="tanh")


def test_fake_implementations_give_the_shapes():
    def meta(shape, dt):
        return torch.empty(shape, dtype=dt, device="meta")
    x = meta((3, 512), torch.bfloat16)
    r = layer_hip.rms_norm_quant_fp8(x, meta((512,), torch.float32), residual=x, keep_norm=True)
    assert r.q.shape == (3, 512) and r.q.dtype == torch.float8_e4m3fn and r.scale.shape == (3, 4)
    assert r.residual.shape == r.norm.shape == (3, 512) and r.norm.dtype == torch.bfloat16
    r = layer_hip.rms_norm_quant_fp8(x, meta((512,), torch.float32))
    assert r.residual is None and r.norm is None
    q, s = layer_hip.swiglu_quant_fp8(x)
    assert q.shape == (3, 256) and s.shape == (3, 2) and s.dtype == torch.float32
    out = layer_hip.block_scaled_mm(r.q, r.scale, meta((100, 512), torch.float8_e4m3fn), meta((1, 4), torch.float32))
    assert out.shape == (3, 100) and out.dtype == torch.bfloat16
    w, ids = layer_hip.route_topk(meta((3, 64), torch.bfloat16), 6, shared_experts=1)
    assert w.shape == ids.shape == (3, 7) and w.dtype == torch.float32 and ids.dtype == torch.int32


def inference_calls(make, grad):
    """``(what, call)`` of every operator, with one input at a time put through ``grad``."""
    x, w = make((3, 512), torch.bfloat16), make((512,), torch.float32)
    q, s = make((3, 512), torch.float8_e4m3fn), make((3, 4), torch.float32)
    mw, ms = make((100, 512), torch.float8_e4m3fn), make((1, 4), torch.float32)
    logits, bias = make((3, 64), torch.float32), make((64,), torch.float32)
    H = layer_hip
    for keep in (False, True):
        yield "x", lambda: H.rms_norm_quant_fp8(grad(x), w, keep_norm=keep)
        yield "weight", lambda: H.rms_norm_quant_fp8(x, grad(w), keep_norm=keep)
        yield "x", lambda: H.rms_norm_quant_fp8(grad(x), w, residual=x, keep_norm=keep)
        yield "residual", lambda: H.rms_norm_quant_fp8(x, w, residual=grad(x), keep_norm=keep)
        yield "weight", lambda: H.rms_norm_quant_fp8(x, grad(w), residual=x, keep_norm=keep)
    yield "gate_up", lambda: H.swiglu_quant_fp8(grad(x))
    yield "x_scale", lambda: H.block_scaled_mm(q, grad(s), mw, ms)
    yield "w_scale", lambda: H.block_scaled_mm(q, s, mw, grad(ms))
    yield "logits", lambda: H.route_topk(grad(logits), 4, bias=bias)
    yield "logits", lambda: H.route_topk(grad(logits), 4)
    yield "bias", lambda: H.route_topk(logits, 4, bias=grad(bias))


def on_meta(shape, dtype):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_inputs_that_require_gradients_are_refused_while_tracing_too():
    for name, call in inference_calls(on_meta, lambda t: t.detach().requires_grad_()):
        with pytest.raises(RuntimeError, match=f"{name} requires a gradient"):
            call()
        with torch.no_grad():
            call()
        with torch.inference_mode():
            call()
    for _, call in inference_calls(on_meta, lambda t: t):
        call()


def test_inputs_with_a_forward_mode_tangent_are_refused():
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        for name, call in inference_calls(on_meta, lambda t: fwd.make_dual(t, torch.empty_like(t))):
            with pytest.raises(RuntimeError, match=f"{name} carries a tangent"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):    # (which stops gradients, not tangents)
                call()
        for _, call in inference_calls(on_meta, lambda t: t):
            call()


def test_transformed_functions_are_refused():
    x, w = on_meta((3, 512), torch.float32), on_meta((512,), torch.float32)
    with pytest.raises(RuntimeError, match="weight carries a tangent"):
        torch.func.jvp(lambda v: layer_hip.rms_norm_quant_fp8(x, v).scale, (w,), (w,))
    with pytest.raises(RuntimeError, match="weight requires a gradient"):
        torch.func.grad(lambda v: layer_hip.rms_norm_quant_fp8(x, v).scale.sum())(w)
    with pytest.raises(RuntimeError, match="logits requires a gradient"):
        torch.func.vjp(lambda v: layer_hip.route_topk(v, 4)[0], x)


# ---- the oracle itself -------------------------------------------------------------------------------------
def test_oracle_norm_and_swiglu_by_hand():
    x = torch.zeros((1, 128))
    x[0, 0], x[0, 1] = 3.0, -4.0
    y, h = L.rms_norm(x, torch.full((128,), 2.0), 0.0)
    rms = 5.0 / math.sqrt(128.0)
    assert torch.allclose(y[0, :2], torch.tensor([6.0 / rms, -8.0 / rms], dtype=torch.float64))
    v, scale = L.group_scales(y)
    assert abs(scale.item() - 8.0 / rms / 448.0) < 1e-15 and v[0, 1].item() == -448.0
    g = torch.tensor([[0.0, 1.0, 2.0, 3.0]])
    assert torch.allclose(L.swiglu(g), torch.tensor([[0.0, 3.0 / (1.0 + math.exp(-1.0))]], dtype=torch.float64))


def test_oracle_mm_puts_scales_on_their_blocks():
    x, w = torch.ones((2, 256)), torch.ones((130, 256))
    xs = torch.tensor([[1.0, 2.0], [4.0, 8.0]])
    ws = torch.tensor([[1.0, 0.5], [16.0, 32.0]])
    out, size, dropped = L.block_scaled_mm(x, xs, w, ws)
    assert out[0, 0] == 128 * (1 + 1) and out[1, 127] == 128 * (4 + 4) and out[0, 128] == 128 * (16 + 64) and torch.equal(out, size)
    assert torch.allclose(dropped, 7 * 2.0 ** -13 * out / 8)


def test_oracle_route_by_hand():
    l = torch.tensor([[0.0, 2.0, 2.0, -1.0, 1.0, 1.0]])
    w, ids = L.route_topk(l, 3)
    assert ids.tolist() == [[1, 2, 4]]                 # ties to the lowest index
    e = [math.exp(2), math.exp(2), math.exp(1)]
    assert torch.allclose(w, torch.tensor([[v / sum(e) for v in e]], dtype=torch.float64))
    # with a bias: chosen by score + bias, weighted by score; groups by their two best
    w, ids = L.route_topk(l, 2, scoring="sigmoid", bias=torch.tensor([0.9, 0, 0, 0, 0, 0.0]), num_groups=3, top_groups=1,
                          shared_experts=1, shared_weight=0.5)
    assert ids.tolist() == [[0, 1, 6]] and abs(w.sum().item() - 1.5) < 1e-12
    w, ids = L.route_topk(torch.full((1, 4), -math.inf), 2, shared_experts=1)
    assert ids.tolist() == [[0, 1, 4]] and w.tolist() == [[0.0, 0.0, 1.0]]
    w, ids = L.route_topk(torch.tensor([[math.nan, 1.0, 2.0]]), 2)
    assert ids.tolist() == [[2, 1]] and bool(w.isnan().all())
