"""The HIP operators around the fused experts against their definitions in float64 (oracle/layer_oracle.py).

Tolerances.  u = 2^-24 is the most a fp32 operation is off, relatively; 2^-8 a rounding to bf16.
* norm: a sum of K squares taken in at most 128 + 32 additions one behind the other is at most 160 u off, its root half that; with
  the division, the root, the sum h and two products 100 u cover y: NORM.
* SwiGLU: exp(x) by any method that rounds x log2(e) once is (|x| + 8) u off, and every further step u: (|g| + 16) u.
* codes: e4m3 is half a step off, 2^-4 of the value or 2^-10 below its normal numbers, plus what y and the scale are off.
* product: at most K / 128 + 128 additions one behind the other, u of the sum over magnitudes each; the scales' products 2 u; a
  rounding to bf16; and what the matrix core drops of a sum of eight products (oracle.block_scaled_mm).
* router: 64 bits rounded to fp32 once, u; scores computed in fp32 are (|l - top| + 32) u off.  A score below fp32's normal numbers
  has no 24 bits to be right in: 2^-126 more.
"""
import pytest
import torch

from oracle import layer_oracle as L

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
NORM = 100 * U


def half_step(dtype):
    return 2.0 ** -8 if dtype == torch.bfloat16 else U


def assert_within(got, want, tol, what):
    """|got - want| <= tol, element for element; NaN exactly where want is."""
    got = got.detach().cpu().double()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    fine = want.isfinite()
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()]), f"{what}: infinities"
    off = ((got - want).abs() - tol)[fine]
    assert off.numel() == 0 or off.max() <= 0, f"{what}: {off.max().item():.3g} more than allowed"


def assert_codes(q, scale, y, rel):
    """q, scale are those of y [M, K] (float64), which the kernel has within rel."""
    v, s = L.group_scales(y)
    assert q.dtype == torch.float8_e4m3fn and scale.dtype == torch.float32
    assert_within(scale, s, (rel + 2 * U) * s.abs(), "scale")
    wide = v.clone()
    tol = torch.maximum(v.abs() * 2.0 ** -4, torch.full_like(v, 2.0 ** -10)) + (2 * rel + 8 * U) * v.abs()
    assert_within(q.float(), wide, tol, "codes")


def activations(M, K, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((M, K), generator=g) * (0.1 + 4 * torch.rand((M, 1), generator=g))
    x[:, torch.randint(0, K, (max(1, K // 300),), generator=g)] *= 30
    return x.to(dtype)


# ---- norm --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("residual,keep", [(False, False), (True, True), (True, False), (False, True)])
@pytest.mark.parametrize("M,K,dtype,wdtype", [
    (1, 128, torch.bfloat16, torch.bfloat16), (1, 7168, torch.bfloat16, torch.bfloat16), (3, 256, torch.float32, torch.float32),
    (5, 2048, torch.bfloat16, torch.float32), (2, 2048, torch.float32, torch.bfloat16), (67, 1152, torch.bfloat16, torch.bfloat16),
    (2, 8320, torch.bfloat16, torch.bfloat16), (2, 4224, torch.float32, torch.float32), (2, 16512, torch.bfloat16, torch.float32),
    (2, 65536, torch.bfloat16, torch.bfloat16), (2, 65536, torch.float32, torch.float32), (1030, 640, torch.bfloat16, torch.bfloat16)])
def test_norm(M, K, dtype, wdtype, residual, keep):
    from alpha_moe_python import layer_hip
    print(f"case norm M={M} K={K} {dtype} {wdtype} {residual} {keep}", flush=True)
    g = torch.Generator().manual_seed(K)
    x = activations(M, K, M + K, dtype)
    w = (1 + 0.3 * torch.randn(K, generator=g)).to(wdtype)
    res = activations(M, K, M + K + 1, dtype) if residual else None
    x[0, :128] = 0                                   # a group of zeros (without a residual)
    if residual and M > 1:
        res[1] = -x[1]                               # a row that cancels: y is 0 everywhere
    xd, rd = x.to(DEV), res.to(DEV) if residual else None
    r = layer_hip.rms_norm_quant_fp8(xd, w.to(DEV), 1e-6, residual=rd, keep_norm=keep)
    y, h = L.rms_norm(x, w, 1e-6, res)
    assert_codes(r.q, r.scale, y, NORM)
    assert (r.residual is not None) == residual and (r.norm is not None) == keep
    if residual:
        assert torch.equal(r.residual.cpu(), (x.float() + res.float()).to(dtype))
        assert torch.equal(rd.cpu(), res)            # the input stays
    if keep:
        assert_within(r.norm, y, (half_step(dtype) + NORM) * y.abs(), "norm")
    assert torch.equal(xd.cpu(), x)


def test_norm_of_rows_that_are_not_numbers():
    from alpha_moe_python import layer_hip
    x = activations(4, 512, 3, torch.bfloat16)
    x[0, 5] = float("nan")
    x[1, 200] = float("inf")
    x[2, 300] = 2.0 ** 100                           # its square is past fp32: the row's length is infinite
    w = torch.ones(512)
    w[130] = float("nan")
    r = layer_hip.rms_norm_quant_fp8(x.to(DEV), w.to(DEV), keep_norm=True)
    q, s, n = r.q.float().cpu(), r.scale.cpu(), r.norm.float().cpu()
    assert bool(q[0].isnan().all()) and bool(s[0].isnan().all()) and bool(n[0].isnan().all())
    assert bool(q[:, 128:256].isnan().all()) and bool(s[:, 1].isnan().all())     # the weight's group, in every row
    assert bool((n[1, 256:] == 0).all()) and bool((q[1, 256:] == 0).all())       # finite values over an infinite length
    assert bool((q[2, 256:] == 0).all()) and bool((s[2, 2:] == 1e-10 / 448).all())
    y, _ = L.rms_norm(x[3:, :128], w[:128], 1e-6)
    keep = torch.cat([x[3:, :128], x[3:, 256:]], 1)
    full, _ = L.rms_norm(keep, torch.ones(384), 1e-6)
    assert bool(q[3, :128].isfinite().all()) and bool(q[3, 256:].isfinite().all()) and full.shape == (1, 384) and y.shape == (1, 128)


def test_norm_in_place_and_nothing_beside_its_rows():
    """residual_out may be residual or x; bytes behind the last row stay as they were"""
    import alpha_moe
    fn = alpha_moe.c_abi.alpha_moe_rms_norm_quant_fp8
    import ctypes
    P, I = ctypes.c_void_p, ctypes.c_int
    fn.restype, fn.argtypes = I, [P, P, P, I, I, ctypes.c_float, P, P, P, P, I, I, P]
    M, K = 3, 384
    x, res, w = activations(M, K, 1, torch.bfloat16), activations(M, K, 2, torch.bfloat16), torch.ones(K)
    y, _ = L.rms_norm(x, w, 1e-6, res)
    total = (x.float() + res.float()).to(torch.bfloat16)
    for into in ("residual", "x"):
        bufs = {k: torch.cat([v.flatten(), torch.full((256,), 7.0, dtype=v.dtype)]).to(DEV) for k, v in (("x", x), ("residual", res))}
        q = torch.full((M * K + 256,), 0x55, dtype=torch.uint8, device=DEV)
        s = torch.full((M * K // 128 + 64,), 5.0, device=DEV)
        n = torch.full((M * K + 256,), 7.0, dtype=torch.bfloat16, device=DEV)
        wd = w.to(DEV)
        rc = fn(bufs["x"].data_ptr(), bufs["residual"].data_ptr(), wd.data_ptr(), 0, 1, 1e-6, q.data_ptr(), s.data_ptr(),
                bufs[into].data_ptr(), n.data_ptr(), M, K, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert rc == 0
        assert torch.equal(bufs[into][:M * K].cpu().view(M, K), total)
        assert_codes(q[:M * K].view(torch.float8_e4m3fn).view(M, K), s[:M * K // 128].view(M, -1), y, NORM)
        assert bool((q[M * K:] == 0x55).all()) and bool((s[M * K // 128:] == 5).all()) and bool((n[M * K:] == 7).all())
        assert bool((bufs[into][M * K:] == 7).all())


# ---- SwiGLU ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("M,I,dtype", [(1, 128, torch.bfloat16), (7, 768, torch.bfloat16), (3, 256, torch.float32),
                                       (33, 1408, torch.bfloat16), (257, 2048, torch.bfloat16), (129, 640, torch.float32)])
def test_swiglu(M, I, dtype):
    from alpha_moe_python import layer_hip
    print(f"case swiglu M={M} I={I} {dtype}", flush=True)
    x = activations(M, 2 * I, M + I).clamp(-80, 80).to(dtype)
    x[0, :64] = 0
    x[0, I + 128:] = 0
    q, s = layer_hip.swiglu_quant_fp8(x.to(DEV))
    y = L.swiglu(x)
    gate = x[:, :I].double().abs()
    # (an element's own error, and its group's largest element's in the scale)
    rel = (gate.reshape(M, -1, 128).amax(-1) + 16) * U
    assert_codes(q, s, y, rel.max().item())


def test_swiglu_far_gates_and_values_that_are_not_numbers():
    from alpha_moe_python import layer_hip
    x = torch.ones((4, 768), dtype=torch.float32)
    x[0, :384] = torch.linspace(-200, -100, 384)     # exp overflows: silu is -0
    x[1, :384] = torch.linspace(100, 3e38, 384)      # silu(g) = g
    x[2, 3] = float("nan")
    x[2, 384 + 130] = float("inf")                   # up: an infinity in its group
    x[2, 384 + 300] = float("nan")
    x[3, 5] = float("-inf")                          # -inf * 0
    q, s = layer_hip.swiglu_quant_fp8(x.to(DEV))
    q, s = q.float().cpu(), s.cpu()
    assert bool((q[0].abs() == 0).all()) and bool((s[0] == torch.tensor(1e-10) / 448).all())
    assert_codes(q[1:2].to(torch.float8_e4m3fn), s[1:2], x[1:2, :384].double(), 4 * U)
    assert bool(q[2, :128].isnan().all()) and bool(s[2, 0].isnan())
    assert s[2, 1].item() == float("inf") and bool(q[2, 130].isnan()) and bool((q[2, 131:256] == 0).all())
    assert bool(q[2, 256:].isnan().all())
    assert bool(q[3, :128].isnan().all()) and bool(q[3, 128:].isfinite().all())


# ---- block-scaled product ----------------------------------------------------------------------------------
def mm_problem(M, N, K, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((M, K), generator=g).mul_(60).clamp_(-448, 448).to(torch.float8_e4m3fn)
    w = torch.randn((N, K), generator=g).mul_(60).clamp_(-448, 448).to(torch.float8_e4m3fn)
    xs = torch.rand((M, K // 128), generator=g) * 0.02 + 1e-4
    ws = torch.rand(((N + 127) // 128, K // 128), generator=g) * 0.001 + 1e-6
    return x, xs, w, ws


def assert_mm(out, x, xs, w, ws):
    want, size, dropped = L.block_scaled_mm(x, xs, w, ws)
    K = x.shape[1]
    sums = (K // 128 + 130) * U * size + dropped
    assert_within(out, want, sums + 2.0 ** -8 * (want.abs() + sums), "product")


MM_SIZES = [(1, 1, 128), (1, 4096, 256), (2, 17, 384), (7, 129, 1152), (15, 130, 256), (16, 128, 512), (17, 100, 640), (31, 64, 2048),
            (32, 257, 128), (33, 576, 896), (61, 2112, 1024), (64, 256, 1280), (65, 192, 256), (100, 3, 384), (127, 1000, 512),
            (128, 512, 128), (129, 385, 256), (200, 640, 384), (255, 511, 256), (257, 769, 384), (300, 1030, 1024), (513, 260, 640),
            (5, 300, 65536), (70, 130, 16384), (9, 5000, 128), (30, 3300, 256), (60, 4200, 384), (350, 2200, 640), (200, 7300, 256),
            (520, 4100, 512), (1000, 7000, 256), (700, 4000, 640), (1030, 4097, 128), (2100, 4200, 256), (2050, 7200, 384),
            (4000, 4500, 128), (16400, 130, 256), (3, 40000, 256), (150, 300, 65536), (4090, 4091, 256)]


@pytest.mark.parametrize("M,N,K", MM_SIZES)
def test_mm(M, N, K):
    from alpha_moe_python import layer_hip
    print(f"case mm M={M} N={N} K={K}", flush=True)
    x, xs, w, ws = mm_problem(M, N, K, M * 7 + N + K)
    out = layer_hip.block_scaled_mm(x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV))
    assert out.dtype == torch.bfloat16 and out.shape == (M, N)
    assert_mm(out, x, xs, w, ws)


@pytest.mark.parametrize("M,N,K", [(1, 300, 1024), (19, 300, 1024), (61, 520, 2048), (130, 300, 1024), (400, 700, 640), (1100, 1300, 384),
                                   (260, 7200, 512), (600, 7100, 1024), (1500, 4100, 640), (4090, 4088, 512)])
def test_mm_puts_every_element_and_scale_in_its_place(M, N, K):
    """whole numbers and scales that are powers of two: fp32 holds every partial sum, so the product is exact up to its rounding to bf16"""
    from alpha_moe_python import layer_hip
    print(f"case mm exact M={M} N={N} K={K}", flush=True)
    g = torch.Generator().manual_seed(M + N + K)
    x = torch.randint(-2, 3, (M, K), generator=g).float().to(torch.float8_e4m3fn)
    w = torch.randint(-2, 3, (N, K), generator=g).float().to(torch.float8_e4m3fn)
    xs = 2.0 ** torch.randint(-1, 3, (M, K // 128), generator=g).float()
    ws = 2.0 ** torch.randint(-2, 2, ((N + 127) // 128, K // 128), generator=g).float()
    out = layer_hip.block_scaled_mm(x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV))
    want = L.block_scaled_mm(x, xs, w, ws)[0]
    assert torch.equal(want.float().double(), want) and torch.equal(out.cpu(), want.float().to(torch.bfloat16))


@pytest.mark.parametrize("M,N,K", [(1, 300, 2048), (61, 520, 2048), (200, 4200, 2048), (260, 7200, 1024), (700, 4100, 1024), (1500, 4100, 1024),
                                   (4090, 4088, 2048)])
def test_mm_with_scales_at_any_multiple_of_four_bytes(M, N, K):
    """how the tokens' scales are loaded depends on where they lie; which sums are made, and their order, does not"""
    from alpha_moe_python import layer_hip
    print(f"case mm scales M={M} N={N} K={K}", flush=True)
    x, xs, w, ws = [t.to(DEV) for t in mm_problem(M, N, K, M + N + K)]
    want = layer_hip.block_scaled_mm(x, xs, w, ws)
    for shift in (1, 2, 3):
        store = torch.full((xs.numel() + 8,), float("nan"), device=DEV)
        moved = store[shift:shift + xs.numel()].view_as(xs)
        moved.copy_(xs)
        assert moved.data_ptr() % 16 == 4 * shift
        assert torch.equal(layer_hip.block_scaled_mm(x, moved, w, ws), want)


@pytest.mark.parametrize("M", [1, 40, 300, 9000, 40000])
def test_mm_keeps_what_is_not_a_number(M):
    from alpha_moe_python import layer_hip
    x, xs, w, ws = mm_problem(M, 300, 512, M)
    x.view(torch.uint8)[M // 2, 100] = 0x7f          # NaN
    w.view(torch.uint8)[7, 200] = 0xff
    ws[1, 3] = float("inf")
    xs[0, 2] = float("nan")
    out = layer_hip.block_scaled_mm(x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV)).cpu()
    want, size, dropped = L.block_scaled_mm(x, xs, w, ws)
    assert bool(out[0].isnan().all()) and bool(out[M // 2].isnan().all()) and bool(out[:, 7].isnan().all())
    rest = torch.ones(M, dtype=torch.bool)
    rest[0] = rest[M // 2] = False
    cols = torch.cat([torch.arange(0, 7), torch.arange(8, 128), torch.arange(256, 300)])
    assert bool((~out[rest][:, 128:256].isfinite()).all())
    a, b, c = out[rest][:, cols].double(), want[rest][:, cols], (140 * U * size + dropped)[rest][:, cols]
    assert bool(((a - b).abs() <= c + 2.0 ** -8 * (b.abs() + c)).all())


@pytest.mark.parametrize("M,N", [(1, 130), (3, 64), (20, 100), (63, 33), (70, 130), (300, 260), (520, 4100), (1030, 4097), (2100, 4200), (2050, 7200), (4090, 4091)])
def test_mm_writes_its_rows_and_nothing_else(M, N):
    import ctypes
    import alpha_moe
    P, I = ctypes.c_void_p, ctypes.c_int
    fn = alpha_moe.c_abi.alpha_moe_block_scaled_mm
    fn.restype, fn.argtypes = I, [P, P, P, P, P, I, I, I, P]
    x, xs, w, ws = mm_problem(M, N, 640, M + N)
    dev = [t.to(DEV) for t in (x, xs, w, ws)]
    out = torch.full((M * N + 4096,), 7.0, dtype=torch.bfloat16, device=DEV)
    rc = fn(*[t.data_ptr() for t in dev], out.data_ptr(), M, N, 640,
            torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert rc == 0 and bool((out[M * N:] == 7).all())
    assert_mm(out[:M * N].view(M, N), x, xs, w, ws)


def test_mm_of_more_than_4_gib():
    """weights, activations and results whose offsets pass 32 bits"""
    from alpha_moe_python import layer_hip
    g = torch.Generator(device=DEV).manual_seed(1)

    def codes(n, k):
        t = torch.randint(0, 0x78, (n, k), generator=g, device=DEV, dtype=torch.uint8)
        return t.view(torch.float8_e4m3fn)
    for M, N, K in ((3, 66000, 65536), (66000, 5, 65536), (40000, 60000, 128)):
        print(f"case mm large M={M} N={N} K={K}", flush=True)
        x, w = codes(M, K), codes(N, K)
        xs = torch.rand((M, K // 128), generator=g, device=DEV)
        ws = torch.rand(((N + 127) // 128, K // 128), generator=g, device=DEV)
        out = layer_hip.block_scaled_mm(x, xs, w, ws)
        rows = torch.tensor(sorted({0, 1, M // 2, M - 2, M - 1}))
        cols = torch.tensor(sorted({0, 1, N // 2, N - 2, N - 1}))
        some_x = x.view(torch.uint8)[rows.to(DEV)].view(torch.float8_e4m3fn).cpu()
        for col in cols.tolist():
            want, size, dropped = L.block_scaled_mm(some_x, xs[rows.to(DEV)].cpu(), w[col:col + 1].cpu(), ws[col // 128:col // 128 + 1].cpu())
            got = out[:, col][rows.to(DEV)].cpu().double()
            sums = ((K // 128 + 130) * U * size + dropped)[:, 0]
            assert bool(((got - want[:, 0]).abs() <= sums + 2.0 ** -8 * (want[:, 0].abs() + sums)).all()), (M, N, K, col)
        del x, w, out


# ---- router ------------------------------------------------------------------------------------------------
def assert_route(logits, top_k, **kw):
    from alpha_moe_python import layer_hip
    dev = dict(kw)
    if kw.get("bias") is not None:
        dev["bias"] = kw["bias"].to(DEV)
    w, ids = layer_hip.route_topk(logits.to(DEV), top_k, **dev)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32
    want, want_ids = L.route_topk(logits, top_k, **kw)
    assert torch.equal(ids.cpu().long(), want_ids)
    assert_within(w, want, (64 + 32) * U * want.abs() + 2.0 ** -126, "weights")
    return w, ids


ROUTES = [dict(E=1, top_k=1), dict(E=8, top_k=8), dict(E=60, top_k=4), dict(E=64, top_k=6), dict(E=100, top_k=64), dict(E=128, top_k=8),
          dict(E=160, top_k=6, num_groups=8, top_groups=3), dict(E=256, top_k=8, num_groups=8, top_groups=4, shared_experts=1, shared_weight=0.4),
          dict(E=256, top_k=8, num_groups=64, top_groups=3), dict(E=64, top_k=3, num_groups=64, top_groups=3), dict(E=257, top_k=9),
          dict(E=512, top_k=10), dict(E=700, top_k=20, num_groups=7, top_groups=2), dict(E=1024, top_k=8, num_groups=16, top_groups=1),
          dict(E=4096, top_k=33, num_groups=4, top_groups=2, shared_experts=70), dict(E=1500, top_k=2),
          dict(E=4095, top_k=12, num_groups=5, top_groups=2), dict(E=4096, top_k=5, num_groups=64, top_groups=7),
          dict(E=48, top_k=5, num_groups=3, top_groups=2), dict(E=36, top_k=4, num_groups=6, top_groups=3),
          dict(E=128, top_k=6, num_groups=2, top_groups=1), dict(E=512, top_k=16, num_groups=4, top_groups=2)]


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("case", ROUTES, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()))
def test_route(case, scoring, biased, renormalize):
    kw = dict(case)
    E, top_k = kw.pop("E"), kw.pop("top_k")
    print(f"case route {case} {scoring} {biased} {renormalize}", flush=True)
    g = torch.Generator().manual_seed(E + top_k)
    bias = 0.2 * torch.randn(E, generator=g) if biased else None
    for M, dtype in ((1, torch.float32), (9, torch.bfloat16)):
        logits = (2 * torch.randn((M, E), generator=g)).to(dtype)
        assert_route(logits, top_k, scoring=scoring, bias=bias, renormalize=renormalize, **kw)


@pytest.mark.parametrize("biased", [False, True])
def test_route_ties_go_to_the_lowest_index(biased):
    g = torch.Generator().manual_seed(5)
    bias = torch.randint(0, 2, (256,), generator=g).float() / 4 if biased else None
    logits = torch.randint(-1, 2, (50, 256), generator=g).float()
    logits[0] = 0
    logits[1] = -0.0
    logits[1, ::3] = 0.0                             # one value with two signs
    assert_route(logits, 20, bias=bias)
    assert_route(logits, 8, bias=bias, scoring="sigmoid", num_groups=8, top_groups=4)
    assert_route(logits.to(torch.bfloat16), 30, bias=bias, num_groups=16, top_groups=4, renormalize=False)


def test_route_scores_nearer_than_fp32_tells():
    """sigmoid(logit) + bias that differ by some 1e-9: fp32 would call them equal, or turn them round"""
    e = torch.arange(64, dtype=torch.float64)
    logits = (0.3 + e * 1e-7).float().repeat(4, 1)
    bias = (0.5 - torch.sigmoid(logits[0].double()) + (e.flip(0) * 7 % 64) * 2e-9).float()
    assert_route(logits, 16, scoring="sigmoid", bias=bias)
    assert_route(40 + logits * 20, 16, scoring="sigmoid", bias=torch.zeros(64))       # saturated: equal in fp32
    assert_route(40 + logits * 20, 16, scoring="sigmoid")


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,scale", [(64, 1, 0.3), (256, 8, 0.1), (200, 4, 0.1), (96, 6, 1000.0), (700, 7, 0.1)])
def test_route_neighbours_and_groups_that_are_almost_equal(E, groups, scale, scoring):
    """in every row one pair of good experts, or a pair of groups, whose choices differ by fp32's last bits of a logit or not at all:
    the order of two, the last that is chosen and the first that is not, and the last group that stays"""
    g = torch.Generator().manual_seed(E)
    bias = (scale * torch.randn(E, generator=g)).float()
    size = E // groups
    if groups > 1:
        bias = bias[:size].repeat(groups)            # (groups alike, so that equal logits make equal groups)
    M, top_k = 150, 8
    logits = torch.randn((M, E), generator=g)
    for m in range(M):
        if groups > 1 and m % 2:
            worth = (torch.sigmoid(logits[m].double()) + bias.double()).view(groups, size).topk(2).values.sum(-1)
            order = worth.argsort(descending=True)
            a, b = order[groups // 2 - 1].item(), order[groups // 2].item()
            copy = logits[m, a * size:(a + 1) * size].clone()
            logits[m, b * size:(b + 1) * size] = copy
            if m % 3:
                logits[m, b * size:(b + 1) * size] = torch.nextafter(copy, torch.tensor(9.0 if m % 3 == 1 else -9.0))
        elif scoring == "sigmoid":
            choice = torch.sigmoid(logits[m].double()) + bias.double()
            order = choice.argsort(descending=True)
            i = m % (top_k + 1)
            a, b = order[i].item(), order[i + 1].item()
            want = choice[a] - bias[b].double()      # the score that makes b's choice a's
            if 0.01 < want < 0.99:
                logits[m, b] = torch.log(want / (1 - want)).float()
        else:
            logits[m, m % E] = logits[m, (m * 7 + 1) % E]
    for kw in (dict(), dict(num_groups=groups, top_groups=max(1, groups // 2))):
        assert_route(logits, top_k, scoring=scoring, bias=bias, **kw)
    assert_route(logits, 64, scoring=scoring, bias=bias)
    assert_route(logits, 63, scoring=scoring, bias=bias)


def test_route_with_infinite_biases():
    g = torch.Generator().manual_seed(11)
    logits = torch.randn((20, 64), generator=g)
    bias = 0.1 * torch.randn(64, generator=g)
    bias[3], bias[50] = float("inf"), float("inf")
    bias[10:30] = -float("inf")
    for scoring in ("softmax", "sigmoid"):
        assert_route(logits, 8, scoring=scoring, bias=bias)
        assert_route(logits, 60, scoring=scoring, bias=bias)
        assert_route(logits, 8, scoring=scoring, bias=bias.clamp(max=0), num_groups=8, top_groups=6)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_masked_experts_and_empty_rows(scoring, dtype):
    g = torch.Generator().manual_seed(6)
    logits = torch.randn((6, 64), generator=g)
    logits[0, 5:] = -float("inf")                    # fewer experts left than top_k
    logits[1] = -float("inf")                        # none
    logits[2] = torch.finfo(dtype).min               # masked with the type's lowest value, all of them
    logits[3, 1:] = torch.finfo(dtype).min
    logits[4] *= 1e4
    logits = logits.to(dtype)
    for kw in (dict(), dict(num_groups=8, top_groups=2), dict(renormalize=False, shared_experts=2, shared_weight=0.25)):
        assert_route(logits, 8, scoring=scoring, **kw)
        if scoring == "softmax" or not kw:
            assert_route(logits, 8, scoring=scoring, bias=0.1 * torch.randn(64, generator=g), **kw)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_rows_with_nan_and_infinity(scoring):
    from alpha_moe_python import layer_hip
    g = torch.Generator().manual_seed(7)
    logits = torch.randn((5, 128), generator=g)
    logits[0, 3] = float("nan")
    logits[1] = float("nan")
    logits[2, 7] = float("inf")
    bias = 0.1 * torch.randn(128, generator=g)
    bias[9] = float("nan")
    for b in (None, bias):
        for kw in (dict(), dict(num_groups=4, top_groups=2)):
            w, ids = layer_hip.route_topk(logits.to(DEV), 8, scoring=scoring, bias=None if b is None else b.to(DEV), **kw)
            w, ids = w.cpu(), ids.cpu()
            assert bool(((ids >= 0) & (ids < 128)).all()) and all(len(set(r.tolist())) == 8 for r in ids)
            assert bool(w[:2].isnan().all()) and 3 not in ids[0].tolist()
            if b is not None:
                assert not (ids[3:] == 9).any()
            if scoring == "softmax":
                assert bool(w[2].isnan().all())      # infinity minus infinity
            else:
                assert bool(w[2].isfinite().all())
            rest = [3, 4]
            want, want_ids = L.route_topk(logits[rest], 8, scoring=scoring, bias=b, **kw)
            assert torch.equal(ids[rest].long(), want_ids)
            assert_within(w[rest], want, 96 * U * want + 2.0 ** -126, "weights")


# ---- all of them -------------------------------------------------------------------------------------------
def all_ops(M, seed=0, K=512, N=384, E=64):
    """Inputs on the GPU and a function that calls the four operators on them."""
    from alpha_moe_python import layer_hip
    x, res = activations(M, K, seed, torch.bfloat16).to(DEV), activations(M, K, seed + 1, torch.bfloat16).to(DEV)
    w = torch.ones(K, dtype=torch.bfloat16, device=DEV)
    _, _, mw, ms = (t.to(DEV) for t in mm_problem(1, 2 * N, K, 3))
    gate = torch.randn((E, K), generator=torch.Generator().manual_seed(4)).to(DEV)
    bias = 0.1 * torch.randn(E, generator=torch.Generator().manual_seed(5)).to(DEV)

    def call():
        r = layer_hip.rms_norm_quant_fp8(x, w, residual=res, keep_norm=True)
        gu = layer_hip.block_scaled_mm(r.q, r.scale, mw, ms)
        q, s = layer_hip.swiglu_quant_fp8(gu)
        logits = (r.norm.float() * gate.sum(0)).reshape(M, E, -1).sum(-1)
        weights, ids = layer_hip.route_topk(logits, 6, scoring="sigmoid", bias=bias, num_groups=8, top_groups=4, shared_experts=1)
        return [r.q.view(torch.uint8), r.scale, r.residual, r.norm, gu, q.view(torch.uint8), s, weights, ids]
    return x, call


@pytest.mark.parametrize("M", [1, 20, 64, 300])
def test_bit_for_bit_from_run_to_run_and_on_two_streams(M):
    x, call = all_ops(M)
    want = call()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(call())
    torch.cuda.synchronize()
    for g in got:
        for a, b in zip(g, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("M", [1, 20, 64, 300])
def test_captured_and_replayed(M):
    x, call = all_ops(M)
    x2, call2 = all_ops(M, seed=50)
    call(), call2()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    graphs = []
    for c in (call, call2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = c()
        graphs.append((g, out))
    for step in range(4):
        for xs, c, (g, out) in ((x, call, graphs[0]), (x2, call2, graphs[1])):
            xs.copy_(activations(M, x.shape[1], 100 + step, torch.bfloat16).to(DEV))
            want = [t.clone() for t in c()]          # eager work between the replays
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b), step


def test_no_rows():
    from alpha_moe_python import layer_hip
    x = torch.empty((0, 256), dtype=torch.bfloat16, device=DEV)
    r = layer_hip.rms_norm_quant_fp8(x, torch.ones(256, device=DEV), residual=x, keep_norm=True)
    assert r.q.shape == (0, 256) and r.scale.shape == (0, 2) and r.residual.shape == (0, 256) and r.norm.shape == (0, 256)
    q, s = layer_hip.swiglu_quant_fp8(x)
    assert q.shape == (0, 128) and s.shape == (0, 1)
    _, _, w, ws = (t.to(DEV) for t in mm_problem(1, 100, 256, 0))
    assert layer_hip.block_scaled_mm(r.q, r.scale, w, ws).shape == (0, 100)
    weights, ids = layer_hip.route_topk(torch.empty((0, 8), device=DEV), 2, shared_experts=1)
    assert weights.shape == ids.shape == (0, 3)


def test_refusals():
    from alpha_moe_python import layer_hip as H
    x = torch.zeros((4, 256), dtype=torch.bfloat16, device=DEV)
    w = torch.ones(256, dtype=torch.bfloat16, device=DEV)
    xq, xs, mw, ws = (t.to(DEV) for t in mm_problem(4, 100, 256, 0))
    logits = torch.zeros((4, 64), device=DEV)
    odd = torch.zeros(4 * 256 + 8, dtype=torch.bfloat16, device=DEV)[4:4 + 1024].view(4, 256)      # 8 bytes off
    bad = [lambda: H.rms_norm_quant_fp8(x.half(), w), lambda: H.rms_norm_quant_fp8(x, w.half()), lambda: H.rms_norm_quant_fp8(x, w[:128]),
           lambda: H.rms_norm_quant_fp8(x[:, :200].contiguous(), w[:200]), lambda: H.rms_norm_quant_fp8(x.t(), w[:4]),
           lambda: H.rms_norm_quant_fp8(x, w, residual=x.float()), lambda: H.rms_norm_quant_fp8(x, w, residual=x[:2]),
           lambda: H.rms_norm_quant_fp8(x, w.cpu()), lambda: H.rms_norm_quant_fp8(x, w, group_size=64), lambda: H.rms_norm_quant_fp8(odd, w),
           lambda: H.rms_norm_quant_fp8(x[0], w), lambda: H.rms_norm_quant_fp8(x[:, ::2], w[:128]),
           lambda: H.swiglu_quant_fp8(x.half()), lambda: H.swiglu_quant_fp8(x[:, :128].contiguous()), lambda: H.swiglu_quant_fp8(odd),
           lambda: H.swiglu_quant_fp8(x, 64),
           lambda: H.block_scaled_mm(xq.float(), xs, mw, ws), lambda: H.block_scaled_mm(xq, xs.double(), mw, ws),
           lambda: H.block_scaled_mm(xq, xs[:, :1].contiguous(), mw, ws), lambda: H.block_scaled_mm(xq, xs, mw[:, :128].contiguous(), ws),
           lambda: H.block_scaled_mm(xq, xs, mw, ws[:, :1].contiguous()),
           lambda: H.block_scaled_mm(xq, xs.t(), mw, ws), lambda: H.block_scaled_mm(xq, xs, mw.cpu(), ws),
           lambda: H.block_scaled_mm(xq, xs, mw[:0], ws[:0]),
           lambda: H.route_topk(logits.half(), 2), lambda: H.route_topk(logits, 65), lambda: H.route_topk(logits, 0),
           lambda: H.route_topk(logits, 2, bias=torch.zeros(63, device=DEV)), lambda: H.route_topk(logits, 2, bias=torch.zeros(64)),
           lambda: H.route_topk(logits, 2, num_groups=3), lambda: H.route_topk(logits, 9, num_groups=8, top_groups=1),
           lambda: H.route_topk(logits, 2, num_groups=2, top_groups=3), lambda: H.route_topk(logits, 2, shared_experts=-1),
           lambda: H.route_topk(logits.t(), 2), lambda: H.route_topk(logits, 2, scoring="relu")]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError, NotImplementedError)):
            call()
            print(f"refusal {i} went through", flush=True)


def test_products_of_codes_that_require_gradients_are_refused():
    from alpha_moe_python import layer_hip as H
    q, s, mw, ms = (t.to(DEV) for t in mm_problem(4, 100, 256, 0))
    for args in ((q.clone().requires_grad_(), s, mw, ms), (q, s, mw.clone().requires_grad_(), ms), (q, s, mw, ms.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="requires a gradient"):
            H.block_scaled_mm(*args)
        with torch.no_grad():
            H.block_scaled_mm(*args)


def test_inputs_that_require_gradients_are_refused():
    from alpha_moe_python import layer_hip as H
    x = torch.zeros((4, 256), dtype=torch.bfloat16, device=DEV)
    w = torch.nn.Parameter(torch.ones(256, device=DEV))
    leaf = torch.zeros((4, 256), dtype=torch.bfloat16, device=DEV, requires_grad=True)
    logits = torch.zeros((4, 64), device=DEV, requires_grad=True)
    bias = torch.zeros(64, device=DEV, requires_grad=True)
    q, s, mw, ms = (t.to(DEV) for t in mm_problem(4, 100, 256, 0))
    calls = [lambda: H.rms_norm_quant_fp8(x, w), lambda: H.rms_norm_quant_fp8(leaf, w.detach()),
             lambda: H.rms_norm_quant_fp8(x, w.detach(), residual=leaf), lambda: H.swiglu_quant_fp8(leaf),
             lambda: H.block_scaled_mm(q, s.requires_grad_(), mw, ms), lambda: H.route_topk(logits, 4),
             lambda: H.route_topk(logits.detach(), 4, bias=bias)]
    for call in calls:
        with pytest.raises(RuntimeError, match="requires a gradient"):
            call()
        with torch.no_grad():
            call()
        with torch.inference_mode():
            call()


def test_schemas_and_fakes_say_what_the_operators_do():
    """no result shares memory with another or with an input; shapes, types and strides are those of the fake implementations"""
    import alpha_moe_ops  # noqa: F401
    o = torch.ops.alpha_moe
    x, w = torch.randn((5, 512), device=DEV).to(torch.bfloat16), torch.ones(512, device=DEV)
    q, s, mw, ms = (t.to(DEV) for t in mm_problem(5, 130, 512, 0))
    logits = torch.randn((5, 64), device=DEV)
    both = ("test_schema", "test_faketensor")
    for op, args, utils in ((o.rms_norm_quant_fp8.default, (x, w, 1e-6, 128), both),
                            (o.rms_norm_quant_fp8.keep_norm, (x, w, 1e-6, 128), both),
                            (o.add_rms_norm_quant_fp8.default, (x, x.clone(), w, 1e-6, 128), both),
                            (o.add_rms_norm_quant_fp8.keep_norm, (x, x.clone(), w, 1e-6, 128), both),
                            (o.swiglu_quant_fp8.default, (x, 128), both),
                            (o.block_scaled_mm.default, (q, s, mw, ms), both[1:]),     # (the schema's check multiplies its inputs)
                            (o.route_topk.default, (logits, None, 4, False, 1, 1, True, 1, 1.0), both)):
        torch.library.opcheck(op, args, test_utils=utils)
