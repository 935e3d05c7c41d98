"""Tokens sorted by expert and back, on the GPU, against the oracle's loops in float64.

Tolerances.  u = 2^-24.  The sort moves values: bit for bit.  A combined value is a sum of top_k products (one rounding each, with the
addition), then a product with the factor, which is itself rounded to fp32: (top_k + 2) u of the sum over magnitudes, and the
rounding to the result's type.  A row's gradient is two products of fp32 numbers and the factor: 3 u, and the rounding.  A weight's
gradient adds up K products, at most K / 64 + 8 of them one behind the other in a thread, then 6 + 4 sums over threads, the factor: (K / 64 + 24)
u of the sum over magnitudes.  Subnormal results: 2^-126 u more.
"""
import pytest
import torch

import alpha_moe
from alpha_moe_python import layer_hip
from oracle import layer_oracle as L
from test_gpu_layer import DEV, U, assert_within, half_step

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def make_ids(M, top_k, E, kind, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "one":
        return torch.full((M, top_k), E - 1, dtype=torch.int32)
    if kind == "none":
        return torch.tensor([-1, E, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32).repeat(M * top_k)[:M * top_k].reshape(M, top_k)
    ids = torch.randint(0, E, (M, top_k), generator=g, dtype=torch.int32)        # (the same expert twice, too)
    if kind == "some":
        ids[torch.rand((M, top_k), generator=g) < 0.4] = -1
        ids[torch.rand((M, top_k), generator=g) < 0.1] = E
    if kind == "padded":
        ids[M - M // 3:] = -1
    return ids


def make_rows(M, K, dtype, seed):
    x = torch.randn((M, K), generator=torch.Generator().manual_seed(seed))
    return x.to(FP8) if dtype == FP8 else x.to(dtype)


def bits(t):
    return t.cpu().contiguous().view(torch.uint8)


def check_sort(x, ids, E, scale=None):
    dev = lambda t: None if t is None else t.to(DEV)
    r = layer_hip.sort_tokens(dev(x), dev(ids), E, x_scale=dev(scale))
    slots, offsets, row_of_slot = L.sort_slots(ids, E)
    live = int(offsets[-1])
    assert torch.equal(r.offsets.cpu(), offsets) and r.offsets.dtype == torch.int32
    assert torch.equal(r.row_of_slot.cpu(), row_of_slot) and r.row_of_slot.dtype == torch.int32
    token = slots // ids.shape[1]
    for got, src in ((r.rows, x), (r.scale, scale)):
        if src is None:
            assert got is None
            continue
        want = src.view(torch.uint8)[token].clone() if src.dtype == FP8 else src[token].clone()
        want[live:] = 0
        assert got.dtype == src.dtype and torch.equal(bits(got), bits(want))
    return r


@pytest.mark.parametrize("kind", ["all", "some", "one", "none", "padded"])
@pytest.mark.parametrize("M,top_k,E,K,dtype", [
    (1, 1, 1, 1, torch.bfloat16), (1, 9, 257, 7168, FP8), (1, 64, 4096, 128, FP8), (3, 2, 5, 7, torch.bfloat16), (5, 10, 8, 3, torch.float32),
    (64, 8, 64, 129, torch.bfloat16), (33, 3, 3, 333, torch.float32), (100, 7, 60, 8, torch.bfloat16), (61, 9, 257, 2048, FP8),
    (2, 17, 512, 8200, torch.bfloat16), (2, 3, 8, 16500, torch.float32), (1024, 8, 4096, 4, torch.bfloat16),
    (1025, 8, 256, 20, torch.bfloat16), (911, 9, 7, 128, FP8), (2731, 3, 60, 9, torch.bfloat16), (8193, 1, 1, 2, torch.bfloat16),
    (1021, 10, 512, 256, torch.float32), (300, 64, 4096, 128, FP8), (5000, 8, 127, 1, torch.float32), (40000, 2, 255, 5, torch.bfloat16),
    (1100, 8, 3, 9001, torch.bfloat16), (1500, 6, 128, 4104, torch.float32)])
def test_sort(M, top_k, E, K, dtype, kind):
    print(f"case sort M={M} top_k={top_k} E={E} K={K} {dtype} {kind}", flush=True)
    x = make_rows(M, K, dtype, M + K)
    scale = torch.rand((M, K // 128)) if dtype == FP8 and M % 2 else None
    check_sort(x, make_ids(M, top_k, E, kind, M), E, scale)


def test_sort_of_many_slots():
    """segments longer than a thousand slots, and more slots than a workgroup's 16 bit"""
    for M, top_k, E in ((600_000, 1, 300), (70_000, 10, 2)):
        print(f"case many slots {M} {top_k} {E}", flush=True)
        ids = make_ids(M, top_k, E, "some", 5)
        x = torch.arange(M, dtype=torch.float32)[:, None]
        r = layer_hip.sort_tokens(x.to(DEV), ids.to(DEV), E)
        e = ids.flatten().long()
        e = torch.where((e >= 0) & (e < E), e, E)
        order = torch.sort(e, stable=True)[1]
        live = int((e < E).sum())
        assert torch.equal(r.rows.cpu()[:live, 0].long(), order[:live] // top_k) and not bool(r.rows[live:].any())
        row = torch.empty_like(order)
        row[order] = torch.arange(M * top_k)
        assert torch.equal(r.row_of_slot.cpu().flatten().long(), torch.where(e < E, row, ~row))
        assert torch.equal(r.offsets.cpu().long(), torch.cat([torch.zeros(1, dtype=torch.long), torch.bincount(e, minlength=E + 1)[:E].cumsum(0)]))


def test_sort_of_nothing():
    for dtype in (torch.bfloat16, FP8):
        r = layer_hip.sort_tokens(torch.empty((0, 128), device=DEV).to(dtype), torch.empty((0, 4), dtype=torch.int32, device=DEV), 5)
        assert r.rows.shape == (0, 128) and r.row_of_slot.shape == (0, 4) and r.offsets.tolist() == [0] * 6
    out = layer_hip.combine_tokens(torch.empty((0, 7), device=DEV), r.row_of_slot)
    assert out.shape == (0, 7)


CASES = [(1, 1, 1, 1), (1, 9, 257, 7168), (3, 4, 5, 7), (61, 9, 64, 333), (16, 2, 3, 2056), (7, 64, 100, 50), (4, 13, 9, 9000), (2, 3, 4, 20000),
         (1200, 8, 60, 24), (5, 10, 512, 4100)]


def check_combine(rows, ids, E, weights, scaling, dtype):
    M, top_k = ids.shape
    _, _, at = L.sort_slots(ids, E)
    got = layer_hip.combine_tokens(rows.to(DEV), at.to(DEV), None if weights is None else weights.to(DEV), scaling)
    want, size = L.combine_tokens(rows, at, weights, scaling)
    assert got.dtype == dtype
    assert_within(got, want, half_step(dtype) * want.abs() + (top_k + 2) * U * size + 2.0 ** -133, "combined")


@pytest.mark.parametrize("kind", ["all", "some", "none", "padded"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,top_k,E,K", CASES)
def test_combine(M, top_k, E, K, dtype, kind):
    print(f"case combine M={M} top_k={top_k} E={E} K={K} {dtype} {kind}", flush=True)
    ids = make_ids(M, top_k, E, kind, M + 1)
    rows = make_rows(M * top_k, K, dtype, K)
    weights = torch.rand((M, top_k), generator=torch.Generator().manual_seed(3))
    check_combine(rows, ids, E, weights, 1.0, dtype)
    check_combine(rows, ids, E, None, 2.5, dtype)


def check_grads(rows, at, weights, g, scaling):
    """gradients of combine_tokens against the formulas"""
    M, top_k = at.shape
    dtype, K = rows.dtype, rows.shape[1]
    rd = rows.to(DEV).requires_grad_()
    wd = None if weights is None else weights.to(DEV).requires_grad_()
    out = layer_hip.combine_tokens(rd, at.to(DEV), wd, scaling)
    got = torch.autograd.grad(out, [rd] if wd is None else [rd, wd], g.to(DEV))
    want_rows, want_weights, size = L.combine_tokens_grad(g, rows, at, weights, scaling)
    assert got[0].dtype == dtype and got[0].shape == rows.shape
    assert_within(got[0], want_rows, (half_step(dtype) + 3 * U) * want_rows.abs() + 2.0 ** -133, "gradient of the rows")
    if wd is not None:
        assert got[1].dtype == torch.float32
        assert_within(got[1], want_weights, (K / 64 + 24) * U * size + 2.0 ** -133, "gradient of the weights")
        only = torch.autograd.grad(layer_hip.combine_tokens(rows.to(DEV), at.to(DEV), wd, scaling), wd, g.to(DEV))[0]
        assert torch.equal(only, got[1])
        only = torch.autograd.grad(layer_hip.combine_tokens(rd, at.to(DEV), weights.to(DEV), scaling), rd, g.to(DEV))[0]
        assert torch.equal(only, got[0])


@pytest.mark.parametrize("kind", ["all", "some", "none"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,top_k,E,K", CASES)
def test_gradients(M, top_k, E, K, dtype, kind):
    print(f"case gradients M={M} top_k={top_k} E={E} K={K} {dtype} {kind}", flush=True)
    ids = make_ids(M, top_k, E, kind, M + 2)
    slots, offsets, at = L.sort_slots(ids, E)
    g = make_rows(M, K, dtype, 9)
    rows = make_rows(M * top_k, K, dtype, K)
    weights = torch.rand((M, top_k), generator=torch.Generator().manual_seed(3))
    check_grads(rows, at, weights, g, 1.5)
    check_grads(rows, at, None, g, 1.0)
    x = make_rows(M, K, dtype, 10).to(DEV).requires_grad_()
    s = layer_hip.sort_tokens(x, ids.to(DEV), E)
    assert s.rows.requires_grad and not s.offsets.requires_grad and not s.row_of_slot.requires_grad
    got = torch.autograd.grad(s.rows, x, rows.to(DEV))[0]
    want, size = L.combine_tokens(rows, at)
    assert_within(got, want, half_step(dtype) * want.abs() + (top_k + 2) * U * size + 2.0 ** -133, "gradient of the tokens")


@pytest.mark.parametrize("K", [5, 256])
def test_gradients_against_differences(K):
    """sum(out * g) is linear in the rows and in the weights: a difference of two values of it is the gradient, whatever the step;
    with steps and values of few bits every sum is exact"""
    M, top_k, E = 6, 3, 4
    g = torch.Generator().manual_seed(K)
    small = lambda *shape: torch.randint(-3, 4, shape, generator=g).float()
    ids = make_ids(M, top_k, E, "some", 4).to(DEV)
    x, w, c = small(M, K).to(DEV).requires_grad_(), small(M, top_k).to(DEV).requires_grad_(), small(M, K).to(DEV)
    scale = small(M * top_k, K).to(DEV)

    def loss(x, w):
        s = layer_hip.sort_tokens(x, ids, E)
        return (layer_hip.combine_tokens(s.rows * scale, s.row_of_slot, w, 2.0) * c).sum()

    gx, gw = torch.autograd.grad(loss(x, w), (x, w))
    with torch.no_grad():
        for t, grad in ((x, gx), (w, gw)):
            for i in range(0, t.numel(), max(1, t.numel() // 40)):
                step = torch.zeros_like(t)
                step.view(-1)[i] = 1.0
                plus, minus = (loss(x + d, w) if t is x else loss(x, w + d) for d in (step, -step))
                assert (plus - minus).item() / 2 == grad.view(-1)[i].item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [40, 333, 9000])
def test_what_has_no_expert_is_never_looked_at(dtype, K):
    """rows, weights and gradients behind the last expert hold NaN and infinities"""
    M, top_k, E = 12, 5, 6
    ids = make_ids(M, top_k, E, "some", 8)
    _, offsets, at = L.sort_slots(ids, E)
    rows = make_rows(M * top_k, K, dtype, 1)
    clean = rows.clone()
    rows[int(offsets[-1])::2] = float("nan")
    rows[int(offsets[-1]) + 1::2] = float("inf")
    weights = torch.rand((M, top_k))
    weights[at < 0] = float("nan")
    check_combine(rows, ids, E, weights, 1.0, dtype)
    check_grads(rows, at, weights, make_rows(M, K, dtype, 2), 1.0)
    x = make_rows(M, K, dtype, 3).to(DEV).requires_grad_()
    s = layer_hip.sort_tokens(x, ids.to(DEV), E)
    a, b = (torch.autograd.grad(s.rows, x, r.to(DEV), retain_graph=True)[0] for r in (rows, clean))
    assert torch.equal(a, b)
    # and where they do have one, they are seen
    rows = clean.clone()
    rows[0], rows[1] = float("nan"), float("inf")
    check_combine(rows, ids, E, torch.ones((M, top_k)), 1.0, dtype)


def test_weights_of_zero_and_values_at_the_ends_of_the_types():
    M, top_k, E, K = 4, 3, 5, 64
    ids = make_ids(M, top_k, E, "all", 8)
    _, _, at = L.sort_slots(ids, E)
    rows = make_rows(M * top_k, K, torch.bfloat16, 1)
    rows[:, 0], rows[:, 1], rows[:, 2] = 3.0e38, 1e-40, -3.0e38
    weights = torch.tensor([0.0, -0.0, 2.0 ** -3]).repeat(M, 1)
    check_combine(rows, ids, E, weights, 1.0, torch.bfloat16)
    check_combine(rows.float(), ids, E, weights, 0.5, torch.float32)


def c_abi(name, *args):
    rc = getattr(alpha_moe.c_abi, name)(*args, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return rc


@pytest.mark.parametrize("M,top_k,E,K", [(5, 3, 4, 11), (9, 2, 4, 64), (1500, 7, 30, 11)])
def test_nothing_beside_the_results(M, top_k, E, K):
    """what lies behind each result stays as it was; a map that names rows that do not exist is harmless"""
    def guarded(n, dtype, fill=7):
        return torch.full((n + 512,), fill, dtype=dtype, device=DEV)
    ids = make_ids(M, top_k, E, "some", 3)
    x = make_rows(M, K, torch.bfloat16, 4)
    R = M * top_k
    slots, offsets, at = L.sort_slots(ids, E)
    rows, off, row_of = guarded(R * K, torch.bfloat16), guarded(E + 1, torch.int32), guarded(R, torch.int32)
    need = alpha_moe.c_abi.alpha_moe_sort_workspace_bytes(M, top_k, E)
    ws = torch.full((need + 512,), 7, dtype=torch.uint8, device=DEV)
    xd, idd = x.to(DEV), ids.to(DEV)
    assert c_abi("alpha_moe_sort_tokens", xd.data_ptr(), 2, None, idd.data_ptr(), rows.data_ptr(), None, off.data_ptr(), row_of.data_ptr(),
                 M, K, top_k, E, ws.data_ptr(), need) == 0
    for got, n in ((rows, R * K), (off, E + 1), (row_of, R), (ws, need)):
        assert bool((got[n:] == 7).all())
    want = x[slots // top_k].clone()
    want[int(offsets[-1]):] = 0
    assert torch.equal(rows[:R * K].view(R, K).cpu(), want) and torch.equal(row_of[:R].view(M, top_k).cpu(), at)
    bad = at.clone()
    bad[0, 0], bad[1, 1], bad[2, 0], bad[3, 1] = R, 2 ** 31 - 1, ~R, -2 ** 31
    known = bad.clone()
    known[0, 0] = known[1, 1] = -1
    out, gr, gw = guarded(M * K, torch.bfloat16), guarded(R * K, torch.bfloat16), guarded(R, torch.float32)
    w = torch.rand((M, top_k))
    bd, wd, rd = bad.to(DEV), w.to(DEV), want.to(DEV)
    assert c_abi("alpha_moe_combine_tokens", rd.data_ptr(), 0, bd.data_ptr(), wd.data_ptr(), out.data_ptr(), M, K, top_k, 1.0) == 0
    sums, size = L.combine_tokens(want, known, w)
    assert_within(out[:M * K].view(M, K), sums, 2.0 ** -8 * sums.abs() + (top_k + 2) * U * size, "sums")
    assert c_abi("alpha_moe_combine_tokens_grad", xd.data_ptr(), rd.data_ptr(), 0, bd.data_ptr(), wd.data_ptr(), gr.data_ptr(),
                 gw.data_ptr(), M, K, top_k, 1.0) == 0
    for got, n in ((out, M * K), (gr, R * K), (gw, R)):
        assert bool((got[n:] == 7).all())
    assert gw[0].item() == 0 and gw[top_k + 1].item() == 0


def test_gradients_of_gradients():
    """a sort's gradient is a combination and has one itself; a combination's gradient has none and says so"""
    M, top_k, E, K = 5, 3, 4, 8
    ids = make_ids(M, top_k, E, "some", 3).to(DEV)
    x = make_rows(M, K, torch.float32, 1).to(DEV).requires_grad_()
    s = layer_hip.sort_tokens(x, ids, E)
    g = make_rows(M * top_k, K, torch.float32, 2).to(DEV).requires_grad_()
    gx = torch.autograd.grad(s.rows, x, g, create_graph=True)[0]
    gg = torch.autograd.grad(gx, g, torch.ones_like(gx))[0]
    assert torch.equal(gg, torch.where(torch.arange(M * top_k, device=DEV)[:, None] < s.offsets[-1], 1.0, 0.0).expand(-1, K))
    rows = s.rows.detach().requires_grad_()
    w = torch.rand((M, top_k), device=DEV, requires_grad=True)
    out = layer_hip.combine_tokens(rows, s.row_of_slot, w)
    with pytest.raises(RuntimeError, match="requires a gradient"):
        torch.autograd.grad(out.sum(), (rows, w), create_graph=True)


def test_views_and_expanded_gradients():
    """gradients arrive expanded or transposed, rows as a result that is part of a graph; inputs that are not contiguous are refused"""
    M, top_k, E, K = 9, 2, 4, 16
    ids = make_ids(M, top_k, E, "all", 3).to(DEV)
    x = make_rows(M, K, torch.float32, 1).to(DEV).requires_grad_()
    s = layer_hip.sort_tokens(x, ids, E)
    layer_hip.combine_tokens(s.rows, s.row_of_slot).sum().backward()             # (a gradient of strides 0)
    assert torch.equal(x.grad, torch.full_like(x, top_k))
    s = layer_hip.sort_tokens(x, ids, E)
    g = torch.randn((K, M * top_k), device=DEV).t()
    assert torch.equal(torch.autograd.grad(s.rows, x, g, retain_graph=True)[0], torch.autograd.grad(s.rows, x, g.contiguous())[0])
    with pytest.raises(RuntimeError, match="contiguous"):
        layer_hip.sort_tokens(x.detach().t().contiguous().t(), ids, E)
    with pytest.raises(RuntimeError, match="contiguous"):
        layer_hip.combine_tokens(s.rows.detach(), s.row_of_slot.t().contiguous().t())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [7, 64, 333])
def test_tensors_that_start_anywhere(dtype, K):
    """parts of larger tensors, as gradients of concatenated results are: any multiple of a value's size"""
    M, top_k, E = 9, 3, 5
    ids = make_ids(M, top_k, E, "some", 3)
    _, _, at = L.sort_slots(ids, E)
    part = lambda t: torch.cat([t.flatten()[:1], t.flatten()]).to(DEV)[1:].view(t.shape)
    x, rows, g, w = make_rows(M, K, dtype, 1), make_rows(M * top_k, K, dtype, 2), make_rows(M, K, dtype, 3), torch.rand((M, top_k))
    assert part(x).data_ptr() % 16 != 0
    a, b = (layer_hip.sort_tokens(t, ids.to(DEV), E) for t in (part(x), x.to(DEV)))
    assert torch.equal(a.rows, b.rows)
    xd = x.to(DEV).requires_grad_()
    s = layer_hip.sort_tokens(xd, ids.to(DEV), E)
    both = torch.cat([s.rows[:0], torch.ones((1, K), dtype=dtype, device=DEV), s.rows])          # (its gradient is a part that starts behind a row)
    want = L.combine_tokens(rows, at)[0]
    got = torch.autograd.grad(both, xd, torch.cat([rows[:1], rows]).to(DEV))[0]
    assert_within(got, want, half_step(dtype) * want.abs() + 8 * U * L.combine_tokens(rows, at)[1], "gradient of the tokens")
    for r, gg in ((part(rows), g.to(DEV)), (rows.to(DEV), part(g)), (part(rows), part(g))):
        rd, wd = r.requires_grad_(), w.to(DEV).requires_grad_()
        got = torch.autograd.grad(layer_hip.combine_tokens(rd, at.to(DEV), wd), (rd, wd), gg)
        rp, wp = rows.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
        want = torch.autograd.grad(layer_hip.combine_tokens(rp, at.to(DEV), wp), (rp, wp), g.to(DEV))
        assert torch.equal(got[0], want[0])
        assert_within(got[1], want[1].cpu().double(), (K / 32 + 48) * U * L.combine_tokens_grad(g, rows, at, w)[2], "gradient of the weights")


def test_offsets_past_32_bits():
    """rows of more than 4 GiB, there and back"""
    M, top_k, E, K = 6000, 8, 40, 57344
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn((M, K), generator=g, device=DEV, dtype=torch.bfloat16)
    ids = torch.randint(0, E, (M, top_k), generator=g, device=DEV, dtype=torch.int32)
    s = layer_hip.sort_tokens(x, ids, E)
    order = torch.sort(ids.flatten(), stable=True)[1]
    for lo in (0, 20000, M * top_k - 300):           # (also behind 4 GiB: row 37450 and on)
        assert torch.equal(s.rows[lo:lo + 300], x[order[lo:lo + 300] // top_k])
    assert s.rows.numel() * 2 > 2 ** 32
    out = layer_hip.combine_tokens(s.rows, s.row_of_slot, None, 1 / top_k)
    assert torch.equal(out, x)                       # (the mean of eight equal values: sums of three bits more are exact in fp32)
    rows = s.rows.requires_grad_()
    got = torch.autograd.grad(layer_hip.combine_tokens(rows, s.row_of_slot), rows, x)[0]
    assert torch.equal(got[-200:], x[order[-200:] // top_k]) and torch.equal(got[:200], x[order[:200] // top_k])


def test_operators_trace_with_their_gradients():
    """schemas, fake implementations and the registration of the gradients, as torch's own checks see them"""
    M, top_k, E, K = 5, 3, 4, 12
    ids = make_ids(M, top_k, E, "some", 3).to(DEV)
    x = torch.randn((M, K), device=DEV, requires_grad=True)
    at = layer_hip.sort_tokens(x.detach(), ids, E).row_of_slot
    rows, w = torch.randn((M * top_k, K), device=DEV, requires_grad=True), torch.rand((M, top_k), device=DEV, requires_grad=True)
    import alpha_moe_ops  # noqa: F401  (fake implementations)
    O = torch.ops.alpha_moe
    torch.library.opcheck(O.sort_tokens.default, (x, ids, E))
    torch.library.opcheck(O.combine_tokens.default, (rows, at, w, 0.5))
    torch.library.opcheck(O.combine_tokens.default, (rows, at, None, 1.0))


def test_refusals():
    x, ids = torch.zeros((4, 128), device=DEV), torch.zeros((4, 2), dtype=torch.int32, device=DEV)
    rows, at, w = torch.zeros((8, 128), device=DEV), torch.zeros((4, 2), dtype=torch.int32, device=DEV), torch.ones((4, 2), device=DEV)
    q, sc = x.to(FP8), torch.ones((4, 1), device=DEV)
    H = layer_hip
    for call, message in (
            (lambda: H.sort_tokens(x.half(), ids, 4), "bfloat16, float32 or float8"), (lambda: H.sort_tokens(x[0], ids, 4), r"\[M, K\]"),
            (lambda: H.sort_tokens(x, ids.long(), 4), "dtype"), (lambda: H.sort_tokens(x, ids[:3], 4), "top_k"),
            (lambda: H.sort_tokens(x, ids.cpu(), 4), "must be on"), (lambda: H.sort_tokens(x, ids[:, 0], 4), "contiguous"),
            (lambda: H.sort_tokens(x, ids, 0), "num_experts"), (lambda: H.sort_tokens(x, ids, 4097), "num_experts"),
            (lambda: H.sort_tokens(x, torch.zeros((4, 65), dtype=torch.int32, device=DEV), 4), "64"),
            (lambda: H.sort_tokens(x, torch.zeros((4, 0), dtype=torch.int32, device=DEV), 4), "top_k"),
            (lambda: H.sort_tokens(x, ids, 4, x_scale=sc), "goes with codes"), (lambda: H.sort_tokens(q, ids, 4, x_scale=sc[:3]), "x_scale"),
            (lambda: H.sort_tokens(q[:, :64].contiguous(), ids, 4), "128"), (lambda: H.sort_tokens(q, ids, 4, x_scale=sc.half()), "dtype"),
            (lambda: H.sort_tokens(torch.zeros((4 * 128 + 8,), device=DEV).to(FP8)[8:].view(4, 128), ids, 4), "multiple of 16"),
            (lambda: H.combine_tokens(rows.half(), at), "bfloat16 or float32"), (lambda: H.combine_tokens(rows[:7], at), "one row for each"),
            (lambda: H.combine_tokens(rows, at, w[:, :1]), "contiguous"), (lambda: H.combine_tokens(rows, at, w[:3]), "shape"), (lambda: H.combine_tokens(rows, at, w.bfloat16()), "dtype"),
            (lambda: H.combine_tokens(rows, at.long()), "dtype"), (lambda: H.combine_tokens(rows, at, w.cpu()), "must be on"),
            (lambda: H.sort_tokens(q.requires_grad_(), ids, 4), "requires a gradient")):
        with pytest.raises(RuntimeError, match=message):
            call()


def test_streams_and_replays():
    """captured with the backward passes, replayed between eager calls; then two streams at once"""
    M, top_k, E, K = 700, 16, 40, 72                                     # (more slots than one launch sorts)
    g = torch.Generator().manual_seed(2)
    x = torch.randn((M, K), generator=g).to(DEV).requires_grad_()
    w = torch.rand((M, top_k), generator=g).to(DEV).requires_grad_()
    ids, c = make_ids(M, top_k, E, "some", 1).to(DEV), torch.randn((M, K), generator=g).to(DEV)

    def step(x, w):
        s = layer_hip.sort_tokens(x, ids, E)
        out = layer_hip.combine_tokens(s.rows * s.rows, s.row_of_slot, w)
        return (out.detach(), s.row_of_slot, *torch.autograd.grad(out, (x, w), c))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, w)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = step(x, w)
    for i in range(3):
        with torch.no_grad():
            x.copy_(torch.randn((M, K), generator=g))
            ids.copy_(make_ids(M, top_k, E, ("some", "one", "all")[i], i))
        graph.replay()
        torch.cuda.synchronize()
        want = step(x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_())
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i
    streams = [torch.cuda.Stream() for _ in range(2)]
    inputs = [torch.randn((M, K), generator=g).to(DEV) for _ in streams]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for st, t in zip(streams, inputs):
            with torch.cuda.stream(st):
                got.append(layer_hip.sort_tokens(t, ids, E).rows)
    torch.cuda.synchronize()
    want = [layer_hip.sort_tokens(t, ids, E).rows for t in inputs]
    assert all(torch.equal(a, want[i % 2]) for i, a in enumerate(got))
