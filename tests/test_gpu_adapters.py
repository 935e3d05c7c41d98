"""Adapters of many requests beside a shared projection, on the GPU, against the float64 oracle.

Tolerances.  u = 2^-24.  The first product adds up K exact products in fp32, in an order that is the matrix core's: at most K additions
behind each other, 2 u each if it cuts instead of rounding, some 64 more for the scales and the parts: (2 K + 64) u of the sum over
magnitudes.  The rank's values are then good to 2^-16, their second product is 2 rank additions of 2 u and a few roundings: 2^-16 + (4 rank +
12) u.  The result is rounded to bf16, 2^-8.
"""
import ctypes

import pytest
import torch

import alpha_moe
from alpha_moe_python import layer_hip
from alpha_moe_python.prep import per_token_group_quant_fp8
from oracle import layer_oracle as L
from test_gpu_layer import DEV, U, assert_within

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def problem(M, N, K, rank, adapters, ids, fp8=False, scaled=True, seed=0):
    g = torch.Generator().manual_seed(seed + M + N)
    x = torch.randn((M, K), generator=g) * (0.3 + torch.rand((M, 1), generator=g))
    x, xs = per_token_group_quant_fp8(x, 128) if fp8 else (x.to(BF), None)
    base = torch.randn((M, N), generator=g).to(BF)
    a = (torch.randn((adapters, rank, K), generator=g) / K ** 0.5).to(BF)
    b = torch.randn((adapters, N, rank), generator=g).to(BF)
    scale = 0.5 + torch.rand(adapters, generator=g) if scaled else None
    if ids == "runs":
        ids = (torch.arange(M) * 7 // max(1, M) * 3) % adapters
    elif ids == "mixed":
        ids = torch.randint(-1, adapters + 1, (M,), generator=g)
    elif ids == "none":
        ids = torch.tensor([-1, adapters, 2 ** 31 - 1, -2 ** 31]).repeat(M)[:M]
    elif ids == "same":
        ids = torch.full((M,), adapters - 1)
    return dict(base=base, x=x, a=a, b=b, adapter_ids=ids.to(torch.int32), scale=scale, x_scale=xs)


def run(p):
    return layer_hip.add_adapters(**{k: None if v is None else v.to(DEV) for k, v in p.items()})


def check(p, got):
    want, inner, outer = L.add_adapters(p["base"], p["x"], p["a"], p["b"], p["adapter_ids"], p["scale"], p["x_scale"])
    K, rank = p["x"].shape[1], p["a"].shape[1]
    off = (2 * K + 64) * U * inner + (2.0 ** -16 + (4 * rank + 12) * U) * outer
    assert got.dtype == BF
    assert_within(got, want, off + 2.0 ** -8 * (want.abs() + off), "adapted")
    none = (p["adapter_ids"] < 0) | (p["adapter_ids"] >= p["a"].shape[0])
    assert torch.equal(got.cpu()[none], p["base"][none])


@pytest.mark.parametrize("ids", ["runs", "mixed", "none", "same"])
@pytest.mark.parametrize("M,N,K,rank,adapters,fp8", [
    (1, 1, 128, 8, 1, False), (1, 4096, 7168, 16, 8, False), (2, 17, 256, 24, 3, True), (15, 63, 384, 32, 40, False), (16, 64, 640, 16, 5, True),
    (17, 65, 128, 40, 2, False), (33, 257, 1152, 64, 33, True), (61, 2112, 1024, 8, 48, True), (64, 300, 512, 128, 7, False),
    (100, 129, 256, 72, 100, True), (257, 1000, 384, 48, 9, False), (600, 130, 128, 16, 600, False), (1025, 66, 256, 16, 20, False),
    (1100, 255, 128, 32, 6, True), (1030, 513, 384, 56, 11, True), (1040, 64, 256, 104, 5, False), (2000, 31, 128, 8, 70, True),
    (5, 96, 65536, 16, 2, True), (3, 40, 16384, 128, 3, False),
    (2100, 33, 128, 16, 9, False), (2300, 1040, 128, 24, 7, True), (2070, 1100, 256, 64, 3, False), (2080, 70, 128, 48, 12, True),
    (2060, 40, 128, 128, 5, False)])
def test_adapters(M, N, K, rank, adapters, fp8, ids):
    print(f"case adapters M={M} N={N} K={K} rank={rank} of {adapters} fp8={fp8} {ids}", flush=True)
    p = problem(M, N, K, rank, adapters, ids, fp8, scaled=M % 2 == 1)
    got = run(p)
    check(p, got)
    assert torch.equal(got, run(p))


@pytest.mark.parametrize("M,rank,fp8", [(1, 8, False), (40, 16, True), (30, 72, False), (1200, 16, False), (1300, 24, True), (1200, 40, False)])
def test_integers_are_exact(M, rank, fp8):
    """small integers, whose sums fp32 holds and whose rank values 16 bits hold: bit for bit, so every value is in its place"""
    g = torch.Generator().manual_seed(M)
    N, K, adapters = 75, 256, 6
    x = torch.randint(-4, 5, (M, K), generator=g).float()
    p = dict(base=torch.randint(-8, 9, (M, N), generator=g).to(BF), x=x.to(torch.float8_e4m3fn if fp8 else BF),
             a=torch.randint(-2, 3, (adapters, rank, K), generator=g).to(BF), b=torch.randint(-1, 2, (adapters, N, rank), generator=g).to(BF),
             adapter_ids=torch.randint(0, adapters, (M,), generator=g, dtype=torch.int32), scale=2.0 ** torch.arange(adapters).float(),
             x_scale=2.0 ** torch.randint(-2, 1, (M, 2), generator=g).float() if fp8 else None)
    want = L.add_adapters(p["base"], p["x"], p["a"], p["b"], p["adapter_ids"], p["scale"], p["x_scale"])[0]
    assert torch.equal(run(p).cpu(), want.float().to(BF))


@pytest.mark.parametrize("M,rank", [(40, 16), (40, 72), (1200, 24), (1200, 40)])
def test_other_requests_are_never_looked_at(M, rank):
    """NaN and infinities in another adapter, another token's activations, or the scale of an adapter that nobody has"""
    p = problem(M, 70, 256, rank, 5, "mixed", scaled=True)
    clean = run(p).cpu()
    bad = {k: None if v is None else v.clone() for k, v in p.items()}
    bad["a"][2], bad["b"][2], bad["scale"][2] = float("nan"), float("inf"), float("nan")
    bad["x"][3], bad["base"][4] = float("nan"), float("inf")
    got = run(bad).cpu()
    keep = p["adapter_ids"] != 2
    keep[3] = keep[4] = False
    assert torch.equal(got[keep], clean[keep]) and bool(got[p["adapter_ids"] == 2].isnan().all())
    if 0 <= int(p["adapter_ids"][3]) < 5:
        assert bool(got[3].isnan().all())


def test_values_at_the_ends_of_the_types():
    """rank values that are infinite, past bf16's largest number, or subnormal"""
    K, N, rank = 128, 64, 8
    x = torch.zeros((4, K), dtype=BF)
    x[0, 0], x[1, 0], x[2, 0], x[3, 0] = 3.0e38, 1.6987e38, 1e-38, float("inf")
    a, b = torch.zeros((1, rank, K), dtype=BF), torch.zeros((1, N, rank), dtype=BF)
    a[0, :, 0], b[0, :, 0] = 2.0, 0.5
    base = torch.zeros((4, N), dtype=BF)
    ids = torch.zeros(4, dtype=torch.int32, device=DEV)
    got = layer_hip.add_adapters(*(t.to(DEV) for t in (base, x, a, b)), ids).cpu().float()
    # 2 * 3.0e38 and 2 * 2^127 (1.6987e38 in bf16) are past fp32, and an infinity meets seven zeros of b
    assert bool(got[[0, 1, 3]].isnan().all())
    assert bool(((got[2] - x[2, 0].float()).abs() <= 2.0 ** -8 * 1e-38 + 2.0 ** -133).all())
    # without zeros in b: infinite; and rank values up to fp32's largest, whose upper bits are no infinity
    a[0, :, 0], b[0] = 1.0, 2.0 ** -4
    x[1, 0] = 3.3895e38
    got = layer_hip.add_adapters(*(t.to(DEV) for t in (base, x, a, b)), ids).cpu().float()
    assert bool((got[3] == float("inf")).all())
    for m in range(3):                               # (eight ranks of a sixteenth: half of x)
        assert bool(((got[m] - x[m, 0].float() / 2).abs() <= 2.0 ** -8 * x[m, 0].float() / 2 + 2.0 ** -133).all())


def test_no_rows_and_refusals():
    p = {k: None if v is None else v.to(DEV) for k, v in problem(4, 64, 256, 16, 3, "mixed").items()}
    H = layer_hip.add_adapters
    none = dict(p, base=p["base"][:0], x=p["x"][:0], adapter_ids=p["adapter_ids"][:0])
    assert H(**none).shape == (0, 64)
    for kw, message in ((dict(base=p["base"].float()), "dtype"), (dict(x=p["x"].float()), "dtype"), (dict(x=p["x"][:3]), r"\[M, K\]"),
                        (dict(x_scale=torch.ones((4, 2), device=DEV)), "dtype"), (dict(a=p["a"][:, :12].contiguous()), "rank"),
                        (dict(a=p["a"][:, :8].contiguous()), r"\[L, N, rank\]"), (dict(b=p["b"][:2]), r"\[L, N, rank\]"),
                        (dict(a=p["a"][..., :128].contiguous()), "K of x"), (dict(adapter_ids=p["adapter_ids"].long()), "dtype"),
                        (dict(adapter_ids=p["adapter_ids"][:3]), r"\[M\]"), (dict(scale=p["scale"][:2]), r"\[L\]"),
                        (dict(scale=p["scale"].cpu()), "must be on"), (dict(base=p["base"].t().contiguous().t()), "contiguous"),
                        (dict(b=p["b"].clone().requires_grad_()), "requires a gradient"),
                        (dict(x=torch.zeros(4 * 256 + 1, dtype=BF, device=DEV)[1:].view(4, 256)), "multiple of 16")):
        with pytest.raises(RuntimeError, match=message):
            H(**dict(p, **kw))


@pytest.mark.parametrize("M,N,rank", [(5, 33, 8), (70, 130, 40), (1100, 35, 16)])
def test_nothing_beside_the_rows_and_in_place(M, N, rank):
    K, adapters = 256, 4
    p = problem(M, N, K, rank, adapters, "mixed")
    d = {k: None if v is None else v.to(DEV) for k, v in p.items()}
    want = run(p)
    need = alpha_moe.c_abi.alpha_moe_adapters_workspace_bytes(M, N, K, rank, adapters)
    ws = torch.full((need + 512,), 7, dtype=torch.uint8, device=DEV)
    out = torch.cat([p["base"].flatten(), torch.full((2048,), 7.0, dtype=BF)]).to(DEV)
    rc = alpha_moe.c_abi.alpha_moe_add_adapters(out.data_ptr(), d["x"].data_ptr(), None, d["a"].data_ptr(), d["b"].data_ptr(),
                                                d["adapter_ids"].data_ptr(), d["scale"].data_ptr(), out.data_ptr(), M, N, K, rank, adapters,
                                                ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert rc == 0 and torch.equal(out[:M * N].view(M, N), want) and bool((out[M * N:] == 7).all()) and bool((ws[need:] == 7).all())


def test_replays_and_streams():
    p = {k: None if v is None else v.to(DEV) for k, v in problem(50, 200, 640, 32, 9, "mixed", fp8=True).items()}
    layer_hip.add_adapters(**p)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        out = layer_hip.add_adapters(**p)
    g = torch.Generator().manual_seed(1)
    for i in range(3):
        p["adapter_ids"].copy_(torch.randint(-1, 9, (50,), generator=g, dtype=torch.int32))
        p["base"].normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, layer_hip.add_adapters(**p)), i
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    others = [p, dict(p, adapter_ids=p["adapter_ids"].flip(0).contiguous())]
    torch.cuda.synchronize()
    for _ in range(4):
        for s, q in zip(streams, others):
            with torch.cuda.stream(s):
                got.append(layer_hip.add_adapters(**q))
    torch.cuda.synchronize()
    want = [layer_hip.add_adapters(**q) for q in others]
    assert all(torch.equal(t, want[i % 2]) for i, t in enumerate(got))


def test_offsets_past_32_bits():
    """adapters of more than 4 GiB each way"""
    L_, rank, K, N, M = 300, 128, 65536, 70000, 9
    a = torch.zeros((L_, rank, K), dtype=BF, device=DEV)
    b = torch.zeros((L_, N, rank), dtype=BF, device=DEV)
    assert a.numel() * 2 > 2 ** 32 and b.numel() * 2 > 2 ** 32
    ids = torch.tensor([299, 0, 298, 299, 150, -1, 299, 298, 0], dtype=torch.int32)
    for l in set(ids.tolist()) - {-1}:
        a[l, l % rank, K - 1], b[l, N - 1, l % rank], b[l, 5, l % rank] = 2.0, 3.0, float(l % 7)
    x = torch.zeros((M, K), dtype=BF, device=DEV)
    x[:, K - 1] = torch.arange(1, M + 1).to(BF).to(DEV)
    base = torch.ones((M, N), dtype=BF, device=DEV)
    got = layer_hip.add_adapters(base, x, a, b, ids.to(DEV)).cpu()
    for m, l in enumerate(ids.tolist()):
        want = torch.ones(N)
        if l >= 0:
            want[N - 1], want[5] = 1 + 6.0 * (m + 1), 1 + 2.0 * (m + 1) * (l % 7)
        assert torch.equal(got[m].float(), want), m


@pytest.mark.parametrize("M,N,rank,fp8", [(1, 70, 8, False), (20, 64, 16, True), (40, 257, 24, False), (40, 33, 40, False), (9, 130, 128, True),
                                          (2100, 1100, 32, False), (2100, 1090, 64, True), (2100, 1100, 128, False), (8200, 1100, 8, False)])
def test_rank_values_of_24_bits_and_what_cancels(M, N, rank, fp8):
    """One rank's value needs 24 bits, and base and a second rank's value cancel the upper ones: every sum is exact in fp32 (multiples of
    2^-23 below 4, times the token's power of two), and so is the result, which is the lower bits."""
    K, adapters = 128, 3
    low = [1, 2.0 ** -3, 2.0 ** -6]                                    # 2^-17 (1 + 2^-3 + 2^-6): seven bits
    x = torch.zeros((M, K))
    x[:, 0], x[:, 1] = 1.0, 2.0 ** -8
    x[:, 2:5] = torch.tensor(low)
    size = 2.0 ** (torch.arange(M) % 5 - 2).float()[:, None]
    a, b = torch.zeros((adapters, rank, K), dtype=BF), torch.zeros((adapters, N, rank), dtype=BF)
    if fp8:                                                            # (the powers of two in the scales and in a: codes hold 2^-6 and up)
        x[:, 1] = 1.0
        scale, x = size.clone(), x.to(torch.float8_e4m3fn)
    else:
        scale, x = None, (x * size).to(BF)
    first, second = 1, rank - 1
    a[:, first, 0], a[:, first, 1], a[:, first, 2:5] = 1.0, 2.0 ** -8 if fp8 else 1.0, 2.0 ** -17
    a[:, second, 1] = -(2.0 ** -8) if fp8 else -1.0
    sign = (1.0 - 2.0 * (torch.arange(N) % 2)) * 2.0 ** (torch.arange(N) % 3).float()
    b[:, :, first], b[:, :, second] = sign.to(BF), sign.to(BF)
    base = (-size * sign).to(BF)
    got = layer_hip.add_adapters(base.to(DEV), x.to(DEV), a.to(DEV), b.to(DEV), (torch.arange(M) % adapters).to(torch.int32).to(DEV),
                                 x_scale=None if scale is None else scale.to(DEV))
    assert torch.equal(got.cpu().float(), sum(low) * 2.0 ** -17 * size * sign)


@pytest.mark.parametrize("M,N,rank", [(3, 7, 8), (40, 64, 16), (70, 129, 40), (2100, 1091, 24), (2100, 1091, 72)])
def test_tokens_without_an_adapter_keep_their_bits(M, N, rank):
    """a zero's sign, NaN of any payload, subnormals: what base holds is what they get"""
    p = problem(M, N, 128, rank, 3, "mixed")
    odd = torch.tensor([-0x8000, 0x7f81, 0x7fff, -1, -0x7f, 0x7f80, -0x80, 1, -0x7fff, 0], dtype=torch.int16)
    p["base"] = odd.repeat(M * N // 10 + 1)[:M * N].reshape(M, N).view(BF)
    p["adapter_ids"][0] = -1
    none = (p["adapter_ids"] < 0) | (p["adapter_ids"] >= 3)
    assert torch.equal(run(p).cpu().view(torch.int16)[none], p["base"].view(torch.int16)[none])


# (tokens of a tile in the first and the second kernel, 256 columns that a workgroup of the second takes), M, N, K, rank, adapters, fp8.
# K of up to four blocks is in one part, whatever the tile
TILES = [
    ((16, 16, 1), 40, 70, 128, 16, 5, False), ((16, 16, 1), 61, 200, 384, 8, 9, True), ((16, 16, 1), 700, 1300, 512, 32, 9, True),
    ((16, 16, 1), 500, 333, 256, 64, 6, False),
    ((16, 16, 1), 300, 257, 384, 128, 9, True), ((64, 16, 1), 2000, 1100, 256, 40, 9, False), ((64, 16, 1), 8200, 130, 128, 8, 7, True),
    ((16, 64, 1), 4000, 1091, 256, 16, 9, False), ((16, 64, 1), 2100, 1100, 384, 24, 5, True),
    ((64, 64, 1), 8200, 1100, 128, 8, 11, False), ((64, 64, 1), 8200, 1025, 256, 8, 11, True), ((64, 64, 1), 4200, 1091, 384, 16, 9, False),
    ((64, 64, 1), 4200, 1100, 128, 16, 9, True), ((64, 64, 1), 2800, 1090, 256, 24, 9, False), ((64, 64, 1), 2100, 1090, 512, 32, 4, True),
    ((64, 64, 1), 2800, 1100, 128, 40, 30, False), ((64, 64, 1), 2100, 1091, 256, 64, 9, True), ((64, 32, 1), 2100, 1100, 128, 72, 9, False),
    ((64, 32, 1), 2100, 1091, 256, 128, 9, True),
    ((64, 64, 2), 8200, 6001, 128, 8, 37, False), ((64, 64, 2), 8200, 6081, 128, 24, 9, True), ((64, 64, 3), 8200, 9100, 128, 64, 9, False),
    ((64, 32, 2), 4200, 6001, 128, 72, 9, False), ((64, 64, 4), 8200, 12101, 128, 16, 9, True), ((64, 32, 4), 8200, 7000, 128, 128, 9, False)]


def plan_of(M, N, K, rank, adapters):
    plan = (ctypes.c_int * 6)()
    assert alpha_moe.c_abi.alpha_moe_adapters_plan(M, N, K, rank, adapters, plan) == 0
    return plan[0], plan[2], plan[5]


@pytest.mark.parametrize("tiles,M,N,K,rank,adapters,fp8", TILES)
def test_every_tile_and_run(tiles, M, N, K, rank, adapters, fp8):
    """Every token has the bits that it has in a call of few tokens (smaller tiles, one group of columns to a workgroup: sums are the same for K
    of one part); a sample of tokens against the oracle."""
    print(f"case tiles {tiles} M={M} N={N} K={K} rank={rank} of {adapters} fp8={fp8}", flush=True)
    assert plan_of(M, N, K, rank, adapters) == tiles
    g = torch.Generator().manual_seed(N)
    # requests of some 40 tokens, so that tiles have one, two and more of them, and a part where every token has its own
    ids = torch.randint(-1, adapters, (M // 40 + 2,), generator=g).repeat_interleave(40)[:M]
    ids[M // 3:M // 3 + 150] = torch.randint(-1, adapters + 1, (M,), generator=g)[:len(ids[M // 3:M // 3 + 150])]
    p = problem(M, N, K, rank, adapters, ids, fp8)
    d = {k: None if v is None else v.to(DEV) for k, v in p.items()}
    got = layer_hip.add_adapters(**d)
    rows = ("base", "x", "adapter_ids", "x_scale")
    for lo in range(0, M, 509):
        part = {k: v[lo:lo + 509].clone() if k in rows and v is not None else v for k, v in d.items()}
        assert plan_of(len(part["x"]), N, K, rank, adapters) == (16, 16, 1)
        assert torch.equal(got[lo:lo + 509], layer_hip.add_adapters(**part)), lo
    pick = torch.unique(torch.cat([torch.randint(0, M, (150,), generator=g), torch.tensor([0, M - 1])]))
    check({k: v[pick] if k in rows and v is not None else v for k, v in p.items()}, got[pick.to(DEV)])


@pytest.mark.parametrize("M,N,rank,fp8", [(8200, 1100, 8, False), (4200, 1091, 16, True), (2800, 1090, 24, False), (2100, 1100, 64, True),
                                          (2100, 1091, 128, False), (8200, 6001, 8, False)])
def test_large_tiles_look_at_no_other_request(M, N, rank, fp8):
    """NaN and infinities in another adapter and in another token, in tiles that hold both"""
    K, adapters = 128, 5
    assert plan_of(M, N, K, rank, adapters)[:2] == (64, 32 if rank > 64 else 64)
    p = problem(M, N, K, rank, adapters, "mixed", fp8)
    clean = run(p)
    bad = {k: None if v is None else v.clone() for k, v in p.items()}
    bad["a"][2], bad["b"][2], bad["scale"][2] = float("nan"), float("inf"), float("nan")
    for m in (77, M - 3):
        bad["x"][m:m + 1] = torch.full((1, K), float("nan")).to(p["x"].dtype)
    if fp8:
        bad["x_scale"][M - 9] = float("inf")
    got = run(bad)
    keep = p["adapter_ids"] != 2
    keep[77] = keep[M - 3] = keep[M - 9] = False
    assert torch.equal(got.cpu()[keep], clean.cpu()[keep])
    assert bool(got[(p["adapter_ids"] == 2).to(DEV)].isnan().all())
    for m in (77, M - 3):
        if 0 <= int(p["adapter_ids"][m]) < adapters:
            assert bool(got[m].isnan().all())
