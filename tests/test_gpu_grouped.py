"""The block-scaled product of sorted tokens with their experts' weights, on the GPU, expert by expert against the float64 oracle with
the tolerance of the ungrouped product (test_gpu_layer.py)."""
import ctypes

import pytest
import torch

import alpha_moe
from alpha_moe_python import layer_hip
from alpha_moe_python.prep import block_quant_fp8, per_token_group_quant_fp8
from oracle import layer_oracle as L
from test_gpu_layer import DEV, assert_mm

pytestmark = pytest.mark.gpu


def quantised(w):
    """codes and scales of [N, K]; the last block of rows may be short"""
    N, K = w.shape
    q, scale = block_quant_fp8(torch.nn.functional.pad(w, (0, 0, 0, -N % 128)))
    return q[:N].contiguous(), scale


def problem(counts, tail, N, K, seed):
    g = torch.Generator().manual_seed(seed)
    E, R = len(counts), sum(counts) + tail
    x, xs = per_token_group_quant_fp8(torch.randn((R, K), generator=g) * (0.2 + torch.rand((R, 1), generator=g)), 128)
    w, ws = zip(*(quantised(torch.randn((N, K), generator=g) * (0.05 + 0.1 * e / E)) for e in range(E)))
    offsets = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    return x, xs, offsets, torch.stack(w), torch.stack(ws)


def check(x, xs, offsets, w, ws, out):
    assert out.dtype == torch.bfloat16 and out.shape == (x.shape[0], w.shape[1])
    out = out.cpu()
    for e, (lo, hi) in enumerate(zip(offsets.tolist(), offsets.tolist()[1:])):
        if lo < hi:
            assert_mm(out[lo:hi], x[lo:hi], xs[lo:hi], w[e], ws[e])
    assert not bool(out[int(offsets[-1]):].any())


def run(*args):
    return layer_hip.grouped_block_scaled_mm(*(t.to(DEV) for t in args))


ONES = [1, 0, 1, 1, 0, 0, 1, 2]
CASES = [([1], 0, 1, 128), ([3], 0, 130, 256), ([0, 0, 5, 0], 0, 17, 384), (ONES, 0, 512, 1024), (ONES, 3, 100, 640), ([0] * 9, 7, 129, 128),
         ([8, 9, 16, 17, 1], 0, 96, 384), ([30, 0, 0, 0, 0, 0, 0, 0, 2], 1, 33, 256), ([5, 6, 7, 11, 12], 2, 257, 512),
         ([15, 16, 17, 32, 33], 0, 64, 896), ([20, 25, 1, 0, 40], 9, 131, 256), ([64, 65, 1, 30], 0, 300, 384), ([63, 0, 0, 128], 70, 127, 128),
         ([127, 128, 129, 3], 0, 385, 256), ([300, 1, 0, 77], 5, 128, 640), ([256, 257, 255], 0, 511, 384), ([513, 10], 300, 770, 128),
         ([1000, 3, 0, 2000], 1, 260, 256), ([1] * 65 + [0] * 70 + [2] * 65, 0, 40, 256), ([2, 7] * 150, 11, 24, 128), ([0] * 500 + [40], 0, 48, 256),
         ([2] * 3, 0, 300, 65536), ([40, 100], 0, 130, 16384), ([200, 300], 0, 264, 16384), ([4000, 1, 4191], 0, 130, 128)]


@pytest.mark.parametrize("counts,tail,N,K", CASES)
def test_grouped(counts, tail, N, K):
    print(f"case grouped {counts[:8]} of {len(counts)} tail={tail} N={N} K={K}", flush=True)
    args = problem(counts, tail, N, K, N + K)
    out = run(*args)
    check(*args, out)
    assert torch.equal(out, run(*args))


@pytest.mark.parametrize("spread", [1, 4, 9, 20, 40, 100, 300])
def test_experts_that_have_more_or_fewer_rows_than_the_average(spread):
    """counts from 0 to several times the average, whatever tile the average has chosen"""
    g = torch.Generator().manual_seed(spread)
    counts = (torch.rand(17, generator=g) ** 2 * 3 * spread).int().tolist() + [0, 3 * spread]
    args = problem(counts, spread, 200, 384, spread)
    check(*args, run(*args))


@pytest.mark.parametrize("counts", [[1, 2, 0, 1], [9, 10, 3], [20, 30, 1], [60, 3], [150, 20], [300, 0]])
@pytest.mark.parametrize("N", [2050, 4096, 9000])
def test_many_columns(counts, N):
    """more groups of columns than a few, in every kind of tile"""
    print(f"case many columns {counts} N={N}", flush=True)
    args = problem(counts, 1, N, 128, N)
    check(*args, run(*args))


def test_one_expert_is_the_ungrouped_product():
    for M, N, K in ((5, 300, 256), (70, 130, 384), (600, 512, 256)):
        x, xs, offsets, w, ws = problem([M], 0, N, K, M)
        assert_mm(run(x, xs, offsets, w, ws), x, xs, w[0], ws[0])


def test_no_rows():
    x, xs, offsets, w, ws = problem([1, 2], 0, 10, 128, 1)
    assert run(x[:0], xs[:0], torch.zeros(3, dtype=torch.int32), w, ws).shape == (0, 10)


def test_rows_of_other_experts_are_never_looked_at():
    """NaN codes and scales in an expert's rows and weights stay in that expert's results"""
    counts, N, K = [3, 9, 0, 20, 70, 5], 140, 256
    x, xs, offsets, w, ws = problem(counts, 4, N, K, 3)
    clean = run(x, xs, offsets, w, ws).cpu()
    for e in range(len(counts)):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        bad_x, bad_s, bad_w, bad_ws = x.clone(), xs.clone(), w.clone(), ws.clone()
        bad_x.view(torch.uint8)[lo:hi] = 0x7f
        bad_s[lo:hi] = float("inf")
        bad_w.view(torch.uint8)[e] = 0x7f
        bad_ws[e] = float("nan")
        got = run(bad_x, bad_s, offsets, bad_w, bad_ws).cpu()
        keep = torch.ones(len(x), dtype=torch.bool)
        keep[lo:hi] = False
        assert torch.equal(got[keep], clean[keep]) and bool(got[lo:hi].isnan().all())


@pytest.mark.parametrize("mean", [2, 10, 20, 40, 100, 200])
def test_nothing_beside_the_rows_and_offsets_of_any_kind(mean):
    """bytes behind the result stay; offsets that do not ascend, or reach past the rows, read and write nothing outside the arrays"""
    E, N, K = 5, 77, 256
    counts = [mean, 0, 2 * mean, mean, mean]
    x, xs, offsets, w, ws = problem(counts, 3, N, K, 9)
    R = len(x)
    xd, xsd, wd, wsd = (t.to(DEV) for t in (x, xs, w, ws))
    for off in (offsets, torch.tensor([5, 1, 0, R + 1000, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32), torch.full((6,), -7, dtype=torch.int32),
                torch.full((6,), 2 ** 31 - 1, dtype=torch.int32), torch.tensor([0, 3, 2, 4, 4, R], dtype=torch.int32)):
        out = torch.full((R * N + 4096,), 7.0, dtype=torch.bfloat16, device=DEV)
        od = off.to(DEV)
        rc = alpha_moe.c_abi.alpha_moe_grouped_block_scaled_mm(xd.data_ptr(), xsd.data_ptr(), od.data_ptr(), wd.data_ptr(), wsd.data_ptr(),
                                                               out.data_ptr(), R, N, K, E, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert rc == 0 and bool((out[R * N:] == 7).all())
        if off is offsets:
            check(x, xs, offsets, w, ws, out[:R * N].view(R, N))


def test_refusals():
    x, xs, offsets, w, ws = (t.to(DEV) for t in problem([2, 2], 0, 130, 256, 1))
    H = layer_hip.grouped_block_scaled_mm
    for call, message in ((lambda: H(x.float(), xs, offsets, w, ws), "dtype"), (lambda: H(x, xs, offsets.long(), w, ws), "dtype"),
                          (lambda: H(x, xs, offsets[:2], w, ws), r"\[E \+ 1\]"), (lambda: H(x, xs[:3], offsets, w, ws), "x_scale"),
                          (lambda: H(x, xs, offsets, w, ws[:, :1].contiguous()), "w_scale"), (lambda: H(x, xs, offsets, w[0], ws[0]), r"\[E, N, K\]"),
                          (lambda: H(x, xs, offsets, w.transpose(1, 2), ws), "contiguous"), (lambda: H(x, xs, offsets.cpu(), w, ws), "must be on"),
                          (lambda: H(x[:, :128].contiguous(), xs, offsets, w, ws), "K of x"), (lambda: H(x[:, :64].contiguous(), xs, offsets, w, ws), "128"),
                          (lambda: H(x, xs.requires_grad_(), offsets, w, ws), "requires a gradient")):
        with pytest.raises(RuntimeError, match=message):
            call()


def test_replays_with_other_groups():
    """captured once, replayed with other offsets, between eager calls"""
    counts, N, K = [7, 1, 30, 0, 12], 200, 384
    args = [t.to(DEV) for t in problem(counts, 2, N, K, 4)]
    layer_hip.grouped_block_scaled_mm(*args)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        out = layer_hip.grouped_block_scaled_mm(*args)
    for c in ([50, 0, 0, 0, 2], [0, 0, 0, 0, 0], [10, 10, 10, 10, 10], counts):
        args[2].copy_(torch.tensor([0] + c).cumsum(0).to(torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, layer_hip.grouped_block_scaled_mm(*args))
        check(*(t.cpu() for t in args), out)


@pytest.mark.parametrize("rest", [0, 1, 127, 128, 129, 255])
def test_last_tiles_of_any_length(rest):
    """many rows of few K blocks take the largest tile, whose last one of an expert may be a half one"""
    counts = [256 * k + rest for k in (0, 1, 3)] + [0, 700, 40]
    args = problem(counts, 5, 300, 256, rest)
    check(*args, run(*args))


def test_offsets_past_32_bits():
    """weights of more than 4 GiB and results of more than 4 GiB: small integers, exact"""
    E, N, K = 130, 4096, 8192 + 128
    w = torch.zeros((E, N, K), device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn)
    assert w.numel() > 2 ** 32
    for e in (0, 100, 129):
        w.view(torch.uint8)[e, N - 3, K - 2] = torch.tensor([2.0]).to(torch.float8_e4m3fn).view(torch.uint8).item()
    counts = torch.zeros(E, dtype=torch.int64)
    counts[0], counts[100], counts[129] = 3, 20, 2
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).to(torch.int32).to(DEV)
    x = torch.ones((25, K), device=DEV).to(torch.float8_e4m3fn)
    out = layer_hip.grouped_block_scaled_mm(x, torch.ones((25, K // 128), device=DEV), offsets, w, torch.ones((E, N // 128, K // 128), device=DEV))
    want = torch.zeros((25, N))
    want[:, N - 3] = 2.0
    assert torch.equal(out.cpu().float(), want)
    del w, out
    R, N, K = 40000, 65536, 128                      # (5 GiB of results)
    x = torch.ones((R, K), device=DEV).to(torch.float8_e4m3fn)
    w = torch.zeros((2, N, K), device=DEV).to(torch.float8_e4m3fn)
    w[1, N - 1, 7] = 3.0
    out = layer_hip.grouped_block_scaled_mm(x, torch.ones((R, 1), device=DEV), torch.tensor([0, 17, R - 2], dtype=torch.int32, device=DEV), w,
                                            torch.ones((2, N // 128, 1), device=DEV))
    assert out.numel() * 2 > 2 ** 32
    last = out[:, N - 1]
    assert bool((last[17:R - 2] == 3).all()) and not bool(last[:17].any()) and not bool(last[R - 2:].any())
    assert int(out[-5000:].count_nonzero()) == 4998


@pytest.mark.parametrize("N,K", [(7168, 128), (5000, 256), (7169, 384), (4096, 512), (3000, 640), (2048, 768), (2040, 1152)])
def test_lists_of_tiles(N, K):
    """more tiles of 256 x 256 than units, whole and half ones, K blocks and places of scales of every remainder: a sample of each expert's
    rows against the oracle, all of them against the ungrouped product"""
    g = torch.Generator().manual_seed(N)
    counts = [700, 0, 129, 128, 256, 257, 1, 2000, 385, 1024, 640, 0, 511, 1300, 896, 2500]
    tail = 70
    print(f"case lists N={N} K={K}", flush=True)
    args = problem(counts, tail, N, K, K)
    out = run(*args)
    x, xs, offsets, w, ws = args
    for e, (lo, hi) in enumerate(zip(offsets.tolist(), offsets.tolist()[1:])):
        if lo == hi:
            continue
        pick = torch.unique(torch.cat([torch.randint(lo, hi, (6,), generator=g), torch.tensor([lo, hi - 1])]))
        assert_mm(out.cpu()[pick], x[pick], xs[pick], w[e], ws[e])
        alone = layer_hip.block_scaled_mm(*(t.to(DEV) for t in (x[lo:hi], xs[lo:hi], w[e], ws[e])))
        size = alone.float().abs().max().item()
        assert (out[lo:hi].float() - alone.float()).abs().max().item() <= 2.0 ** -7 * size
    assert not bool(out[int(offsets[-1]):].any())
    assert torch.equal(out, run(*args))


def test_more_tiles_than_lists_of_the_units_hold():
    """above 15360 tiles there are more workgroups than units"""
    counts, tail, N, K = [90000, 0, 47000, 100, 300], 3, 8192, 128
    g = torch.Generator(device=DEV).manual_seed(3)
    R, E = sum(counts) + tail, len(counts)
    x = torch.randn((R, K), generator=g, device=DEV).to(torch.float8_e4m3fn)
    xs, ws = (0.5 + torch.rand(shape, generator=g, device=DEV) for shape in ((R, 1), (E, N // 128, 1)))
    w = torch.randn((E, N, K), generator=g, device=DEV).to(torch.float8_e4m3fn)
    offsets = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    out = layer_hip.grouped_block_scaled_mm(x, xs, offsets.to(DEV), w, ws)
    for e, (lo, hi) in enumerate(zip(offsets.tolist(), offsets.tolist()[1:])):
        if lo < hi:      # one K block: a sum of its own, the same in every tile
            assert torch.equal(out[lo:hi], layer_hip.block_scaled_mm(x[lo:hi], xs[lo:hi], w[e], ws[e])), e
    assert not bool(out[R - tail:].any())


# tile (columns, tokens), counts, rows behind them, N, K: an expert of more than eight tiles of tokens, experts of none and of one row, more than
# one group of columns to each XCD's run, and a number of columns that no tile divides
TILES = [
    ((16, 8), [1, 0, 1, 1], 1, 1000, 640), ((32, 16), [150, 0, 1, 0, 0, 0, 3] + [1, 0] * 30, 5, 2049, 1664),
    ((32, 16), [40, 0, 90, 1, 33, 16, 17, 23], 10, 142, 6528),
    ((128, 64), [560, 0, 1, 64], 30, 2049, 640), ((128, 64), [3, 700, 0, 65], 0, 4099, 1152), ((128, 64), [1030] + [40, 0, 1] * 6, 70, 2562, 1152),
    ((256, 128), [1100, 0, 1] + [30, 128, 0, 129, 20, 5, 8] * 2 + [70] + [0] * 6, 190, 2049, 896),
    ((256, 128), [10, 1200] + [0, 1, 30] * 4 + [129, 200], 130, 2561, 1024), ((256, 128), [0, 2, 1050, 0, 64, 33, 1, 20, 3, 7, 9, 1], 10, 4099, 1024),
    ((256, 256), [2500, 0, 1, 128, 129, 300], 50, 2309, 384)]


@pytest.mark.parametrize("tile,counts,tail,N,K", TILES)
def test_every_tile(tile, counts, tail, N, K):
    print(f"case tile {tile} {counts[:8]} of {len(counts)} tail={tail} N={N} K={K}", flush=True)
    plan = (ctypes.c_int * 2)()
    assert alpha_moe.c_abi.alpha_moe_grouped_mm_plan(sum(counts) + tail, N, K, len(counts), plan) == 0 and tuple(plan) == tile
    args = problem(counts, tail, N, K, N + K)
    out = run(*args)
    check(*args, out)
    assert torch.equal(out, run(*args))
