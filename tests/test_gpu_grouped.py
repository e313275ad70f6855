"""Products grouped by expert and their quantizer against plain 64-bit forms, at the group sizes where they can go wrong: empty groups,
single rows, sizes around a tile, rows of no group, odd feature sizes, every operand order.

Tolerances.  int8: the sum is exact in int32 (|sum| < 2^31 here), its conversion to fp32 is off by at most half a step (2^-24) and so is
each of the two scale multiplies: 3 * 2^-24 relative, plus half a step of the output type; results below the output type's normal range
are not made.  fp8: the matrix core adds at most 16 neighbouring products at a time and cuts each of them off at 2^-13 of the power of two
below the largest one (a product of 2^-13 beside one of 1 is kept, one of 2^-14 is lost; beyond 16 positions both are kept down to 2^-23).
The largest itself loses nothing, so a block of 16 is off by at most 15 * 2^-13 times its largest product, which is at most its sum of |a b|:
15 * 2^-13 * sum |a b| over all blocks.  The blocks are added in fp32, at most one step (2^-23 of a partial sum <= sum |a b|) off each, for
fewer than K blocks: K * 2^-22 covers it.  The value that is rounded at the end is off by that much, so the half step grows by (1 + 2^-8)."""
import pytest
import torch

import gn_kernels
import oracle
from gn_kernels import _cabi

pytestmark = pytest.mark.gpu
DEV = "cuda"
OUT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}

# group sizes, rows behind the last group
SIZES = {
    "one_row": ([1], 0),
    "around_tiles": ([127, 128, 129, 1], 0),
    "empties": ([0, 5, 0, 0, 64, 0], 3),
    "all_empty": ([0, 0], 7),
    "no_rows": ([0, 0, 0], 0),
    "one_big": ([300, 0, 1, 1], 130),
    "many": ([(7 * i) % 5 for i in range(150)], 2),
}


def offs_of(sizes):
    return torch.tensor(sizes, dtype=torch.int32).cumsum(0).to(torch.int32).to(DEV)


def spans(sizes):
    lo = 0
    for n in sizes:
        yield lo, lo + n
        lo += n


def make8(shape, dt, g):
    if dt == "int8":
        return torch.randint(-128, 128, shape, generator=g, dtype=torch.int8)
    return (torch.randn(shape, generator=g) * 2).to(F8[dt])


def scales(shape, out, g):
    return (torch.rand(shape, generator=g) * 0.02 + 0.01).to(OUT[out])


def place(t, order, pitch_pad=0):
    """t on the device with its dims lying in memory in `order` (slowest first); pitch_pad: extra elements behind each innermost row."""
    moved = t.permute(*order).contiguous()
    if pitch_pad:
        wide = torch.zeros((*moved.shape[:-1], moved.shape[-1] + pitch_pad), dtype=moved.dtype)
        wide[..., : moved.shape[-1]].view(torch.int8).copy_(moved.view(torch.int8))
        moved = wide.to(DEV)[..., : moved.shape[-1]]
    else:
        moved = moved.to(DEV)
    return moved.permute(*[order.index(i) for i in range(t.ndim)])


def check(got, want, absum, dt, out, K):
    """want: 64-bit result; absum: the same with absolute values (the scaled sum of |a b|)."""
    assert got.dtype is OUT[out] and got.shape == want.shape
    eps = torch.finfo(OUT[out]).eps / 2 + 3 * 2.0 ** -24
    tol = want.abs() * eps * (1 + 2.0 ** -8)
    if dt != "int8":
        tol = tol + absum * (15 * 2.0 ** -13 + K * 2.0 ** -22) * (1 + 2.0 ** -8)
    err = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), f"worst {(err / tol.clamp_min(1e-300)).max():.3g} of the tolerance"


def rows_ref(A, B, sA, sB, sizes):
    want = torch.zeros(A.shape[0], B.shape[2], dtype=torch.float64)
    absum = want.clone()
    for e, (lo, hi) in enumerate(spans(sizes)):
        s = sA[lo:hi].double() * sB[e].double()
        want[lo:hi] = (A[lo:hi].float().double() @ B[e].float().double()) * s
        absum[lo:hi] = (A[lo:hi].float().double().abs() @ B[e].float().double().abs()) * s
    return want, absum


def depth_ref(A, B, sA, sB, sizes):
    want, absum = [], []
    for e, (lo, hi) in enumerate(spans(sizes)):
        s = sA[e].double() * sB[e].double()
        want.append((A[:, lo:hi].float().double() @ B[lo:hi].float().double()) * s)
        absum.append((A[:, lo:hi].float().double().abs() @ B[lo:hi].float().double().abs()) * s)
    return torch.stack(want), torch.stack(absum)


def run_rows(sizes, pad, K, N, dt, out, order=(0, 2, 1), a_order=(0, 1), pitch=0, scalar=False, dt_b=None):
    g = torch.Generator().manual_seed(K * 7 + N + len(sizes))
    T, E = sum(sizes) + pad, len(sizes)
    A, B = make8((T, K), dt, g), make8((E, K, N), dt_b or dt, g)
    sA, sB = scales((T, 1), out, g), scales((E, 1, 1 if scalar else N), out, g)
    got = gn_kernels.grouped_scaled_mm(place(A, a_order, pitch), place(B, order, pitch), sA.to(DEV), sB.to(DEV), offs_of(sizes))
    want, absum = rows_ref(A, B, sA, sB, sizes)
    check(got, want, absum, dt, out, K)
    assert (got[sum(sizes):] == 0).all()


def run_depth(sizes, pad, M, N, dt, out, a_order=(1, 0), b_order=(0, 1), pitch=0, scalar=False, dt_b=None):
    g = torch.Generator().manual_seed(M * 5 + N + len(sizes))
    T, E = sum(sizes) + pad, len(sizes)
    A, B = make8((M, T), dt, g), make8((T, N), dt_b or dt, g)
    sA, sB = scales((E, M, 1), out, g), scales((E, 1, 1 if scalar else N), out, g)
    got = gn_kernels.grouped_scaled_mm(place(A, a_order, pitch), place(B, b_order, pitch), sA.to(DEV), sB.to(DEV), offs_of(sizes))
    want, absum = depth_ref(A, B, sA, sB, sizes)
    check(got, want, absum, dt, out, max(sizes, default=0))


@pytest.mark.parametrize("name", list(SIZES))
@pytest.mark.parametrize("order", ["nk", "kn"])
@pytest.mark.parametrize("dt", ["int8", "e4m3"])
def test_rows_group_sizes(name, order, dt):
    sizes, pad = SIZES[name]
    run_rows(sizes, pad, 192, 144, dt, "bf16", (0, 2, 1) if order == "nk" else (0, 1, 2))


@pytest.mark.parametrize("name", list(SIZES))
@pytest.mark.parametrize("dt", ["int8", "e4m3"])
def test_depth_group_sizes(name, dt):
    sizes, pad = SIZES[name]
    run_depth(sizes, pad, 144, 272, dt, "bf16")


@pytest.mark.parametrize("K,N", [(1, 1), (16, 16), (17, 15), (128, 130), (333, 100), (256, 256), (512, 264), (1024, 72), (100, 4)])
@pytest.mark.parametrize("order", ["nk", "kn"])
def test_rows_feature_sizes(K, N, order):
    run_rows([3, 130, 0, 61], 2, K, N, "int8", "bf16", (0, 2, 1) if order == "nk" else (0, 1, 2))


@pytest.mark.parametrize("M,N", [(1, 1), (16, 16), (17, 15), (130, 128), (333, 100), (256, 512), (264, 72), (100, 4)])
def test_depth_feature_sizes(M, N):
    run_depth([3, 300, 0, 61], 2, M, N, "int8", "bf16")


@pytest.mark.parametrize("K", [256, 512, 768, 2048])
@pytest.mark.parametrize("order", ["nk", "kn"])
@pytest.mark.parametrize("dt", ["int8", "e4m3"])
def test_rows_large_tiles(K, order, dt):
    """Enough rows per group for the 256-row tiles, edges inside a tile on both sides."""
    run_rows([700, 1, 256, 0, 513], 5, K, 528, dt, "bf16", (0, 2, 1) if order == "nk" else (0, 1, 2))


@pytest.mark.parametrize("sizes", [[700, 1, 256, 0, 513], [2048, 100], [1, 255, 257, 64, 63, 65]])
@pytest.mark.parametrize("dt", ["int8", "e4m3"])
def test_depth_large_tiles(sizes, dt):
    run_depth(sizes, 5, 528, 272, dt, "bf16")


@pytest.mark.parametrize("out", list(OUT))
@pytest.mark.parametrize("scalar", [False, True])
def test_output_types(out, scalar):
    run_rows([40, 0, 97], 3, 256, 136, "int8", out, scalar=scalar)
    run_depth([40, 0, 97], 3, 136, 72, "int8", out, scalar=scalar)


@pytest.mark.parametrize("a", list(F8))
@pytest.mark.parametrize("b", list(F8))
def test_fp8_formats_mix(a, b):
    run_rows([40, 0, 97], 3, 256, 136, a, "bf16", dt_b=b)
    run_depth([40, 0, 97], 3, 136, 72, a, "bf16", dt_b=b)


@pytest.mark.parametrize("order", [(0, 1, 2), (0, 2, 1), (1, 0, 2), (2, 0, 1), (1, 2, 0), (2, 1, 0)])
@pytest.mark.parametrize("a_order", [(0, 1), (1, 0)])
@pytest.mark.parametrize("pitch", [0, 16, 5])
def test_rows_strides(order, a_order, pitch):
    run_rows([5, 33, 0, 90], 4, 64, 48, "int8", "bf16", order, a_order, pitch)


@pytest.mark.parametrize("a_order", [(0, 1), (1, 0)])
@pytest.mark.parametrize("b_order", [(0, 1), (1, 0)])
@pytest.mark.parametrize("pitch", [0, 16, 5])
def test_depth_strides(a_order, b_order, pitch):
    run_depth([5, 33, 0, 90], 4, 64, 48, "int8", "bf16", a_order, b_order, pitch)


def test_int32_sums_are_exact():
    """Sums beyond 2^24: fp32 outputs equal (f32(sum) * sA) * sB bit for bit."""
    A = torch.full((70, 4096), -128, dtype=torch.int8)
    A[:, ::3] = 127
    B = torch.full((2, 4096, 32), 127, dtype=torch.int8)
    B[1] = -128
    one = torch.ones(70, 1)
    got = gn_kernels.grouped_scaled_mm(A.to(DEV), B.to(DEV), one.to(DEV), torch.full((2, 1, 32), 0.1).to(DEV), offs_of([30, 40]))
    s = torch.stack([A[0].long() @ B[e, :, 0].long() for e in range(2)])
    want = torch.cat([s[:1].float().expand(30), s[1:].float().expand(40)])[:, None] * torch.full((1, 32), 0.1)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("shift", [-5, 3, 1000])
def test_ends_that_do_not_fit_stay_inside(shift):
    """Ends beyond T or below zero are clamped: the call returns, and rows of groups that do fit are right."""
    g = torch.Generator().manual_seed(0)
    A, B = make8((64, 64), "int8", g), make8((2, 64, 32), "int8", g)
    sA, sB = scales((64, 1), "f32", g), scales((2, 1, 32), "f32", g)
    offs = torch.tensor([32, 64 + shift], dtype=torch.int32, device=DEV)
    got = gn_kernels.grouped_scaled_mm(A.to(DEV), B.to(DEV), sA.to(DEV), sB.to(DEV), offs)
    want, _ = rows_ref(A, B, sA, sB, [32, min(max(32 + shift, 0), 32)])
    torch.testing.assert_close(got.cpu(), want.float(), rtol=2.0 ** -22, atol=0)
    x = torch.randn(64, 40, generator=g).to(DEV)
    q, s = gn_kernels.quantize_int8_grouped(x, offs)
    wq, ws = quant_ref(x[:32].cpu(), [32])
    assert torch.equal(q[:32].cpu(), wq) and torch.equal(s[0].cpu(), ws[0])


# ends that decrease, with the sizes that they stand for: a value below an earlier one counts as that one, negative ones as 0, ones beyond T as T
DECREASING = {
    "one_step_back": ([300, 120, 700], 1100),
    "back_and_forth": ([2500, 0] * 50, 2500),                       # read as pairs of ends, every second group would hold all rows
    "back_over_a_wave": ([1] * 62 + [2300, 40] + [30] * 70 + [2400], 2500),
    "below_and_beyond": ([-7, 50, -2 ** 31, 2 ** 31 - 1, 3], 2200),
}


def sizes_of(ends, T):
    lo, sizes = 0, []
    for e in ends:
        hi = max(lo, min(max(e, 0), T))
        sizes.append(hi - lo)
        lo = hi
    return sizes


@pytest.mark.parametrize("name", list(DECREASING))
@pytest.mark.parametrize("variant", [0, 1, 5, 6])
def test_ends_that_decrease(name, variant):
    ends, T = DECREASING[name]
    sizes, E, g = sizes_of(ends, T), len(ends), torch.Generator().manual_seed(4)
    assert sum(sizes) <= T and min(sizes) >= 0
    offs = torch.tensor(ends, dtype=torch.int32, device=DEV)
    A, B, D = make8((T, 256), "int8", g), make8((1, 256, 48), "int8", g), make8((T, 32), "int8", g)
    sA, sB, sR = scales((T, 1), "f32", g), scales((E, 1, 48), "f32", g), scales((E, 256, 1), "f32", g)
    sD = scales((E, 1, 32), "f32", g)
    L = _cabi.load()
    L.gnk_set_gemm_variant(variant)
    try:
        rows = gn_kernels.grouped_scaled_mm(A.to(DEV), B.to(DEV).expand(E, 256, 48), sA.to(DEV), sB.to(DEV), offs)
        depth = gn_kernels.grouped_scaled_mm(A.to(DEV).t(), D.to(DEV), sR.to(DEV), sD.to(DEV), offs)
        torch.cuda.synchronize()
    finally:
        L.gnk_set_gemm_variant(-1)
    check(rows, *rows_ref(A, B.expand(E, 256, 48), sA, sB, sizes), "int8", "f32", 256)
    assert (rows[sum(sizes):] == 0).all()
    check(depth, *depth_ref(A.t(), D, sR, sD, sizes), "int8", "f32", T)


@pytest.mark.parametrize("name", list(DECREASING))
@pytest.mark.parametrize("T_extra", [-1000, 0, 3000])               # one launch, two, and pieces of 256 rows for the maxima
def test_quantize_ends_that_decrease(name, T_extra):
    ends, T = DECREASING[name]
    T += T_extra
    if T <= 0:
        T = 500
    sizes = sizes_of(ends, T)
    x = torch.randn(T, 40, generator=torch.Generator().manual_seed(5))
    q, s = gn_kernels.quantize_int8_grouped(x.to(DEV), torch.tensor(ends, dtype=torch.int32, device=DEV))
    wq, ws = quant_ref(x, sizes)
    assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)


# ------------------------------------------------------------------------------------------------ quantizer
def quant_ref(x, sizes):
    """Group by group on the host, bit for bit: scale = amax * fl(1 / 127) in fp32, q = clip(rne(x / max(scale, eps))); a NaN quotient gives
    0, as the dense quantizer does."""
    q = torch.zeros(x.shape, dtype=torch.int8)
    s = torch.zeros(len(sizes), 1, x.shape[1], dtype=x.dtype)
    for e, (lo, hi) in enumerate(spans(sizes)):
        if hi > lo:
            xf = x[lo:hi].float()
            scale = xf.abs().amax(0, keepdim=True) * torch.tensor(1.0 / 127.0, dtype=torch.float32)
            q[lo:hi] = (xf / scale.clamp_min(1e-12)).round().nan_to_num(0.0).clamp(-128, 127).to(torch.int8)
            s[e] = scale.to(x.dtype)
    return q, s


def test_quantize_grouped_is_the_dense_quantizer_up_to_its_scale():
    """Against quantize_int8 group by group: the fp32 scales differ by at most 1.5 steps, so x / scale by at most 127 * 3 * 2^-24 relative
    plus a rounding: values differ by one, and only within 2^-15 of a border."""
    sizes = [1000, 0, 24]
    x = torch.randn(1024, 256, generator=torch.Generator().manual_seed(9))
    q, s = gn_kernels.quantize_int8_grouped(x.to(DEV), offs_of(sizes))
    for e, (lo, hi) in enumerate(spans(sizes)):
        if hi > lo:
            wq, ws = oracle.quantize_int8(x[lo:hi].contiguous(), dim=0)
            assert ((s[e].cpu() - ws).abs() <= ws * 1.5 * 2.0 ** -23).all()
            off = (q[lo:hi].cpu().int() - wq.int()).abs()
            v = x[lo:hi].double() / ws.double()
            assert off.max() <= 1 and ((v - v.floor() - 0.5).abs()[off == 1] <= 2.0 ** -15).all()


@pytest.mark.parametrize("name", list(SIZES))
@pytest.mark.parametrize("C", [1, 8, 100, 264, 333])
@pytest.mark.parametrize("dt", list(OUT))
def test_quantize_grouped(name, C, dt):
    sizes, pad = SIZES[name]
    x = torch.randn(sum(sizes) + pad, C, generator=torch.Generator().manual_seed(C)).to(OUT[dt])
    q, s = gn_kernels.quantize_int8_grouped(x.to(DEV), offs_of(sizes))
    wq, ws = quant_ref(x, sizes)
    assert torch.equal(q.cpu(), wq)
    assert torch.equal(s.cpu().view(torch.int8), ws.view(torch.int8))


@pytest.mark.parametrize("sizes,pad", [([5000, 0, 129, 1, 3000], 9), ([1] * 70 + [4097], 0), ([2048], 0), ([2000, 48], 1), ([1500, 0, 300], 5)])
def test_quantize_grouped_long(sizes, pad):
    """Groups of several partial rows."""
    x = torch.randn(sum(sizes) + pad, 72, generator=torch.Generator().manual_seed(1)).bfloat16()
    q, s = gn_kernels.quantize_int8_grouped(x.to(DEV), offs_of(sizes))
    wq, ws = quant_ref(x, sizes)
    assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)


@pytest.mark.parametrize("view", ["transposed", "padded", "offset"])
def test_quantize_grouped_strides(view):
    sizes = [33, 0, 70]
    base = torch.randn(110, 64, generator=torch.Generator().manual_seed(2)).bfloat16()
    x = {"transposed": torch.randn(64, 110, generator=torch.Generator().manual_seed(2)).bfloat16().T, "padded": base[:, :40], "offset": base[:, 3:43]}[view]
    xd = {"transposed": lambda: x.T.contiguous().to(DEV).T, "padded": lambda: base.to(DEV)[:, :40], "offset": lambda: base.to(DEV)[:, 3:43]}[view]()
    q, s = gn_kernels.quantize_int8_grouped(xd, offs_of(sizes))
    wq, ws = quant_ref(x.contiguous(), sizes)
    assert q.is_contiguous() and torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)


def test_quantize_grouped_special_values():
    """NaN and Inf poison their own (group, column) only; zero columns keep scale 0; tiny columns meet eps."""
    x = torch.randn(30, 16, generator=torch.Generator().manual_seed(3))
    x[4, 0], x[14, 1], x[:10, 2], x[10:20, 3] = float("nan"), float("inf"), 0.0, 1e-20
    sizes = [10, 10, 10]
    q, s = gn_kernels.quantize_int8_grouped(x.to(DEV), offs_of(sizes))
    wq, ws = quant_ref(x, sizes)
    assert torch.equal(q.cpu(), wq)
    assert torch.equal(s.cpu().isnan(), ws.isnan()) and torch.equal(s.cpu().nan_to_num(7.0), ws.nan_to_num(7.0))


@pytest.mark.parametrize("C", [64, 33])
def test_quantize_grouped_stochastic(C):
    """floor(x / scale + u): within one step of x / scale, unbiased over many draws, another draw with another seed, the same with the same."""
    sizes = [40, 0, 23]
    x = torch.randn(66, C, generator=torch.Generator().manual_seed(4)).to(DEV)
    torch.manual_seed(11)
    draws = [gn_kernels.quantize_int8_grouped(x, offs_of(sizes), True) for _ in range(64)]
    torch.manual_seed(11)
    again = gn_kernels.quantize_int8_grouped(x, offs_of(sizes), True)
    assert torch.equal(draws[0][0], again[0]) and not torch.equal(draws[0][0], draws[1][0])
    s = draws[0][1].double()
    v = torch.zeros(66, C, dtype=torch.float64, device=DEV)
    for e, (lo, hi) in enumerate(spans(sizes)):
        v[lo:hi] = x[lo:hi].double() / s[e]
    for q, sc in draws:
        assert torch.equal(sc, draws[0][1])
        assert ((q.double() - v).abs() <= 1 + 1e-4).all()
    # a value's draws have variance <= 1/4: the mean over 64 of them and 63 * C values is off by at most 6 sigma = 6 * 0.5 / sqrt(64 * 63 * C)
    mean = torch.stack([q.double() - v for q, _ in draws])[:, :63].mean()
    assert abs(mean.item()) <= 6 * 0.5 / (64 * 63 * C) ** 0.5 + 1e-4


# ------------------------------------------------------------------------------------------------ streams, graphs
def test_graph_replay_with_other_sizes():
    """Captured once, replayed with other group sizes in the same buffers, eager work and synchronizations between."""
    g = torch.Generator().manual_seed(5)
    T, K, N, E = 200, 256, 136, 4
    A, B = make8((T, K), "int8", g).to(DEV), make8((E, N, K), "int8", g).to(DEV).transpose(1, 2)
    G = make8((T, N), "int8", g).to(DEV)
    x = torch.randn(T, N, generator=g).bfloat16().to(DEV)
    sA, sB, sM = scales((T, 1), "bf16", g).to(DEV), scales((E, 1, N), "bf16", g).to(DEV), scales((E, K, 1), "bf16", g).to(DEV)
    offs = offs_of([50, 50, 50, 50])

    def calls():
        return (gn_kernels.grouped_scaled_mm(A, B, sA, sB, offs), gn_kernels.grouped_scaled_mm(A.T, G, sM, sB, offs), *gn_kernels.quantize_int8_grouped(x, offs))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    for sizes in ([50, 50, 50, 50], [0, 200, 0, 0], [1, 2, 3, 4], [0, 0, 0, 0], [130, 1, 0, 69]):
        offs.copy_(offs_of(sizes))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, calls()):
            assert torch.equal(got, want), sizes


def test_other_stream():
    g = torch.Generator().manual_seed(6)
    A, B = make8((64, 100), "int8", g).to(DEV), make8((2, 100, 30), "int8", g).to(DEV)       # sizes that need the operand copies
    sA, sB = scales((64, 1), "bf16", g).to(DEV), scales((2, 1, 30), "bf16", g).to(DEV)
    offs = offs_of([20, 40])
    want = gn_kernels.grouped_scaled_mm(A, B, sA, sB, offs)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append([gn_kernels.grouped_scaled_mm(A, B, sA, sB, offs) for _ in range(8)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for out in outs for o in out)


@pytest.mark.parametrize("dt", ["int8", "e4m3"])
def test_nothing_to_multiply(dt):
    """No groups, no rows, no features to sum over: zeros of the right shape (scaled sums of nothing)."""
    g = torch.Generator().manual_seed(7)
    none, two = torch.zeros(0, dtype=torch.int32, device=DEV), offs_of([3, 2])
    sc = lambda *s: scales(s, "bf16", g).to(DEV)  # noqa: E731
    e8 = lambda *s: make8(s, dt, g).to(DEV)  # noqa: E731
    for y in (gn_kernels.grouped_scaled_mm(e8(5, 17), e8(0, 17, 24), sc(5, 1), sc(0, 1, 24), none),
              gn_kernels.grouped_scaled_mm(e8(5, 0), e8(2, 0, 24), sc(5, 1), sc(2, 1, 24), two)):
        assert y.shape == (5, 24) and (y == 0).all()
    assert gn_kernels.grouped_scaled_mm(e8(0, 16), e8(2, 16, 24), sc(0, 1), sc(2, 1, 24), offs_of([0, 0])).shape == (0, 24)
    assert gn_kernels.grouped_scaled_mm(e8(5, 16), e8(2, 16, 0), sc(5, 1), sc(2, 1, 0), two).shape == (5, 0)
    y = gn_kernels.grouped_scaled_mm(e8(32, 0), e8(0, 24), sc(2, 32, 1), sc(2, 1, 24), offs_of([0, 0]))
    assert y.shape == (2, 32, 24) and (y == 0).all()
    assert gn_kernels.grouped_scaled_mm(e8(32, 5), e8(5, 24), sc(0, 32, 1), sc(0, 1, 24), none).shape == (0, 32, 24)
    q, s = gn_kernels.quantize_int8_grouped(torch.ones(5, 24, device=DEV), none)
    assert s.shape == (0, 1, 24) and (q == 0).all()
    q, s = gn_kernels.quantize_int8_grouped(torch.ones(0, 24, device=DEV), offs_of([0, 0]))
    assert q.shape == (0, 24) and (s == 0).all()


def test_one_weight_for_all_groups():
    """B expanded over the groups: read in place."""
    g = torch.Generator().manual_seed(8)
    A, B = make8((50, 64), "int8", g), make8((1, 64, 32), "int8", g)
    sA, sB = scales((50, 1), "bf16", g), scales((3, 1, 32), "bf16", g)
    got = gn_kernels.grouped_scaled_mm(A.to(DEV), B.to(DEV).expand(3, 64, 32), sA.to(DEV), sB.to(DEV), offs_of([20, 0, 30]))
    want, absum = rows_ref(A, B.expand(3, 64, 32), sA, sB, [20, 0, 30])
    check(got, want, absum, "int8", "bf16", 64)


def test_refusals_on_device():
    i8 = lambda *s: torch.zeros(*s, dtype=torch.int8, device=DEV)  # noqa: E731
    sc = lambda *s: torch.ones(*s, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    with pytest.raises(RuntimeError):       # offs on the host
        gn_kernels.grouped_scaled_mm(i8(8, 16), i8(2, 16, 16), sc(8, 1), sc(2, 1, 16), torch.tensor([4, 8], dtype=torch.int32))
    with pytest.raises(RuntimeError):
        gn_kernels.quantize_int8_grouped(sc(8, 16), torch.tensor([4, 8], dtype=torch.int32))
    with pytest.raises(RuntimeError):       # a type the quantizer does not take
        gn_kernels.quantize_int8_grouped(torch.zeros(8, 16, dtype=torch.float64, device=DEV), offs_of([4, 4]))
    L = _cabi.load()
    rc = L.gnk_grouped_scaled_mm_rows(i8(8, 17).data_ptr(), _cabi.I8, i8(2, 17, 16).data_ptr(), _cabi.I8, sc(8, 16).data_ptr(), _cabi.BF16, sc(8).data_ptr(),
                                      sc(2, 16).data_ptr(), _cabi.BF16, 0, offs_of([4, 4]).data_ptr(), 8, 2, 16, 17, 17, 1, 272, 16, 1, None, 0, None)
    assert rc == -4 and b"workspace" in L.gnk_last_error()      # K = 17 needs operand copies


# ------------------------------------------------------------------------------------------------ tile variants
@pytest.fixture(params=[1, 5, 6, 0], ids=["tile128", "tile256w4", "tile64", "tile192"])
def forced(request):
    L = _cabi.load()
    old = L.gnk_set_gemm_variant(request.param)
    yield
    L.gnk_set_gemm_variant(old)


@pytest.mark.parametrize("name", list(SIZES))
@pytest.mark.parametrize("dt", ["int8", "e4m3", "e5m2"])
def test_variants_group_sizes(forced, name, dt):
    sizes, pad = SIZES[name]
    for order in ((0, 2, 1), (0, 1, 2)):
        run_rows(sizes, pad, 512, 272, dt, "bf16", order)
    run_depth(sizes, pad, 272, 528, dt, "bf16")


@pytest.mark.parametrize("sizes", [[255, 256, 257], [1, 2, 63, 64, 65], [1023, 1, 1025], [511, 0, 513]])
def test_variants_depth_ends(forced, sizes):
    """Ends on, before and behind every step of the contraction; what lies behind a group must not leak into it."""
    for M, N in ((256, 256), (16, 32), (100, 300)):
        run_depth(sizes, 3, M, N, "int8", "f32")
        run_depth(sizes, 3, M, N, "e4m3", "bf16")


@pytest.mark.parametrize("sizes", [[191, 192, 193], [95, 96, 97, 1], [385, 0, 383]])
def test_variants_row_edges(forced, sizes):
    """Group sizes around the halves and multiples of a 192-row tile."""
    for K, N in ((256, 256), (768, 300), (1024, 16)):
        for order in ((0, 2, 1), (0, 1, 2)):
            run_rows(sizes, 3, K, N, "int8", "f32", order)


@pytest.mark.parametrize("out", list(OUT))
@pytest.mark.parametrize("N", [256, 260, 255])
def test_variants_outputs(forced, out, N):
    run_rows([300, 0, 270], 3, 256, N, "int8", out)
    run_depth([300, 0, 270], 3, N, 264, "int8", out)
    run_depth([300, 0, 270], 3, 264, N, "int8", out, scalar=True)


# ------------------------------------------------------------------------------------------------ contractions cut into parts
LONG = {
    "one": ([5000], 3),
    "short_ones_beside_it": ([0, 4100, 0, 1, 900], 130),
    "just_over_a_step": ([1025, 0, 1023], 0),
    "longest": ([30000], 0),
}


@pytest.mark.parametrize("name", list(LONG))
@pytest.mark.parametrize("M,N", [(144, 272), (17, 15), (64, 64), (300, 130)])
@pytest.mark.parametrize("dt", ["int8", "e4m3", "e5m2"])
@pytest.mark.parametrize("variant", [-1, 1, 5])
def test_depth_in_parts(name, M, N, dt, variant):
    sizes, pad = LONG[name]
    L = _cabi.load()
    L.gnk_set_gemm_variant(variant)
    try:
        if name in ("one", "longest"):                             # the others are split or not as the sizes say
            assert L.gnk_grouped_scaled_mm_depth_split_bytes(sum(sizes) + pad, len(sizes), M, N) >= 2 * 4 * len(sizes) * M * N
        run_depth(sizes, pad, M, N, dt, "bf16")
    finally:
        L.gnk_set_gemm_variant(-1)


@pytest.fixture
def tiles_of_128():
    L = _cabi.load()
    L.gnk_set_gemm_variant(1)
    yield
    L.gnk_set_gemm_variant(-1)


@pytest.mark.parametrize("out", list(OUT))
@pytest.mark.parametrize("scalar", [False, True])
@pytest.mark.parametrize("N", [48, 46])
def test_depth_in_parts_output_types(tiles_of_128, out, scalar, N):
    run_depth([3000, 0, 2500], 1, 40, N, "int8", out, scalar=scalar)
    run_depth([3000, 0, 2500], 1, 40, N, "e5m2", out, scalar=scalar)


def test_depth_in_parts_strides(tiles_of_128):
    for a_order, b_order, pitch in (((0, 1), (0, 1), 0), ((1, 0), (1, 0), 0), ((1, 0), (0, 1), 3), ((0, 1), (1, 0), 16)):
        run_depth([4000, 100], 5, 60, 33, "int8", "bf16", a_order=a_order, b_order=b_order, pitch=pitch)


def test_depth_with_less_room_for_its_parts(tiles_of_128):
    """The C entry with room for all parts, for half of them, for one and for none, and with the slab behind copied operands: the same int8 result."""
    L, g = _cabi.load(), torch.Generator().manual_seed(3)
    sizes, M, N = [6000, 500], 64, 96
    T, E = sum(sizes), len(sizes)
    A, B = make8((T, M), "int8", g).to(DEV), make8((T, N), "int8", g).to(DEV)
    sA, sB, offs = scales((E, M, 1), "f32", g).to(DEV), scales((E, 1, N), "f32", g).to(DEV), offs_of(sizes)
    room = L.gnk_grouped_scaled_mm_depth_split_bytes(T, E, M, N)
    assert room > 0
    want = None
    for n in (0, E * M * N * 4, room // 2, room, room + 4096):
        C, ws = torch.empty(E, M, N, device=DEV), torch.empty(max(n, 1), dtype=torch.uint8, device=DEV)
        rc = L.gnk_grouped_scaled_mm_depth(A.data_ptr(), _cabi.I8, B.data_ptr(), _cabi.I8, C.data_ptr(), _cabi.DTYPE_CODE[torch.float32], sA.data_ptr(), sB.data_ptr(),
                                           _cabi.DTYPE_CODE[torch.float32], 0, offs.data_ptr(), T, E, M, N, 1, M, N, 1, ws.data_ptr() if n else None, n,
                                           torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        want = C if want is None else want
        assert torch.equal(C, want)
    check(want, *depth_ref(A.cpu().t(), B.cpu(), sA.cpu(), sB.cpu(), sizes), "int8", "f32", T)


def test_depth_in_parts_repeats_and_replays(tiles_of_128):
    """fp8 sums depend on their order: equal calls give equal bits, on other streams and in a graph replayed with other sizes too."""
    g = torch.Generator().manual_seed(6)
    T, M, N = 8000, 96, 80
    A, B = make8((T, M), "e4m3", g).to(DEV), make8((T, N), "e4m3", g).to(DEV)
    sA, sB = scales((2, M, 1), "bf16", g).to(DEV), scales((2, 1, N), "bf16", g).to(DEV)
    offs = offs_of([5000, 2000])
    call = lambda: gn_kernels.grouped_scaled_mm(A.t(), B, sA, sB, offs)  # noqa: E731
    want = call()
    torch.cuda.synchronize()
    for s in [torch.cuda.Stream() for _ in range(2)]:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs = [call() for _ in range(5)]
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for sizes in ([5000, 2000], [0, 8000], [10, 0], [5000, 2000]):
        offs.copy_(offs_of(sizes))
        graph.replay()
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        check(eager, *depth_ref(A.cpu().t(), B.cpu(), sA.cpu(), sB.cpu(), sizes), "e4m3", "bf16", T)
