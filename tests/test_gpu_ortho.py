"""orthogonalize against the iteration in 64 bits.

Tolerance, in the norm of the result.  The kernels round S, Q - mu I and X once each per step to fp16 (as S 2^10, (Q - mu I) 2^s, X 2^10; mu = p(mean diagonal of S) below 512 rows, else 0) and the result to its type;
sums are fp32, K * 2^-24 of sum |a b| off at most, which moves some of those roundings to the neighbouring fp16 value and nothing else.  So the
same iteration in 64 bits with the same roundings (`rounded`) has errors of the same size, drawn anew where a sum lay next to a border: the kernels'
error may be at most twice the emulation's, plus half a step of the result's type, plus 2^-11 |X|, one fp16 rounding of X, for matrices so small
that there is nothing to average over."""
import math

import pytest
import torch

import gn_kernels
from gn_kernels import _cabi

pytestmark = pytest.mark.gpu
DEV = "cuda"
COEFFS = (3.4445, -4.7750, 2.0315)
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def iterate(G, steps, co, eps, rounded):
    a, b, c = co
    X = G.double().cpu()
    sq = 32768.0
    while sq * (abs(a) + 2 * abs(b) + 4 * abs(c)) >= 16384:
        sq /= 2

    def q(t, scale):
        return (t * scale).half().double() / scale if rounded else t

    norm = X.norm().item()
    if G.dtype is torch.float32 and norm > 0:        # X_0 of bf16 and fp16 inputs is exact
        X = q(X, 2.0 ** (14 - math.floor(math.log2(norm))))
    X = X / max(norm, eps)
    tall = X.shape[0] > X.shape[1]
    X = X.T if tall else X
    for i in range(steps):
        S = q(X @ X.T, 1024.0)
        s = S.diagonal().mean().item()
        mu = a + b * s + c * s * s if rounded and S.shape[0] < 512 else 0.0
        X = q((a - mu) * torch.eye(S.shape[0], dtype=S.dtype) + b * S + c * S @ S, sq) @ X + mu * X
        X = q(X, 1024.0) if i + 1 < steps else X
    return X.T if tall else X


def reference(G, steps=5, co=COEFFS, eps=1e-7):
    """The result in 64 bits, and the tolerance of the module's comment for the norm of the difference."""
    X = iterate(G, steps, co, eps, False)
    own = (iterate(G, steps, co, eps, True) - X).norm().item()
    return X, 2 * own + (torch.finfo(G.dtype).eps / 2 + 2.0 ** -11) * X.norm().item()


def matrix(m, n, dt, seed=0, kind="momentum"):
    g = torch.Generator().manual_seed(seed)
    if kind == "gauss":
        return torch.randn(m, n, generator=g).to(DT[dt])
    r = max(1, min(m, n) // 8)
    return ((torch.randn(m, r, generator=g) @ torch.randn(r, n, generator=g)) / r ** 0.5 + 0.3 * torch.randn(m, n, generator=g)).mul(1e-3).to(DT[dt])


def compare(got, G, **kw):
    want, tol = reference(G, **kw)
    assert got.dtype is G.dtype and got.shape == G.shape and torch.isfinite(got).all()
    err = (got.double().cpu() - want).norm().item()
    assert err <= tol, f"{err:.3e} off, tolerance {tol:.3e}, norm {want.norm():.3e}"


@pytest.fixture(params=[-1, 1, 5, 6], ids=["auto", "tile128", "tile256w4", "tile64"])
def forced(request):
    L = _cabi.load()
    old = L.gnk_set_gemm_variant(request.param)
    yield
    L.gnk_set_gemm_variant(old)


@pytest.mark.parametrize("m,n", [(1, 1), (1, 70), (70, 1), (2, 3), (16, 16), (127, 129), (128, 128), (129, 127), (255, 300), (300, 257), (333, 999), (999, 333), (640, 384), (520, 900), (1100, 700)])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_shapes(forced, m, n, dt):
    G = matrix(m, n, dt, seed=m + n)
    compare(gn_kernels.orthogonalize(G.to(DEV)), G)


@pytest.mark.parametrize("m,n", [(96, 200), (200, 96), (256, 256)])
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("kind", ["gauss", "momentum"])
def test_types(m, n, dt, kind):
    G = matrix(m, n, dt, kind=kind)
    compare(gn_kernels.orthogonalize(G.to(DEV)), G)


@pytest.mark.parametrize("lead", [(3,), (2, 2), (17,)])
@pytest.mark.parametrize("m,n", [(40, 150), (150, 40)])
def test_stacks(forced, lead, m, n):
    G = torch.stack([matrix(m, n, "bf16", seed=i) * 4.0 ** (i - 4) for i in range(torch.Size(lead).numel())]).view(*lead, m, n)
    got = gn_kernels.orthogonalize(G.to(DEV))
    for x, g in zip(got.view(-1, m, n), G.view(-1, m, n)):
        compare(x, g)


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e-4, 1.0, 1e4, 1e30])
def test_scale_of_the_input(scale):
    """Any magnitude that bf16 holds: the norm is taken in 64 bits, below eps the input is divided by eps."""
    G = (matrix(48, 80, "f32") * 1e3 * scale).bfloat16()
    compare(gn_kernels.orthogonalize(G.to(DEV)), G)


@pytest.mark.parametrize("steps,co", [(1, COEFFS), (2, COEFFS), (10, (2.0, -1.5, 0.5)), (6, (1.875, -1.25, 0.375))])
def test_steps_and_coefficients(steps, co):
    G = matrix(64, 130, "bf16")
    compare(gn_kernels.orthogonalize(G.to(DEV), steps=steps, coefficients=co), G, steps=steps, co=co)


def test_special_values():
    """Zeros stay zeros; a NaN or Inf poisons its own matrix only."""
    G = torch.stack([matrix(30, 50, "bf16", seed=i) for i in range(4)])
    G[0] = 0
    G[1, 3, 4], G[2, 7, 0] = float("nan"), float("inf")
    got = gn_kernels.orthogonalize(G.to(DEV)).cpu()
    assert (got[0] == 0).all() and got[1].isnan().all() and got[2].isnan().all()
    compare(got[3], G[3])


def test_strides():
    base = matrix(70, 140, "bf16")
    for view in (base.T, base[:, ::2], base[3:60, 5:]):
        d = base.to(DEV)
        dv = d.T if view.shape == (140, 70) and view.stride() == (1, 140) else d[:, ::2] if view.stride() == (140, 2) else d[3:60, 5:]
        got = gn_kernels.orthogonalize(dv)
        assert got.is_contiguous()
        compare(got, view.contiguous())


def test_orthogonal_result():
    """What it is for: with the default coefficients every singular value above 1e-2 of the norm ends in [0.6, 1.3], as in 64 bits."""
    G = matrix(120, 200, "bf16", kind="gauss")
    s = torch.linalg.svdvals(gn_kernels.orthogonalize(G.to(DEV)).double().cpu())
    assert s.min() > 0.6 and s.max() < 1.3


def test_graph_and_streams():
    G = torch.stack([matrix(100, 180, "bf16", seed=i) for i in range(2)]).to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = gn_kernels.orthogonalize(G)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gn_kernels.orthogonalize(G)
    for k in range(3):
        G.mul_(1.0 + k).add_(1e-4 * k)
        graph.replay()
        torch.cuda.synchronize()
        want = gn_kernels.orthogonalize(G)
        assert torch.equal(out, want)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs += [gn_kernels.orthogonalize(G) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_large_stack_takes_two_streams():
    """A stack that is split over two streams: against the definition (64 bits, on the device), from another stream while its own next call is on the way,
    and captured (one stream there) with the same bits."""
    B, n = 2, 4096
    G = torch.stack([torch.randn(n, n, generator=torch.Generator(device=DEV).manual_seed(i), device=DEV) for i in range(B)]).bfloat16()
    got = gn_kernels.orthogonalize(G)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        again = [gn_kernels.orthogonalize(G) for _ in range(3)]
    here = gn_kernels.orthogonalize(G)
    torch.cuda.synchronize()
    assert all(torch.equal(x, got) for x in (*again, here))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gn_kernels.orthogonalize(G)
    for k in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, gn_kernels.orthogonalize(G))
        assert torch.equal(out, got)
    X = G[1].double()
    X = X / X.norm()
    for _ in range(5):
        S = X @ X.T
        X = COEFFS[0] * X + COEFFS[1] * (S @ X) + COEFFS[2] * (S @ (S @ X))
    # the fp16 roundings leave 1.2e-3 of the norm at 512 x 512 for this kind of matrix (the emulation of the other tests; it does not grow with the
    # size, every rounding being relative): twice that, and the bf16 result's half step
    assert (got[1].double() - X).norm() <= (2 * 1.2e-3 + 2.0 ** -8) * X.norm()


def test_refusals():
    with pytest.raises(RuntimeError):
        torch.ops.gn_kernels.orthogonalize(torch.zeros(4, 4, dtype=torch.float64, device=DEV), 5, *COEFFS, 1e-7)
    with pytest.raises(RuntimeError):
        torch.ops.gn_kernels.orthogonalize(torch.zeros(4, 4, device=DEV), 0, *COEFFS, 1e-7)
    with pytest.raises(RuntimeError):
        torch.ops.gn_kernels.orthogonalize(torch.zeros(4, 4, device=DEV), 5, 1e6, 0.0, 0.0, 1e-7)
    assert gn_kernels.orthogonalize(torch.zeros(0, 4, 5, device=DEV)).shape == (0, 4, 5)
    assert gn_kernels.orthogonalize(torch.zeros(3, 0, 5, device=DEV)).shape == (3, 0, 5)


# ------------------------------------------------------------------------------------------------ results of more than 8 bits
# Every matrix is kept in two fp16 parts: |v - hi| <= 2^-11 |v|, the rounding of that 2^-22 |v|; a product drops lo lo, 2^-22 of sum |a b|.  Four such
# perturbations per step (S, S^2, Q, X), each stretched by later steps by at most a = 3.4445: 4 (a^5 - 1) / (a - 1) 2^-22 = 1.9e-4 of the norm, 3e-4 with the
# fp32 sums and norms that shrink to 0.7 on the way; plus half a step of the result's type.  (One fp16 part per matrix is off by 1.1e-3.)
def compare_closely(got, G, **kw):
    want = iterate(G, kw.get("steps", 5), kw.get("co", COEFFS), 1e-7, False)
    assert got.dtype is G.dtype and got.shape == G.shape
    err = (got.double().cpu() - want).norm().item() / want.norm().item()
    tol = 3e-4 + torch.finfo(G.dtype).eps / 2
    assert err <= tol, f"{err:.3e} off, tolerance {tol:.3e}"
    return err


@pytest.mark.parametrize("m,n", [(1, 1), (3, 2), (36, 2230), (200, 96), (129, 127), (333, 999), (999, 333), (600, 600), (1100, 700)])
@pytest.mark.parametrize("dt", ["f16", "f32"])
@pytest.mark.parametrize("kind", ["gauss", "momentum"])
def test_more_bits(forced, m, n, dt, kind):
    G = matrix(m, n, dt, seed=m, kind=kind)
    compare_closely(gn_kernels.orthogonalize(G.to(DEV)), G)


@pytest.mark.parametrize("dt", ["f16", "f32"])
@pytest.mark.parametrize("scale", [1e-4, 1.0, 200.0])
def test_more_bits_stacks_scales_steps(dt, scale):
    G = torch.stack([matrix(150, 260, dt, seed=i, kind="gauss") * scale for i in range(5)])
    got = gn_kernels.orthogonalize(G.to(DEV))
    for x, g in zip(got, G):
        compare_closely(x, g)
    for steps in (1, 2, 4):
        compare_closely(gn_kernels.orthogonalize(G[0].to(DEV), steps=steps), G[0], steps=steps)
    compare_closely(gn_kernels.orthogonalize(G[1].to(DEV), coefficients=(2.0, -1.5, 0.5)), G[1], co=(2.0, -1.5, 0.5))


def test_more_bits_large_stack_and_graph():
    """Two streams outside a captured graph, one inside: the same bits."""
    G = torch.stack([matrix(2048, 4224, "f16", seed=i, kind="gauss") for i in range(3)]).to(DEV)
    want = gn_kernels.orthogonalize(G)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gn_kernels.orthogonalize(G)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    X = want[0].float()
    one = torch.linalg.svdvals(X[:, :2048].contiguous())
    assert torch.isfinite(want).all() and one.max() < 1.5
    sub = G[:1, :512, :1024].contiguous()
    compare_closely(gn_kernels.orthogonalize(sub)[0], sub[0].cpu())


def test_more_bits_special_values():
    for dt in (torch.float16, torch.float32):
        G = torch.randn(3, 40, 70, generator=torch.Generator().manual_seed(1)).to(dt)
        G[0, 3, 5], G[1] = float("nan"), 0.0
        got = gn_kernels.orthogonalize(G.to(DEV))
        assert got[0].isnan().all() and (got[1] == 0).all()
        compare_closely(got[2], G[2])


def test_workspace_is_half_for_bf16():
    L, d = _cabi.load(), _cabi.DTYPE_CODE
    need = lambda dt: L.gnk_orthogonalize_workspace_bytes_of(d[dt], 2, 500, 700)  # noqa: E731
    assert need(torch.bfloat16) < 0.51 * need(torch.float32) and need(torch.float16) == need(torch.float32) == L.gnk_orthogonalize_workspace_bytes(2, 500, 700)
    G = matrix(500, 700, "f16").to(DEV)
    out, ws = torch.empty_like(G), torch.empty(L.gnk_orthogonalize_workspace_bytes_of(d[torch.bfloat16], 1, 500, 700), dtype=torch.uint8, device=DEV)
    rc = L.gnk_orthogonalize(G.data_ptr(), d[G.dtype], out.data_ptr(), d[G.dtype], 1, 500, 700, 5, *COEFFS, 1e-7, ws.data_ptr(), ws.numel(), None)
    assert rc == -4 and b"workspace" in L.gnk_last_error()


@pytest.mark.parametrize("m,n", [(64, 4000), (4000, 64), (130, 1600), (100, 1530)])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_long_contractions(forced, m, n, dt):
    """24 steps of 64 and more: four sets of waves."""
    G = matrix(m, n, dt, seed=n)
    (compare if dt == "bf16" else compare_closely)(gn_kernels.orthogonalize(G.to(DEV)), G)


@pytest.mark.parametrize("g_dt,out_dt", [("bf16", "f32"), ("f32", "bf16"), ("f16", "bf16"), ("bf16", "f16")])
def test_result_of_another_type(g_dt, out_dt):
    """The C entry takes the two types apart: the result's decides how many bits the matrices are kept to."""
    L, d = _cabi.load(), _cabi.DTYPE_CODE
    m, n = 150, 310
    G = matrix(m, n, g_dt, seed=2, kind="gauss").to(DEV)
    out = torch.empty(m, n, dtype=DT[out_dt], device=DEV)
    ws = torch.empty(L.gnk_orthogonalize_workspace_bytes_of(d[out.dtype], 1, m, n), dtype=torch.uint8, device=DEV)
    assert L.gnk_orthogonalize(G.data_ptr(), d[G.dtype], out.data_ptr(), d[out.dtype], 1, m, n, 5, *COEFFS, 1e-7, ws.data_ptr(), ws.numel(),
                               torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    want, tol = reference(G.cpu())
    err = (out.double().cpu() - want).norm().item()
    if out_dt != "bf16":
        tol = (3e-4 + torch.finfo(out.dtype).eps / 2) * want.norm().item()
    else:
        tol += torch.finfo(out.dtype).eps / 2 * want.norm().item()
    assert err <= tol
