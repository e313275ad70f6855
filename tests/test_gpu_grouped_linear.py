"""`F.grouped_mm` on a stack of experts' weights kept as a MixedPrecisionLinearWeight: forward and both gradients.

Against the formula: the same quantized operands multiplied in 64 bits.  int8 sums are exact, the conversion and the two scale products are
3 * 2^-24 off, the bf16 result half a step more.  The row quantizers divide by 127 and the group quantizer multiplies by its reciprocal: the
oracle below does the same.
Against differences: sum(y * g) is linear in x and in w apart from the quantization, so central differences of the unquantized sum in 64 bits
are its gradient exactly; a quantized operand is off by at most half a step of its scale, amax / 254 (1 + 2^-20), plus the rounding of the scale
to bf16 (2^-8 of the value), and the errors of a product's sum are bounded term by term."""
import pytest
import torch
import torch.nn.functional as F
from torch import nn

import oracle
from subclasses import MixedPrecisionConfig, MixedPrecisionLinearWeight, convert_mixed_precision_experts
from tests.test_gpu_grouped import offs_of, quant_ref, spans

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(sizes, pad, K, N, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(sum(sizes) + pad, K, generator=g).bfloat16()
    w = (torch.randn(len(sizes), N, K, generator=g) / K ** 0.5).bfloat16()
    gy = (torch.randn(sum(sizes) + pad, N, generator=g) * 1e-2).bfloat16()
    return x, w, gy


def step(x, w, gy, offs, op=F.grouped_mm):
    xd = x.to(DEV).requires_grad_()
    wd = nn.Parameter(MixedPrecisionLinearWeight(w.to(DEV), MixedPrecisionConfig()))
    y = op(xd, wd.transpose(-2, -1), offs=offs)
    y.backward(gy.to(DEV))
    return y.detach(), xd.grad, wd.grad


def formula(x, w, gy, sizes):
    E, N, K = w.shape
    y, gx, gw = torch.zeros(gy.shape, dtype=torch.float64), torch.zeros(x.shape, dtype=torch.float64), torch.zeros(w.shape, dtype=torch.float64)
    xc, xcs = quant_ref(x, sizes)
    gc, gcs = quant_ref(gy, sizes)
    wc, wcs = quant_ref(w.reshape(E * N, K), [N] * E)
    d = lambda q, s: q.double() * s.double()  # noqa: E731
    for e, (lo, hi) in enumerate(spans(sizes)):
        if hi == lo:
            continue
        y[lo:hi] = d(*oracle.quantize_int8(x[lo:hi].contiguous(), dim=1)) @ d(*oracle.quantize_int8(w[e].contiguous(), dim=1)).T
        gx[lo:hi] = d(*oracle.quantize_int8(gy[lo:hi].contiguous(), dim=1)) @ d(wc[e * N:(e + 1) * N], wcs[e])
        gw[e] = d(gc[lo:hi], gcs[e]).T @ d(xc[lo:hi], xcs[e])
    return y, gx, gw


@pytest.mark.parametrize("sizes,pad,K,N", [([5, 0, 130, 1], 3, 64, 48), ([300, 290], 0, 256, 512), ([0, 0], 4, 32, 16), ([7, 9], 0, 33, 21), ([1], 0, 16, 16), ([0, 0], 0, 32, 16), ([3], 2, 48, 1)])
@pytest.mark.parametrize("op", [F.grouped_mm, torch._grouped_mm])
def test_against_the_formula(sizes, pad, K, N, op):
    x, w, gy = make(sizes, pad, K, N)
    for got, want in zip(step(x, w, gy, offs_of(sizes), op), formula(x, w, gy, sizes)):
        got = got._data if isinstance(got, MixedPrecisionLinearWeight) else got
        assert got.dtype is torch.bfloat16 and got.shape == want.shape
        tol = want.abs() * (2.0 ** -8 + 2.0 ** -21)
        assert ((got.cpu().double() - want).abs() <= tol).all()


def test_against_differences():
    sizes, K, N = [40, 0, 25], 48, 32
    x, w, gy = make(sizes, 2, K, N, seed=1)
    _, gx, gw = step(x, w, gy, offs_of(sizes))
    gw = gw._data if isinstance(gw, MixedPrecisionLinearWeight) else gw
    X, W, G = x.double(), w.double(), gy.double()

    def loss(X, W):
        return sum(((X[lo:hi] @ W[e].T) * G[lo:hi]).sum() for e, (lo, hi) in enumerate(spans(sizes)))

    def slack(v, dim):      # |quantized - v|, element by element
        amax = v.abs().amax(dim, keepdim=True)
        return amax / 254 * (1 + 2.0 ** -20) + (v.abs() + amax / 254) * 2.0 ** -8

    h = 2.0 ** -4
    for t, i, e in ((0, 0, 0), (39, 47, 0), (40, 3, 2), (64, 10, 2)):
        D = torch.zeros_like(X)
        D[t, i] = h
        diff = (loss(X + D, W) - loss(X - D, W)) / (2 * h)
        dg, dw = slack(G[t:t + 1], 1)[0], slack(W[e], 0)[:, i]
        tol = (G[t].abs() * dw + W[e, :, i].abs() * dg + dg * dw).sum() + diff.abs() * 2.0 ** -7 + 1e-12
        assert (gx[t, i].cpu().double() - diff).abs() <= tol
    assert (gx[65:] == 0).all()
    for e, n, k in ((0, 0, 0), (0, 31, 47), (2, 5, 9)):
        lo, hi = list(spans(sizes))[e]
        D = torch.zeros_like(W)
        D[e, n, k] = h
        diff = (loss(X, W + D) - loss(X, W - D)) / (2 * h)
        dg, dx = slack(G[lo:hi], 0)[:, n], slack(X[lo:hi], 0)[:, k]
        tol = (G[lo:hi, n].abs() * dx + X[lo:hi, k].abs() * dg + dg * dx).sum() + diff.abs() * 2.0 ** -7 + 1e-12
        assert (gw[e, n, k].cpu().double() - diff).abs() <= tol
    assert (gw[1] == 0).all()


class Experts(nn.Module):
    """Two projections of every expert, as models call them."""

    def __init__(self, E, d, ff):
        super().__init__()
        g = torch.Generator().manual_seed(3)
        self.up = nn.Parameter((torch.randn(E, ff, d, generator=g) / d ** 0.5).bfloat16())
        self.down = nn.Parameter((torch.randn(E, d, ff, generator=g) / ff ** 0.5).bfloat16())
        self.conv = nn.Conv1d(4, 4, 3)

    def forward(self, x, offs):
        h = F.silu(F.grouped_mm(x, self.up.transpose(-2, -1), offs=offs))
        return F.grouped_mm(h, self.down.transpose(-2, -1), offs=offs)


def test_module_of_experts_trains():
    """Converted in place, two steps of an optimizer; only the stacks of experts are wrapped; frozen weights get no gradient."""
    m = Experts(3, 64, 96).to(DEV)
    convert_mixed_precision_experts(m)
    assert isinstance(m.up, MixedPrecisionLinearWeight) and isinstance(m.down, MixedPrecisionLinearWeight)
    assert not isinstance(m.conv.weight, MixedPrecisionLinearWeight)
    opt = torch.optim.SGD([m.up, m.down], lr=1e-2)
    x, offs = torch.randn(50, 64, device=DEV).bfloat16(), offs_of([20, 0, 27])
    for _ in range(2):
        before = m.up._data.clone()
        m(x, offs).float().square().sum().backward()
        assert m.up.grad.shape == m.up.shape and m.down.grad.shape == m.down.shape
        opt.step()
        opt.zero_grad()
        assert not torch.equal(m.up._data, before) and torch.equal(m.up._data[1], before[1])
    m.down.requires_grad_(False)
    m(x, offs).float().sum().backward()
    assert m.down.grad is None and m.up.grad is not None


def test_forward_and_backward_in_a_graph():
    """Captured together while an eager graph of the same leaves is alive; replays with other sizes agree with eager passes."""
    x, w, gy = make([30, 30, 30], 5, 64, 48, seed=4)
    xd, wd, gd = x.to(DEV).requires_grad_(), nn.Parameter(MixedPrecisionLinearWeight(w.to(DEV), MixedPrecisionConfig())), gy.to(DEV)
    offs = offs_of([30, 30, 30])

    def once():
        y = F.grouped_mm(xd, wd.transpose(-2, -1), offs=offs)
        return (y.detach(), *torch.autograd.grad(y, (xd, wd), gd))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for sizes in ([30, 30, 30], [0, 90, 1], [1, 0, 0]):
        offs.copy_(offs_of(sizes))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, once()):
            assert torch.equal(got, want)


def test_stochastic_rounding_is_unbiased():
    """Mean of 64 draws of y against the product of the unquantized operands: a draw of one operand is off by less than a step of its scale
    with mean zero; six standard errors of the mean of all outputs, plus bf16's rounding of the outputs and scales (both signs, 2^-8)."""
    x, w, _ = make([64, 64], 0, 64, 32, seed=5)
    xd, wd = x.to(DEV), MixedPrecisionLinearWeight(w.to(DEV), MixedPrecisionConfig(stochastic_rounding=True))
    torch.manual_seed(0)
    with torch.no_grad():
        ys = torch.stack([F.grouped_mm(xd, wd.transpose(-2, -1), offs=offs_of([64, 64])) for _ in range(64)])
    assert not torch.equal(ys[0], ys[1])
    want = torch.cat([x[:64].double() @ w[0].double().T, x[64:].double() @ w[1].double().T])
    absum = torch.cat([x[:64].double().abs() @ w[0].double().abs().T, x[64:].double().abs() @ w[1].double().abs().T])
    # per output and draw: sum over k of (dx w + x dw + dx dw), |dx| <= amax_x / 127, |dw| <= amax_w / 127
    ax, aw = x.double().abs().amax(1, keepdim=True) / 127, w.double().abs().amax(2) / 127
    wn = torch.cat([w[0].double().norm(dim=1).expand(64, -1), w[1].double().norm(dim=1).expand(64, -1)])
    awr = torch.cat([aw[0].expand(64, -1), aw[1].expand(64, -1)])
    sd = ax * wn + awr * x.double().norm(dim=1, keepdim=True) + ax * awr * 8
    err = (ys.double().mean(0).cpu() - want).abs()
    assert (err <= 6 * sd / 8 + (absum + want.abs()) * 2.0 ** -7).all()


@pytest.mark.parametrize("bad", ["bias", "out_dtype", "config", "first", "dims", "offs", "dtype"])
def test_refusals(bad):
    x, w, _ = make([4, 4], 0, 16, 32)
    x = x.to(DEV)
    cfg = MixedPrecisionConfig(grad_weight=False) if bad == "config" else MixedPrecisionConfig()
    wd = MixedPrecisionLinearWeight(w.to(DEV), cfg)
    offs = offs_of([4, 4])
    with pytest.raises((NotImplementedError, RuntimeError)):
        if bad == "first":
            F.grouped_mm(wd, x, offs=offs)
        elif bad == "dims":
            F.grouped_mm(x, MixedPrecisionLinearWeight(w[0].T.contiguous().to(DEV), cfg), offs=offs)
        elif bad == "offs":
            F.grouped_mm(x, wd.transpose(-2, -1), offs=offs[:1])
        elif bad == "dtype":
            F.grouped_mm(x.float(), wd.transpose(-2, -1), offs=offs)
        else:
            F.grouped_mm(x, wd.transpose(-2, -1), offs=offs, **({"bias": w[:, 0].to(DEV)} if bad == "bias" else {"out_dtype": torch.float32} if bad == "out_dtype" else {}))


@pytest.mark.parametrize("sizes,pad,K,N", [([20000, 100], 3, 64, 96), ([9000], 0, 33, 21), ([4000, 0, 4200], 40, 512, 16)])
def test_many_rows_of_small_experts(sizes, pad, K, N):
    """The weight gradient's contraction is long and its tiles are few (cut into parts, or shared by two sets of waves): the call for both gradients, the op by op
    form and the formula agree, and no gradient that is not asked for is made."""
    from gn_kernels import grouped
    from gn_kernels._lib import lib_ops

    x, w, gy = make(sizes, pad, K, N, seed=4)
    offs = offs_of(sizes)
    xd, wd, gd = x.to(DEV), w.to(DEV).transpose(1, 2), gy.to(DEV)
    gx, gw = lib_ops.grouped_linear_int8_backward(gd, xd, wd, offs, True, True)
    one = grouped.linear_backward(gd, xd, wd, offs, True, True, False)
    assert torch.equal(gx, one[0]) and torch.equal(gw, one[1])
    only_w = lib_ops.grouped_linear_int8_backward(gd, xd, wd, offs, False, True)
    assert only_w[0].shape == (0, K) and torch.equal(only_w[1], gw)
    _, want_x, want_w = formula(x, w, gy, sizes)
    eps = (2.0 ** -8 + 3 * 2.0 ** -24) * (1 + 2.0 ** -8)
    for got, want in ((gx, want_x), (gw, want_w)):
        assert ((got.double().cpu() - want).abs() <= eps * want.abs()).all()
