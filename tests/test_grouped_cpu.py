"""The grouped products without a GPU: wrapper checks, Meta implementations, the C ABI's refusals, workspace sizes."""
import pytest
import torch
import torch.nn.functional as F
from torch import nn

import gn_kernels
from gn_kernels import _cabi
from subclasses import MixedPrecisionConfig, MixedPrecisionLinearWeight, convert_mixed_precision_experts


def i8(*s):
    return torch.zeros(*s, dtype=torch.int8, device="meta")


def sc(*s, dt=torch.bfloat16):
    return torch.zeros(*s, dtype=dt, device="meta")


def offs(n, dt=torch.int32):
    return torch.zeros(n, dtype=dt, device="meta")


def test_shapes_and_dtypes():
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        y = gn_kernels.grouped_scaled_mm(i8(10, 16), i8(3, 16, 24), sc(10, 1, dt=dt), sc(3, 1, 24, dt=dt), offs(3))
        assert y.shape == (10, 24) and y.dtype is dt
        y = gn_kernels.grouped_scaled_mm(i8(16, 10), i8(10, 24), sc(3, 16, 1, dt=dt), sc(3, 1, 1, dt=dt), offs(3))
        assert y.shape == (3, 16, 24) and y.dtype is dt
        q, s = gn_kernels.quantize_int8_grouped(sc(10, 24, dt=dt), offs(3))
        assert q.shape == (10, 24) and q.dtype is torch.int8 and s.shape == (3, 1, 24) and s.dtype is dt


@pytest.mark.parametrize("call", [
    lambda: gn_kernels.grouped_scaled_mm(sc(10, 16), i8(3, 16, 24), sc(10, 1), sc(3, 1, 24), offs(3)),                                # A is no 8-bit type
    lambda: gn_kernels.grouped_scaled_mm(i8(10, 16), i8(3, 16, 24).to(torch.float8_e4m3fn), sc(10, 1), sc(3, 1, 24), offs(3)),       # int8 with fp8
    lambda: gn_kernels.grouped_scaled_mm(i8(10, 16), i8(3, 16, 24), sc(10, 1), sc(3, 1, 24, dt=torch.float32), offs(3)),             # scale types differ
    lambda: gn_kernels.grouped_scaled_mm(i8(10, 17), i8(3, 16, 24), sc(10, 1), sc(3, 1, 24), offs(3)),                                # inner sizes
    lambda: gn_kernels.grouped_scaled_mm(i8(10, 16), i8(3, 16, 24), sc(10, 1), sc(3, 1, 24), offs(2)),                                # group counts
    lambda: gn_kernels.grouped_scaled_mm(i8(10, 16), i8(3, 16, 24), sc(9, 1), sc(3, 1, 24), offs(3)),                                 # row scales
    lambda: gn_kernels.grouped_scaled_mm(i8(10, 16), i8(3, 16, 24), sc(10, 1), sc(3, 24), offs(3)),                                   # column scales
    lambda: gn_kernels.grouped_scaled_mm(i8(10, 16), i8(3, 16, 24), sc(10, 2)[:, :1], sc(3, 1, 24), offs(3)),                         # not contiguous
    lambda: gn_kernels.grouped_scaled_mm(i8(10, 16), i8(3, 16, 24), sc(10, 1), sc(3, 1, 24), offs(3, torch.int64)),                   # offs type
    lambda: gn_kernels.grouped_scaled_mm(i8(10, 16), i8(3, 16, 24), sc(10, 1), sc(3, 1, 24), offs(6)[::2]),                           # offs strides
    lambda: gn_kernels.grouped_scaled_mm(i8(16, 10), i8(9, 24), sc(3, 16, 1), sc(3, 1, 24), offs(3)),                                 # contraction sizes
    lambda: gn_kernels.grouped_scaled_mm(i8(16, 10), i8(10, 24), sc(16, 1), sc(3, 1, 24), offs(3)),                                   # scale per group
    lambda: gn_kernels.quantize_int8_grouped(sc(4, 10, 24), offs(3)),
    lambda: gn_kernels.quantize_int8_grouped(sc(10, 24), offs(3, torch.int64)),
])
def test_refusals(call):
    with pytest.raises(AssertionError):
        call()


def test_cabi_refuses_before_it_touches_a_gpu():
    L = _cabi.load()
    rows = lambda *, a=_cabi.I8, b=_cabi.I8, out=_cabi.BF16, s=_cabi.BF16, T=4, E=2, N=16, K=16: L.gnk_grouped_scaled_mm_rows(  # noqa: E731
        None, a, None, b, None, out, None, None, s, 0, None, T, E, N, K, 16, 1, 256, 16, 1, None, 0, None)
    assert rows() == -1 and b"null pointer" in L.gnk_last_error()
    assert rows(b=_cabi.E4M3) == -1 and b"both int8 or both fp8" in L.gnk_last_error()
    assert rows(out=_cabi.I32) == -1 and rows(s=_cabi.I8) == -1 and rows(T=-1) == -1
    assert rows(T=1 << 31) == -2 and rows(E=1 << 20) == -2 and rows(K=(1 << 22) + 1) == -2
    assert rows(T=0) == 0 and rows(N=0) == 0                       # nothing to do
    depth = lambda *, a=_cabi.I8, T=4, E=2, M=16, N=16: L.gnk_grouped_scaled_mm_depth(  # noqa: E731
        None, a, None, _cabi.I8, None, _cabi.BF16, None, None, _cabi.BF16, 0, None, T, E, M, N, 1, 16, 16, 1, None, 0, None)
    assert depth() == -1 and depth(a=_cabi.E5M2) == -1 and depth(M=-2) == -1
    assert depth(E=0) == 0 and depth(M=0) == 0
    quant = lambda *, dt=_cabi.BF16, T=4, E=2, C=16: L.gnk_quantize_int8_grouped(None, dt, None, T, E, C, 16, 1, None, None, 1e-12, 0, 0, 0, None, 0, None)  # noqa: E731
    assert quant() == -1 and quant(dt=_cabi.I8) == -1 and quant(T=-1) == -1 and quant(T=1 << 31) == -2
    assert quant(C=0) == 0 and quant(T=0, E=0) == 0


def test_workspace_is_only_for_operands_that_cannot_be_read_in_place():
    L = _cabi.load()
    a, b = 1 << 20, 1 << 21                                        # 16-byte aligned addresses, never read
    rows = lambda K, N, sat, sbe, sbk, sbn, a=a: L.gnk_grouped_scaled_mm_rows_workspace_bytes(a, b, 100, 3, N, K, sat, 1, sbe, sbk, sbn)  # noqa: E731
    assert rows(64, 48, 64, 48 * 64, 1, 64) == 0                   # (E, N, K) weights
    assert rows(64, 48, 64, 48 * 64, 48, 1) == 0                   # (E, K, N) weights
    assert rows(64, 48, 80, 48 * 64, 48, 1) == 0                   # padded rows
    assert rows(64, 48, 65, 48 * 64, 48, 1) == 100 * 64            # odd pitch of A
    assert rows(64, 48, 64, 48 * 64, 48, 1, a=a + 8) == 100 * 64   # unaligned A
    assert rows(65, 48, 65, 48 * 65, 1, 65) == 100 * 80 + 3 * 48 * 80
    assert rows(64, 50, 64, 50 * 64, 50, 1) == 3 * 64 * 64         # (E, K, N) with N = 50: rows of 64
    depth = lambda M, N, sat, sbt: L.gnk_grouped_scaled_mm_depth_workspace_bytes(a, b, 100, M, N, 1, sat, sbt, 1)  # noqa: E731
    assert depth(64, 48, 64, 48) == 0 and depth(64, 50, 64, 50) == 100 * 64 and depth(63, 48, 64, 48) == 100 * 64
    assert L.gnk_quantize_int8_grouped_workspace_bytes(4000, 4, 64) == (4000 // 128 + 5) * 64 * 4
    assert L.gnk_quantize_int8_grouped_workspace_bytes(1000, 4, 64) == 0           # small calls keep their maxima on chip


# ------------------------------------------------------------------------------------------------ F.grouped_mm on a mixed-precision weight
@pytest.fixture(scope="module")
def cpu_ops():
    """The expert projection's two ops on host tensors, unquantized: what is tested is how autograd and the subclass call them."""
    impl = torch.library.Library("gn_kernels", "IMPL")

    def groups(offs):
        ends = offs.tolist()
        return enumerate(zip([0] + ends[:-1], ends))

    def forward(x, w, offs):
        y = x.new_zeros(x.shape[0], w.shape[2])
        for e, (lo, hi) in groups(offs):
            y[lo:hi] = x[lo:hi] @ w[e]
        return y

    def backward(gy, x, w, offs, need_x, need_w):
        gx, gw = x.new_zeros(x.shape if need_x else (0, x.shape[1])), x.new_zeros((w.shape[0] if need_w else 0, w.shape[2], w.shape[1]))
        for e, (lo, hi) in groups(offs):
            if need_x:
                gx[lo:hi] = gy[lo:hi] @ w[e].T
            if need_w:
                gw[e] = gy[lo:hi].T @ x[lo:hi]
        return gx, gw

    impl.impl("grouped_linear_int8", forward, "CPU")
    impl.impl("grouped_linear_int8_backward", backward, "CPU")
    yield


class Experts(nn.Module):
    def __init__(self, dt=torch.float64):
        super().__init__()
        g = torch.Generator().manual_seed(0)
        self.up = nn.Parameter(torch.randn(3, 12, 8, generator=g, dtype=dt))
        self.down = nn.Parameter(torch.randn(3, 8, 12, generator=g, dtype=dt))
        self.conv = nn.Conv1d(2, 2, 3)
        self.norm = nn.LayerNorm(8)

    def forward(self, x, offs):
        return F.grouped_mm(torch.tanh(F.grouped_mm(x, self.up.transpose(-2, -1), offs=offs)), self.down.transpose(1, 2), offs=offs)


def plain_experts(m, x, sizes):
    up, down = (getattr(p, "_data", p) for p in (m.up, m.down))
    return torch.cat([torch.tanh(part @ up[e].T) @ down[e].T for e, part in enumerate(x.split(sizes))])


def test_conversion_wraps_stacks_of_experts_only():
    m = convert_mixed_precision_experts(Experts())
    assert isinstance(m.up, MixedPrecisionLinearWeight) and isinstance(m.down, MixedPrecisionLinearWeight)
    assert isinstance(m.up, nn.Parameter) or m.up.requires_grad
    assert not isinstance(m.conv.weight, MixedPrecisionLinearWeight) and not isinstance(m.norm.weight, MixedPrecisionLinearWeight)


@pytest.mark.parametrize("op", [F.grouped_mm, torch._grouped_mm])
def test_autograd_of_one_projection(cpu_ops, op):
    """Gradients against the formula and against central differences (exact for a product up to rounding: 2^-52 / h)."""
    g = torch.Generator().manual_seed(1)
    sizes, offs = [3, 0, 4], torch.tensor([3, 3, 7], dtype=torch.int32)
    x, w = torch.randn(7, 8, generator=g, dtype=torch.float64), torch.randn(3, 12, 8, generator=g, dtype=torch.float64)
    gy = torch.randn(7, 12, generator=g, dtype=torch.float64)
    xp, wp = x.clone().requires_grad_(), nn.Parameter(MixedPrecisionLinearWeight(w.clone(), MixedPrecisionConfig()))
    y = op(xp, wp.transpose(-2, -1), offs=offs)
    y.backward(gy)
    gw = wp.grad._data if isinstance(wp.grad, MixedPrecisionLinearWeight) else wp.grad
    want = torch.cat([p @ w[e].T for e, p in enumerate(x.split(sizes))])
    torch.testing.assert_close(y.detach(), want, rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(xp.grad, torch.cat([p @ w[e] for e, p in enumerate(gy.split(sizes))]), rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(gw, torch.stack([a.T @ b for a, b in zip(gy.split(sizes), x.split(sizes))]), rtol=1e-12, atol=1e-12)

    def loss(x, w):
        return sum(((p @ w[e].T) * q).sum() for e, (p, q) in enumerate(zip(x.split(sizes), gy.split(sizes))))

    h = 2.0 ** -10
    for i, j in ((0, 0), (6, 7), (3, 2)):
        d = torch.zeros_like(x)
        d[i, j] = h
        assert abs((loss(x + d, w) - loss(x - d, w)) / (2 * h) - xp.grad[i, j]) < 1e-9
    d = torch.zeros_like(w)
    d[2, 5, 1] = h
    assert abs((loss(x, w + d) - loss(x, w - d)) / (2 * h) - gw[2, 5, 1]) < 1e-9 and (gw[1] == 0).all()


@pytest.mark.parametrize("compiled", [False, True])
@pytest.mark.parametrize("frozen", ["none", "up", "x"])
def test_module_of_experts(cpu_ops, compiled, frozen):
    """Eager and traced (the ops stay opaque nodes): outputs and every gradient that is asked for, none that is not."""
    m = convert_mixed_precision_experts(Experts())
    sizes, offs = [2, 0, 3], torch.tensor([2, 2, 5], dtype=torch.int32)
    x = torch.randn(5, 8, generator=torch.Generator().manual_seed(2), dtype=torch.float64).requires_grad_(frozen != "x")
    if frozen == "up":
        m.up.requires_grad_(False)
    call = torch.compile(m, backend="aot_eager") if compiled else m
    y = call(x, offs)
    y.square().sum().backward()
    ref = Experts()
    xr = x.detach().clone().requires_grad_()
    yr = plain_experts(ref, xr, sizes)
    yr.square().sum().backward()
    torch.testing.assert_close(y.detach(), yr.detach(), rtol=1e-12, atol=1e-12)
    for p, r in ((m.up, ref.up), (m.down, ref.down), (x, xr)):
        if not p.requires_grad:
            assert p.grad is None
            continue
        grad = p.grad._data if isinstance(p.grad, MixedPrecisionLinearWeight) else p.grad
        torch.testing.assert_close(grad, r.grad, rtol=1e-10, atol=1e-12)


def test_every_way_to_transpose_a_stack_stays_wrapped():
    w = MixedPrecisionLinearWeight(torch.randn(3, 4, 6), MixedPrecisionConfig())
    for v in (w.transpose(-2, -1), w.transpose(1, 2), w.mT):
        assert isinstance(v, MixedPrecisionLinearWeight) and v.shape == (3, 6, 4) and torch.equal(v._data, w._data.transpose(1, 2))


def test_two_dimensional_weights_are_viewed_as_before():
    w = MixedPrecisionLinearWeight(torch.randn(4, 6), MixedPrecisionConfig())
    assert isinstance(w.t(), MixedPrecisionLinearWeight) and not isinstance(w.transpose(0, 1), MixedPrecisionLinearWeight)
    assert isinstance(w.detach(), MixedPrecisionLinearWeight)


@pytest.mark.parametrize("kwargs,error", [
    (dict(bias=torch.zeros(3, 12)), NotImplementedError),
    (dict(out_dtype=torch.float32), NotImplementedError),
    (dict(offs=None), NotImplementedError),
    (dict(offs=torch.tensor([1, 2], dtype=torch.int32)), RuntimeError),
])
def test_grouped_mm_refusals(kwargs, error):
    w = MixedPrecisionLinearWeight(torch.zeros(3, 12, 8, dtype=torch.bfloat16), MixedPrecisionConfig())
    args = dict(offs=torch.tensor([1, 2, 4], dtype=torch.int32)) | kwargs
    with pytest.raises(error):
        F.grouped_mm(torch.zeros(4, 8, dtype=torch.bfloat16), w.transpose(-2, -1), **args)
    with pytest.raises(NotImplementedError):
        part = MixedPrecisionLinearWeight(torch.zeros(3, 12, 8, dtype=torch.bfloat16), MixedPrecisionConfig(grad_input=False))
        F.grouped_mm(torch.zeros(4, 8, dtype=torch.bfloat16), part.transpose(-2, -1), offs=torch.tensor([1, 2, 4], dtype=torch.int32))


def test_int8_sums_that_may_not_fit_32_bits():
    L = _cabi.load()
    rows = lambda dt, K: L.gnk_grouped_scaled_mm_rows(None, dt, None, dt, None, _cabi.BF16, None, None, _cabi.BF16, 0, None, 4, 2, 16, K, K, 1, 16 * K, 1, K, None, 0, None)  # noqa: E731
    assert rows(_cabi.I8, 131072) == -2 and b"32 bits" in L.gnk_last_error()
    assert rows(_cabi.I8, 131071) == -1 and rows(_cabi.E4M3, 131072) == -1         # null pointers: the size is taken
    # room for the pieces of a group of more than 130816 rows, whatever else a call asks for
    assert L.gnk_grouped_scaled_mm_depth_split_bytes(130817, 64, 2048, 2048) >= 2 * 2048 * 2048 * 4
    assert L.gnk_grouped_scaled_mm_depth_split_bytes(3 * 130817, 64, 2048, 2048) >= 6 * 2048 * 2048 * 4


@pytest.mark.parametrize("compiled", [False, True])
@pytest.mark.parametrize("turn", [lambda w: w.permute(0, 2, 1), lambda w: w.movedim(1, 2), lambda w: w.permute(0, -1, -2), lambda w: w.swapaxes(1, 2), lambda w: w.mT,
                                  lambda w: torch.permute(w, (0, 2, 1))], ids=["permute", "movedim", "negative", "swapaxes", "mT", "function"])
def test_other_ways_to_transpose_a_stack_reach_the_operator(cpu_ops, turn, compiled):
    """A permuted stack is the mixed-precision weight still: F.grouped_mm on it is the operator's (which is registered for host tensors here; plain grouped_mm in
    float64 does not exist), forward and backward."""
    g = torch.Generator().manual_seed(6)
    x, w, gy = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((5, 8), (2, 12, 8), (5, 12)))
    offs = torch.tensor([2, 5], dtype=torch.int32)
    wp = nn.Parameter(MixedPrecisionLinearWeight(w, MixedPrecisionConfig()))
    assert isinstance(turn(wp), MixedPrecisionLinearWeight) and turn(wp).shape == (2, 8, 12) and torch.equal(turn(wp)._data, w.mT)

    def call(x, wp, offs):
        return F.grouped_mm(x, turn(wp), offs=offs)

    y = (torch.compile(call, backend="aot_eager") if compiled else call)(x, wp, offs)
    y.backward(gy)
    gw = getattr(wp.grad, "_data", wp.grad)
    torch.testing.assert_close(y.detach(), torch.cat([x[:2] @ w[0].T, x[2:] @ w[1].T]), rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(gw, torch.stack([gy[:2].T @ x[:2], gy[2:].T @ x[2:]]), rtol=1e-12, atol=1e-12)


def test_ends_by_position(cpu_ops):
    """torch._grouped_mm takes the ends as its third positional argument."""
    g = torch.Generator().manual_seed(7)
    x, w = torch.randn(5, 8, generator=g, dtype=torch.float64), torch.randn(2, 12, 8, generator=g, dtype=torch.float64)
    wp, offs = MixedPrecisionLinearWeight(w, MixedPrecisionConfig()), torch.tensor([2, 5], dtype=torch.int32)
    y = torch._grouped_mm(x, wp.mT, offs)
    torch.testing.assert_close(y, torch.cat([x[:2] @ w[0].T, x[2:] @ w[1].T]), rtol=1e-12, atol=1e-12)
    for bad in (lambda: torch._grouped_mm(x, wp.mT, offs, torch.zeros(2, 12)), lambda: torch._grouped_mm(x, wp.mT, None), lambda: torch._grouped_mm(x, wp.mT, offs, None, torch.float32)):
        with pytest.raises(NotImplementedError):
            bad()


class Tied(nn.Module):
    def __init__(self):
        super().__init__()
        self.first, self.second = Experts(torch.float32), Experts(torch.float32)
        self.second.up = self.first.up
        self.first.also = self.first.down


def test_shared_stacks_stay_shared():
    m = convert_mixed_precision_experts(Tied())
    assert isinstance(m.first.up, MixedPrecisionLinearWeight) and m.first.up is m.second.up and m.first.also is m.first.down
    assert m.second.down is not m.first.down and isinstance(m.second.down, MixedPrecisionLinearWeight)
    assert sum(isinstance(p, MixedPrecisionLinearWeight) for p in m.parameters()) == 3
    again = convert_mixed_precision_experts(m)
    assert again.first.up is m.second.up and not isinstance(m.first.up._data, MixedPrecisionLinearWeight)


def test_conversion_of_named_stacks_only():
    """Three dims do not make a stack of experts: a position embedding (1, L, D) is one that the caller knows."""
    m = Experts()
    m.positions = nn.Parameter(torch.zeros(1, 5, 8))
    m.inner = Experts()
    convert_mixed_precision_experts(m, filter_fn=lambda name, p: "positions" not in name and name != "inner.down")
    assert isinstance(m.up, MixedPrecisionLinearWeight) and isinstance(m.inner.up, MixedPrecisionLinearWeight)
    assert not isinstance(m.positions, MixedPrecisionLinearWeight) and not isinstance(m.inner.down, MixedPrecisionLinearWeight)


def test_a_slice_of_the_experts_reaches_the_operator(cpu_ops):
    """As a rank that holds some of the experts takes them; the gradient of the others is zero."""
    g = torch.Generator().manual_seed(8)
    x, w = torch.randn(5, 8, generator=g, dtype=torch.float64), torch.randn(4, 12, 8, generator=g, dtype=torch.float64)
    wp = nn.Parameter(MixedPrecisionLinearWeight(w, MixedPrecisionConfig()))
    y = F.grouped_mm(x, wp[1:3].transpose(-2, -1), offs=torch.tensor([2, 5], dtype=torch.int32))
    torch.testing.assert_close(y.detach(), torch.cat([x[:2] @ w[1].T, x[2:] @ w[2].T]), rtol=1e-12, atol=1e-12)
    y.sum().backward()
    gw = getattr(wp.grad, "_data", wp.grad)
    assert gw.shape == w.shape and (gw[0] == 0).all() and (gw[3] == 0).all()
    torch.testing.assert_close(gw[1], x[:2].sum(0).expand(12, 8), rtol=1e-12, atol=1e-12)
