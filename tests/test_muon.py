"""The optimizer around orthogonalize: its arithmetic against the formula on the host (with the operator's definition as the host's
implementation), and a training run on the device."""
import json
import subprocess
import sys
from pathlib import Path

import pytest
import torch
from torch import nn

import gn_kernels
from muon import Muon
from subclasses import MixedPrecisionConfig, MixedPrecisionLinearWeight

ROOT = Path(__file__).resolve().parent.parent


def newton_schulz(G, steps, a, b, c, eps):
    X = G.double()
    X = X / X.flatten(-2).norm(dim=-1)[..., None, None].clamp_min(eps)
    for _ in range(steps):
        S = X @ X.mT
        X = a * X + b * S @ X + c * S @ S @ X
    return X.to(G.dtype)


@pytest.fixture(scope="module")
def cpu_op():
    impl = torch.library.Library("gn_kernels", "IMPL")
    impl.impl("orthogonalize", newton_schulz, "CPU")
    yield


def test_wrapper_refuses_and_infers_shapes():
    for bad in (lambda: gn_kernels.orthogonalize(torch.zeros(4, device="meta")), lambda: gn_kernels.orthogonalize(torch.zeros(4, 4, device="meta", dtype=torch.float64)),
                lambda: gn_kernels.orthogonalize(torch.zeros(4, 4, device="meta"), steps=0), lambda: gn_kernels.orthogonalize(torch.zeros(4, 4, device="meta"), eps=-1.0),
                lambda: gn_kernels.orthogonalize(torch.zeros(4, 4, device="meta"), coefficients=(1.0, 2.0))):
        with pytest.raises(AssertionError):
            bad()
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        y = gn_kernels.orthogonalize(torch.zeros(2, 3, 4, device="meta", dtype=dt))
        assert y.shape == (2, 3, 4) and y.dtype is dt


def test_cabi_refusals_without_a_gpu():
    L = gn_kernels._cabi.load()
    call = lambda *, dt=0, b=1, m=4, n=4, steps=5, a=3.4445, eps=1e-7: L.gnk_orthogonalize(None, dt, None, dt, b, m, n, steps, a, -4.775, 2.0315, eps, None, 0, None)  # noqa: E731
    assert call() == -1 and b"null pointer" in L.gnk_last_error()
    assert call(dt=3) == -1 and call(b=-1) == -1 and call(steps=0) == -1 and call(steps=101) == -1 and call(a=1e5) == -1 and call(a=float("nan")) == -1
    assert call(eps=-1.0) == -1 and call(m=(1 << 20) + 1) == -2 and call(b=1 << 16) == -2
    assert call(b=0) == 0 and call(m=0) == 0
    assert L.gnk_orthogonalize_workspace_bytes(0, 4, 4) == 0 and L.gnk_orthogonalize_workspace_bytes(2, 100, 300) >= 2 * 2 * 2 * (128 * 384 + 128 * 128)


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("wd", [0.0, 0.1])
def test_update_rule(cpu_op, nesterov, wd):
    """Three steps of matrices of two shapes and a stack, against the formula written out."""
    g = torch.Generator().manual_seed(0)
    shapes = [(6, 10), (10, 6), (6, 10), (3, 6, 10)]
    ps = [nn.Parameter(torch.randn(s, generator=g, dtype=torch.float32)) for s in shapes]
    want = [p.detach().clone() for p in ps]
    mom = [torch.zeros_like(p) for p in want]
    opt = Muon(ps, lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=wd)
    for _ in range(3):
        grads = [torch.randn(s, generator=g) for s in shapes]
        for p, gr in zip(ps, grads):
            p.grad = gr.clone()
        opt.step()
        for i, gr in enumerate(grads):
            mom[i] = 0.9 * mom[i] + gr
            u = gr + 0.9 * mom[i] if nesterov else mom[i]
            u = newton_schulz(u, 5, 3.4445, -4.7750, 2.0315, 1e-7)
            want[i] = want[i] * (1 - 0.1 * wd) - 0.1 * max(1.0, u.shape[-2] / u.shape[-1]) ** 0.5 * u
    for p, w in zip(ps, want):
        # a few fp32 roundings per step, of values around 1, through an iteration that stretches small ones by 3.4 per step: 3.4^5 * 2^-22
        torch.testing.assert_close(p.detach(), w, rtol=1e-4, atol=2e-4)


def test_wrapped_weights_and_missing_gradients(cpu_op):
    w = torch.randn(8, 4, generator=torch.Generator().manual_seed(1))
    p = nn.Parameter(MixedPrecisionLinearWeight(w.clone(), MixedPrecisionConfig()))
    q = nn.Parameter(torch.zeros(4, 4))
    opt = Muon([p, q], lr=0.1)
    p.grad = torch.ones(8, 4)
    opt.step()
    assert isinstance(p, MixedPrecisionLinearWeight) and not torch.equal(p._data, w) and torch.equal(q.detach(), torch.zeros(4, 4))
    assert "momentum" not in opt.state[q]


def test_refuses_what_it_cannot_update():
    for bad in (torch.zeros(4), torch.zeros(1, 2, 3, 4)):
        with pytest.raises(ValueError):
            Muon([nn.Parameter(bad)])
    with pytest.raises(ValueError):
        Muon([nn.Parameter(torch.zeros(4, 4))], lr=-1.0)


def test_momentum_is_fp32_and_survives_a_checkpoint(cpu_op):
    """Gradients of 1 and then of 2^-10, which a bf16 momentum near 1 would lose: the state is the fp32 sum, before and after a reload."""
    make = lambda: Muon([nn.Parameter(torch.zeros(2, 4, 4, dtype=torch.bfloat16)), nn.Parameter(torch.zeros(4, 6, dtype=torch.bfloat16))], momentum=1.0 - 2.0 ** -8)  # noqa: E731
    opt = make()
    for value in (1.0, 2.0 ** -10):
        for p in opt.param_groups[0]["params"]:
            p.grad = torch.full_like(p, value)
        opt.step()
    want = 1.0 - 2.0 ** -8 + 2.0 ** -10                       # exact in fp32
    other = make()
    other.load_state_dict(opt.state_dict())
    for o in (opt, other):
        for p in o.param_groups[0]["params"]:
            m = o.state[p]["momentum"]
            assert m.dtype is torch.float32 and (m == want).all()
    assert all(other.state[a]["momentum"] is not opt.state[b]["momentum"]
               for a, b in zip(other.param_groups[0]["params"], opt.param_groups[0]["params"]))


def test_refuses_empty_matrices_and_bad_groups():
    with pytest.raises(ValueError):
        Muon([nn.Parameter(torch.zeros(0, 4))])
    opt = Muon([nn.Parameter(torch.zeros(4, 4))])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [nn.Parameter(torch.zeros(4))]})
    assert len(opt.param_groups) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("quantize", ["none", "mixed_precision"])
def test_training_harness_runs_on_the_device(quantize):
    r = subprocess.run([sys.executable, str(ROOT / "train_bench.py"), "--model", "tiny", "--quantize", quantize, "--batch_size", "2", "--seq_len", "64", "--steps", "2",
                        "--warmup", "1", "--optimizer", "muon"], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stderr[-2000:]
    out = json.loads([l for l in r.stdout.splitlines() if l.startswith("{")][-1])
    assert out["value"] > 0 and "Muon" in out["config"]["workload"]


@pytest.mark.gpu
def test_update_on_the_device():
    """One step of a stack of experts and a Linear's weight: the update is lr times the operator's result."""
    g = torch.Generator().manual_seed(2)
    ps = [nn.Parameter(torch.randn(s, generator=g).bfloat16().cuda()) for s in ((3, 64, 96), (64, 96), (96, 64))]
    before = [p.detach().clone() for p in ps]
    for p in ps:
        p.grad = torch.randn(p.shape, generator=g).bfloat16().cuda()
    Muon(ps, lr=0.5, momentum=0.0, nesterov=False).step()
    for p, b in zip(ps, before):
        u = gn_kernels.orthogonalize(p.grad)
        want = b.double() - 0.5 * max(1.0, p.shape[-2] / p.shape[-1]) ** 0.5 * u.double()
        # the stack and the single call round alike; the sum is rounded to bf16 once (the scaled update once more where the factor is no power of two)
        assert ((p.detach().double() - want).abs() <= 2.0 ** -8 * (want.abs() + u.double().abs())).all()


def test_fp16_gradients_whose_momentum_leaves_fp16(cpu_op):
    """Gradients near fp16's largest value (as a loss scale leaves them): the momentum is 1.9 of them after two steps, more than fp16 holds; the update is the
    formula's, in fp32, rounded once to the weight."""
    g = torch.Generator().manual_seed(3)
    p = nn.Parameter(torch.zeros(6, 10, dtype=torch.float16))
    opt = Muon([p], lr=0.5)
    want, mom = torch.zeros(6, 10, dtype=torch.float64), torch.zeros(6, 10, dtype=torch.float64)
    gr = (torch.randn(6, 10, generator=g).clamp(-1, 1) * 6e4).half()
    for _ in range(2):
        p.grad = gr.clone()
        opt.step()
        mom = 0.95 * mom + gr.double()
        want = want - 0.5 * newton_schulz(gr.double() + 0.95 * mom, 5, 3.4445, -4.7750, 2.0315, 1e-7)
    assert (gr.double() + 0.95 * mom).abs().max() > 65504
    # two roundings to fp16 (2^-11 of values up to 1.3 each) and fp32's in the momentum, stretched by 3.4^5
    assert torch.isfinite(p).all() and ((p.detach().double() - want).abs() <= 2 * 1.3 * 2.0 ** -11 + 2e-4).all()


def test_calls_are_bounded_whatever_the_number_of_layers(cpu_op, monkeypatch):
    """Many equal layers and a stack that is larger than a call: the update of one call per matrix, from calls of at most the bound (not one for everything)."""
    import muon

    per = 4
    monkeypatch.setattr(muon, "_CALL_WORK", per * 6.0 * 6 * 10)
    seen, op = [], muon.orthogonalize
    monkeypatch.setattr(muon, "orthogonalize", lambda G, **kw: seen.append(G.shape[0]) or op(G, **kw))
    g = torch.Generator().manual_seed(4)
    shapes = [(6, 10)] * 7 + [(11, 6, 10), (2, 6, 10), (0, 6, 10)]
    grads = [torch.randn(s, generator=g) for s in shapes]
    ps, alone = ([nn.Parameter(torch.zeros(s)) for s in shapes] for _ in range(2))
    for group in (ps, alone):
        for p, gr in zip(group, grads):
            p.grad = gr.clone()
    Muon(ps, lr=0.1, weight_decay=0.1).step()
    assert sum(seen) == 20 and max(seen) <= per and len(seen) == 5
    for p in alone:
        Muon([p], lr=0.1, weight_decay=0.1).step()
    # the host's products may add in another order for another batch: rounding of values around 1 in 64 bits, then to fp32 (2^-24), and of the update's sum
    for p, q in zip(ps, alone):
        torch.testing.assert_close(p.detach(), q.detach(), rtol=2.0 ** -22, atol=2.0 ** -24)


def test_matrices_per_call():
    from muon import matrices_per_call

    assert matrices_per_call(2048, 5632, 44) == 15 and matrices_per_call(5632, 2048, 16) == 16 and matrices_per_call(2048, 5632, 1) == 1
    assert matrices_per_call(1, 1, 200000) == 50000 and matrices_per_call(64, 1 << 20, 100) == 4 and matrices_per_call(20000, 50000, 3) == 1
    assert matrices_per_call(8, 8, 0) == 1


@pytest.mark.gpu
def test_bounded_calls_on_the_device(monkeypatch):
    """The same in bf16 on the device, where another batch may take other tiles: both updates are within the operator's error of the definition, 2e-3 of the norm
    each, and the result's and the weight's rounding, 2^-8 each."""
    import muon

    g = torch.Generator().manual_seed(5)
    shapes = [(64, 96)] * 5 + [(3, 64, 96)]
    grads = [torch.randn(s, generator=g).bfloat16().cuda() for s in shapes]
    results = []
    for work in (muon._CALL_WORK, 3.0 * 64 * 64 * 96):
        monkeypatch.setattr(muon, "_CALL_WORK", work)
        ps = [nn.Parameter(torch.zeros(s, dtype=torch.bfloat16, device="cuda")) for s in shapes]
        for p, gr in zip(ps, grads):
            p.grad = gr.clone()
        Muon(ps, lr=1.0).step()
        results.append([p.detach().double() for p in ps])
    for a, b in zip(*results):
        assert (a - b).norm() <= 2 * (2e-3 + 2 * 2.0 ** -8) * b.norm() and b.norm() > 0


@pytest.mark.parametrize("kind", ["int8", "bitnet", "mixed_precision"])
def test_quantized_weights_are_updated(cpu_op, kind):
    """Every weight class whose in-place arithmetic an optimizer uses: the step moves it by lr u (u: singular values near 1), however it stores itself."""
    from subclasses import convert_bitnet, convert_int8_quantized_training, convert_mixed_precision

    torch.manual_seed(0)
    m = nn.Sequential(nn.Linear(8, 16, bias=False).bfloat16())
    {"int8": convert_int8_quantized_training, "bitnet": convert_bitnet, "mixed_precision": convert_mixed_precision}[kind](m)
    p = m[0].weight
    values = lambda: (p.dequantize() if kind == "int8" else p._data).double()  # noqa: E731
    before, p.grad = values(), torch.randn(16, 8).bfloat16()
    u = newton_schulz(p.grad.double() * 1.95, 5, 3.4445, -4.7750, 2.0315, 1e-7)
    Muon([p], lr=0.5).step()
    step = values() - before
    # sqrt(2) lr u; bf16's roundings (u, the weight) and, for int8, a step of the row's scale (amax / 127) on either side
    want = -0.5 * 2 ** 0.5 * u
    tol = 2.0 ** -7 + (2 * (values().abs().amax() + before.abs().amax()) / 127 if kind == "int8" else 0.0)
    assert type(p).__name__ != "Parameter" and ((step - want).abs() <= tol).all()
