"""torch.compile (inductor, fullgraph) over the operators of expert layers and orthogonalize on the device: the operators are opaque nodes, so that compiled
calls give the bits of eager ones, also for other group sizes."""
import pytest
import torch
import torch.nn.functional as F
from torch import nn

import gn_kernels
from subclasses import MixedPrecisionConfig, MixedPrecisionLinearWeight
from tests.test_gpu_grouped import DEV, offs_of

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _fresh_dynamo():
    torch._dynamo.reset()
    yield
    torch._dynamo.reset()


@pytest.mark.parametrize("turn", [lambda w: w.transpose(-2, -1), lambda w: w.permute(0, 2, 1)], ids=["transpose", "permute"])
def test_expert_projection(turn):
    g = torch.Generator().manual_seed(0)
    x, w, gy = (torch.randn(s, generator=g).bfloat16().to(DEV) for s in ((100, 64), (3, 96, 64), (100, 96)))

    def call(x, w, offs):
        return F.grouped_mm(x, turn(w), offs=offs)

    compiled = torch.compile(call, fullgraph=True)
    for sizes in ([40, 0, 57], [0, 100, 0]):
        results = []
        for fn in (call, compiled):
            xd, wd = x.clone().requires_grad_(), nn.Parameter(MixedPrecisionLinearWeight(w.clone(), MixedPrecisionConfig()))
            y = fn(xd, wd, offs_of(sizes))
            y.backward(gy)
            results.append((y.detach(), xd.grad, getattr(wd.grad, "_data", wd.grad)))
        for a, b in zip(*results):
            assert torch.equal(a, b)


def test_operators():
    g = torch.Generator().manual_seed(1)
    x, y = torch.randn(90, 64, generator=g).bfloat16().to(DEV), torch.randn(90, 48, generator=g).bfloat16().to(DEV)
    offs = offs_of([30, 0, 60])

    def call(x, y, offs):
        (a, sa), (b, sb) = gn_kernels.quantize_int8_grouped(x, offs), gn_kernels.quantize_int8_grouped(y, offs)
        grads = gn_kernels.grouped_scaled_mm(a.T, b, sa.transpose(1, 2).contiguous(), sb, offs)
        return a, sa, grads, gn_kernels.orthogonalize(grads)

    for a, b in zip(call(x, y, offs), torch.compile(call, fullgraph=True)(x, y, offs)):
        assert torch.equal(a, b)
