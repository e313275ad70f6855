"""orthogonalize on stacks that run as two chains of products on two streams: odd numbers of matrices, wide and tall ones, each type of result, against the
iteration in 64 bits (on the device), and the bits of the single chain of a captured call.

Tolerances: fp16 and fp32 results as in `compare_closely` of tests/test_gpu_ortho.py (3e-4 and half a step), bf16 as in its test_large_stack_takes_two_streams
(twice 1.2e-3, the fp16 roundings' share, and bf16's 2^-8)."""
import pytest
import torch

import gn_kernels
from gn_kernels import _cabi
from tests.test_gpu_ortho import COEFFS, DEV, DT

SHAPES = [("f16", 2, 4096, 4096), ("f16", 3, 5632, 2560), ("f32", 3, 2560, 5632), ("bf16", 3, 5632, 2560), ("bf16", 5, 2560, 4224)]


def chains(dt, B, m, n):
    return _cabi.load().gnk_orthogonalize_chains(_cabi.DTYPE_CODE[DT[dt]], B, m, n)


@pytest.mark.parametrize("dt,B,m,n", SHAPES)
def test_the_tested_shapes_run_as_two_chains(dt, B, m, n):
    assert chains(dt, B, m, n) == 2


def test_small_and_single_ones_do_not():
    assert chains("bf16", 1, 4096, 4096) == 1 and chains("bf16", 8, 1024, 4096) == 1 and chains("f16", 2, 3, 4) == 1
    assert chains("bf16", 0, 4096, 4096) == 0 and chains("bf16", 2, 0, 4096) == 0


def definition(G):
    X = G.double()
    X = X / X.norm()
    for _ in range(5):
        S = X @ X.T if X.shape[0] <= X.shape[1] else X.T @ X
        P = COEFFS[1] * S + COEFFS[2] * (S @ S)
        X = COEFFS[0] * X + (P @ X if X.shape[0] <= X.shape[1] else X @ P)
    return X


@pytest.mark.gpu
@pytest.mark.parametrize("dt,B,m,n", SHAPES)
def test_against_the_definition_and_one_chain(dt, B, m, n):
    assert chains(dt, B, m, n) == 2
    g = torch.Generator(device=DEV).manual_seed(m + B)
    G = torch.stack([torch.randn(m, n, generator=g, device=DEV) * 4.0 ** -i for i in range(B)]).to(DT[dt])
    got = gn_kernels.orthogonalize(G)
    tol = 3e-4 + torch.finfo(G.dtype).eps / 2 if dt != "bf16" else 2 * 1.2e-3 + 2.0 ** -8
    for x, one in zip(got, G):
        want = definition(one)
        assert (x.double() - want).norm() <= tol * want.norm()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gn_kernels.orthogonalize(G)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, got)


@pytest.mark.gpu
def test_from_two_streams_at_once():
    """Both callers' second chains share a stream: results as alone, with inputs that the next call's work overwrites only behind its own stream."""
    g = torch.Generator(device=DEV).manual_seed(1)
    Gs = [torch.randn(3, 5632, 2560, generator=g, device=DEV).half() for _ in range(2)]
    want = [gn_kernels.orthogonalize(G) for G in Gs]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in Gs], [[], []]
    for _ in range(3):
        for i, (s, G) in enumerate(zip(streams, Gs)):
            with torch.cuda.stream(s):
                outs[i].append(gn_kernels.orthogonalize(G))
                outs[i].append(gn_kernels.orthogonalize(G + 0))         # an input that is freed while the call is on the way
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(x, w) for x in o)
