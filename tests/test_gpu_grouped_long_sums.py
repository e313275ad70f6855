"""int8 sums of more products than 32 bits are sure to hold (127 * 127 of them overflow from 133145 on, 128 * 128 from 131072): weight gradients over that many
rows of one expert, with columns of one sign, as a constant feature has them.

Tolerance: the sum is exact, its conversion to fp32 and the two scale multiplies are at most 2^-24 off each, and the result half a step of its type
(`check` of tests/test_gpu_grouped.py, int8)."""
import pytest
import torch
import torch.nn.functional as F
from torch import nn

import gn_kernels
from gn_kernels import _cabi
from subclasses import MixedPrecisionConfig, MixedPrecisionLinearWeight
from tests.test_gpu_grouped import DEV, OUT, check, offs_of, scales, spans

pytestmark = pytest.mark.gpu

LONG_ROWS = 130816
SIZES = {
    "one": [140000],
    "one_of_three": [131, 140000, 0],
    "border": [LONG_ROWS, LONG_ROWS + 1, 7],
    "three_pieces": [5, 0, 2 * LONG_ROWS + 1, 64],
    "many_groups": [3] * 40 + [133200] + [2] * 30 + [LONG_ROWS + 300],
}


def operands(sizes, M, N, out, seed=0):
    """Columns of 127, of -128, and random ones."""
    g = torch.Generator().manual_seed(seed)
    T, E = sum(sizes), len(sizes)
    A = torch.randint(-128, 128, (T, M), generator=g, dtype=torch.int8)
    B = torch.randint(-128, 128, (T, N), generator=g, dtype=torch.int8)
    for t in (A, B):
        t[:, 0::3] = 127
        t[:, 1::3] = -128
    return A.to(DEV).T, B.to(DEV), scales((E, M, 1), out, g).to(DEV), scales((E, 1, N), out, g).to(DEV)


def in_64_bits(A, B, sA, sB, sizes):
    """fp64 sums of whole numbers below 2^53: exact in any order."""
    want = [(A[:, lo:hi].double().contiguous() @ B[lo:hi].double()) * sA[e].double() * sB[e].double() for e, (lo, hi) in enumerate(spans(sizes))]
    return torch.stack(want).cpu()


@pytest.fixture(params=[-1, 1, 5, 6], ids=["auto", "tile128", "tile256w4", "tile64"])
def forced(request):
    L = _cabi.load()
    old = L.gnk_set_gemm_variant(request.param)
    yield request.param
    L.gnk_set_gemm_variant(old)


@pytest.mark.parametrize("name", list(SIZES))
@pytest.mark.parametrize("M,N", [(48, 33), (300, 264)])
def test_depth(forced, name, M, N):
    sizes = SIZES[name]
    A, B, sA, sB = operands(sizes, M, N, "f32")
    got = gn_kernels.grouped_scaled_mm(A, B, sA, sB, offs_of(sizes))
    check(got, in_64_bits(A, B, sA, sB, sizes), None, "int8", "f32", 0)


@pytest.mark.parametrize("out", list(OUT))
@pytest.mark.parametrize("scalar", [False, True])
@pytest.mark.parametrize("N", [64, 34])
def test_depth_pieces_output_types(out, scalar, N):
    """The caller has room for the pieces of long groups and not for parts of all of them."""
    L, code = _cabi.load(), _cabi.DTYPE_CODE
    sizes, M = [10, 140000, 3], 36
    A, B, sA, sB = operands(sizes, M, N, out)
    sA, sB = sA * 2.0 ** -12, sB[:, :, :1].contiguous() if scalar else sB          # within fp16's range
    T, E, offs = sum(sizes), len(sizes), offs_of(sizes)
    copies = L.gnk_grouped_scaled_mm_depth_workspace_bytes(A.data_ptr(), B.data_ptr(), T, M, N, *A.stride(), *B.stride())
    pieces = (T // LONG_ROWS + T // (LONG_ROWS + 1)) * M * N * 4
    assert L.gnk_grouped_scaled_mm_depth_split_bytes(T, E, M, N) >= pieces
    C = torch.empty(E, M, N, dtype=OUT[out], device=DEV)

    def call(room):
        ws = torch.empty(max(1, (copies + 15) // 16 * 16 + room), dtype=torch.uint8, device=DEV)
        return L.gnk_grouped_scaled_mm_depth(A.data_ptr(), code[A.dtype], B.data_ptr(), code[B.dtype], C.data_ptr(), code[C.dtype], sA.data_ptr(), sB.data_ptr(),
                                             code[sA.dtype], int(scalar), offs.data_ptr(), T, E, M, N, *A.stride(), *B.stride(), ws.data_ptr(), ws.numel(),
                                             torch.cuda.current_stream().cuda_stream)

    assert call(pieces) == 0
    torch.cuda.synchronize()
    want = in_64_bits(A, B, sA, sB, sizes)
    tol = want.abs() * (torch.finfo(OUT[out]).eps / 2 + 3 * 2.0 ** -24) * (1 + 2.0 ** -8) + (2.0 ** -25 if out == "f16" else 0.0)     # fp16's subnormal step
    assert torch.isfinite(C).all() and ((C.double().cpu() - want).abs() <= tol).all()
    assert call(pieces - 16) == -4 and b"workspace" in L.gnk_last_error()


def test_rows_form_refuses_longer_sums():
    A = torch.zeros(2, 131072, dtype=torch.int8, device=DEV)
    B = torch.zeros(1, 131072, 16, dtype=torch.int8, device=DEV)
    one = torch.ones(2, 1, device=DEV)
    with pytest.raises(RuntimeError, match="32 bits"):
        gn_kernels.grouped_scaled_mm(A, B, one, one[:1, :, None], offs_of([2]))
    A, B = A[:, :131071].contiguous(), B[:, :131071].contiguous()
    A.fill_(-128), B.fill_(-128)
    got = gn_kernels.grouped_scaled_mm(A, B, one, one[:1, :, None], offs_of([2]))
    assert (got.double() == float(torch.tensor(16384.0 * 131071).float())).all()


def test_graph_replays_with_other_sizes():
    """Captured with short groups, replayed with a long one and back."""
    T, M, N = 140000, 40, 48
    A, B, sA, sB = operands([T // 2, T // 2], M, N, "f32")
    offs = offs_of([T // 2, T // 2])
    L = _cabi.load()
    old = L.gnk_set_gemm_variant(6)                  # pieces, not parts
    try:
        gn_kernels.grouped_scaled_mm(A, B, sA, sB, offs)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = gn_kernels.grouped_scaled_mm(A, B, sA, sB, offs)
        for sizes in ([T // 2, T // 2], [T, 0], [3, T - 10], [T // 2, 5]):
            offs.copy_(offs_of(sizes))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, gn_kernels.grouped_scaled_mm(A, B, sA, sB, offs))
            check(out, in_64_bits(A, B, sA, sB, sizes), None, "int8", "f32", 0)
    finally:
        L.gnk_set_gemm_variant(old)


def test_weight_gradient_of_constant_columns():
    """F.grouped_mm: an input of ones against a gradient of ones, 140000 rows of one expert: every gradient is the number of rows (rounded to bf16; the two
    scales, 1 / 127 rounded to bf16, are 2^-8 off each: (1 + 2^-8)^3 - 1 < 3.02 * 2^-8)."""
    T, K, N = 140000, 64, 48
    x = torch.ones(T, K, dtype=torch.bfloat16, device=DEV)
    w = nn.Parameter(MixedPrecisionLinearWeight(torch.zeros(2, N, K, dtype=torch.bfloat16, device=DEV), MixedPrecisionConfig()))
    offs = offs_of([T - 4, 4])
    F.grouped_mm(x, w.transpose(-2, -1), offs=offs).backward(torch.ones(T, N, dtype=torch.bfloat16, device=DEV))
    gw = getattr(w.grad, "_data", w.grad).double()
    for e, rows in enumerate((T - 4, 4)):
        assert ((gw[e] - rows).abs() <= rows * 3.02 * 2.0 ** -8).all()
