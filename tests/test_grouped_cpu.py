"""The grouped products without a GPU: wrapper checks, Meta implementations, the C ABI's refusals, workspace sizes."""
import pytest
import torch

import gn_kernels
from gn_kernels import _cabi


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
