"""Products grouped by expert: `grouped_scaled_mm`, and `quantize_int8_grouped` in front of its weight gradients.

Rows are sorted by expert and the group sizes live on the device: `offs` holds each group's end, as `torch.nn.functional.grouped_mm`
takes it.  The reference has no counterpart (its Linears are dense); the operands, scales and result types are those of `scaled_mm`
(kernels/gn_kernels/triton_mm.py:349-373 of the reference), one product per group.  Nothing is read back from the device, so the ops
trace under torch.compile and can be captured into a HIP graph that is replayed with other group sizes.
"""
from __future__ import annotations

import torch
from torch import Tensor

from . import _cabi
from ._lib import lib, lib_ops
from .mm import _FP8, _check_scale_dtype
from .quantize import _sr_args, draw_rng

lib.define("grouped_scaled_mm(Tensor A, Tensor B, Tensor scale_A, Tensor scale_B, Tensor offs) -> Tensor")
lib.define("grouped_scaled_mm_depth(Tensor A, Tensor B, Tensor scale_A, Tensor scale_B, Tensor offs) -> Tensor")
lib.define("quantize_int8_grouped(Tensor x, Tensor offs, bool stochastic_rounding, float eps, Tensor? rng=None) -> (Tensor, Tensor)")

# `F.grouped_mm` on a mixed-precision weight (subclasses/mixed_precision.py) without stochastic rounding, one call per direction: x (T, K), w (E, K, N),
# offs -> y, and grad_y -> (grad_x, grad_w (E, N, K)); a gradient that is not asked for comes back with no rows.
lib.define("grouped_linear_int8(Tensor x, Tensor w, Tensor offs) -> Tensor")
lib.define("grouped_linear_int8_backward(Tensor grad_y, Tensor x, Tensor w, Tensor offs, bool need_x, bool need_w) -> (Tensor, Tensor)")


def grouped_scaled_mm(A: Tensor, B: Tensor, scale_A: Tensor, scale_B: Tensor, offs: Tensor) -> Tensor:
    """`scaled_mm` for every group of rows; group e holds rows offs[e - 1] .. offs[e] - 1 (offs[-1] = 0).

    * B (E, K, N), scale_B (E, 1, N) or (E, 1, 1); A (T, K), scale_A (T, 1): rows form, (T, N),
      out[t, n] = (f32(A[t] @ B[e]) * scale_A[t]) * scale_B[e, n] with e the group of row t; rows behind offs[-1] come out as zeros.
    * B (T, N), scale_B (E, 1, N) or (E, 1, 1); A (M, T), scale_A (E, M, 1): the contraction runs over each group's rows, (E, M, N),
      out[e, m, n] = (f32(A[m, group e] @ B[group e, n]) * scale_A[e, m]) * scale_B[e, n]; empty groups have a zero sum.

    A and B are both int8, or any mix of float8_e4m3fn / float8_e5m2; any strides, but operands whose contiguous extent is a multiple of
    16 and whose rows are 16-byte aligned are read where they lie: A along K and B along K or N (rows form), A along M and B along N (second
    form).  Others are copied first.  scales are contiguous, the result has their dtype.  offs: int32 on the same device, not decreasing,
    at most T (not checked, as that would wait for the device: a value below an earlier one counts as that one, one beyond T as T).
    int8 sums are exact: over any number of rows in the second form; the first one refuses K > 131071, where they may not fit 32 bits.
    """
    dt, E = A.dtype, offs.shape[0]
    assert (dt is torch.int8 and B.dtype is torch.int8) or (dt in _FP8 and B.dtype in _FP8)
    assert scale_A.dtype is scale_B.dtype
    assert offs.ndim == 1 and offs.dtype is torch.int32 and offs.is_contiguous()
    assert scale_A.is_contiguous() and scale_B.is_contiguous()
    shape_B = tuple(B.shape)
    assert tuple(scale_B.shape) in ((E, 1, shape_B[-1]), (E, 1, 1))
    m, k = A.shape
    if len(shape_B) == 3:
        assert shape_B[0] == E and k == shape_B[1]
        assert tuple(scale_A.shape) == (m, 1)
        return lib_ops.grouped_scaled_mm.default(A, B, scale_A, scale_B, offs)
    assert len(shape_B) == 2 and k == shape_B[0]
    assert tuple(scale_A.shape) == (E, m, 1)
    return lib_ops.grouped_scaled_mm_depth.default(A, B, scale_A, scale_B, offs)


def quantize_int8_grouped(x: Tensor, offs: Tensor, stochastic_rounding: bool = False, *, eps: float = 1e-12):
    """`quantize_int8(x[group e], dim=0)` for every group of rows of x (T, C): (int8 data (T, C) contiguous, scale (E, 1, C) in x.dtype).

    scale = amax * fl(1 / 127), the product that eager torch makes of `amax / 127` on a device; `quantize_int8` divides.  The two scales are
    within 1.5 fp32 steps, and a value next to a rounding border may come out one off from `quantize_int8`'s.
    Groups without rows have scale 0; rows behind offs[-1] come out as zeros.  offs as in `grouped_scaled_mm`."""
    assert x.ndim == 2
    assert offs.ndim == 1 and offs.dtype is torch.int32 and offs.is_contiguous()
    return lib_ops.quantize_int8_grouped(x, offs, stochastic_rounding, eps, draw_rng(stochastic_rounding))


@torch.library.impl(lib, "grouped_scaled_mm", "Meta")
def _rows_meta(A: Tensor, B: Tensor, scale_A: Tensor, scale_B: Tensor, offs: Tensor):
    return torch.empty((A.shape[0], B.shape[2]), device=A.device, dtype=scale_A.dtype)


@torch.library.impl(lib, "grouped_scaled_mm_depth", "Meta")
def _depth_meta(A: Tensor, B: Tensor, scale_A: Tensor, scale_B: Tensor, offs: Tensor):
    return torch.empty((offs.shape[0], A.shape[0], B.shape[1]), device=A.device, dtype=scale_A.dtype)


@torch.library.impl(lib, "quantize_int8_grouped", "Meta")
def _quantize_meta(x: Tensor, offs: Tensor, stochastic_rounding: bool, eps: float, rng: Tensor | None = None):
    return torch.empty(x.shape, dtype=torch.int8, device=x.device), x.new_empty((offs.shape[0], 1, x.shape[1]))


@torch.library.impl(lib, "grouped_linear_int8", "Meta")
def _linear_meta(x: Tensor, w: Tensor, offs: Tensor):
    return x.new_empty((x.shape[0], w.shape[2]))


@torch.library.impl(lib, "grouped_linear_int8_backward", "Meta")
def _linear_backward_meta(grad_y: Tensor, x: Tensor, w: Tensor, offs: Tensor, need_x: bool, need_w: bool):
    E, K, N = w.shape
    return x.new_empty((x.shape[0] if need_x else 0, K)), x.new_empty((E if need_w else 0, N, K))


def _check(op: str, A: Tensor, *others: Tensor) -> None:
    if any(t.device != A.device for t in others):
        raise RuntimeError(f"gn_kernels::{op}: all tensors must be on one device")


@_cabi.device_impl(lib, "grouped_scaled_mm")
def _rows_hip(A: Tensor, B: Tensor, scale_A: Tensor, scale_B: Tensor, offs: Tensor):
    _check_scale_dtype(scale_A, "grouped_scaled_mm")
    _check("grouped_scaled_mm", A, B, scale_A, scale_B, offs)
    (T, K), (E, _, N) = A.shape, B.shape
    C = torch.empty((T, N), device=A.device, dtype=scale_A.dtype)
    L, code = _cabi.load(), _cabi.DTYPE_CODE
    with _cabi.device_of(A):
        nws = L.gnk_grouped_scaled_mm_rows_workspace_bytes(A.data_ptr(), B.data_ptr(), T, E, N, K, *A.stride(), *B.stride())
        ws = torch.empty(nws, device=A.device, dtype=torch.uint8) if nws else None
        rc = L.gnk_grouped_scaled_mm_rows(A.data_ptr(), code[A.dtype], B.data_ptr(), code[B.dtype], C.data_ptr(), code[C.dtype], scale_A.data_ptr(),
                                          scale_B.data_ptr(), code[scale_A.dtype], int(scale_B.shape[2] == 1 and N != 1), offs.data_ptr(), T, E, N, K,
                                          *A.stride(), *B.stride(), ws.data_ptr() if nws else None, nws, _cabi.stream_of(A))
    _cabi.check(rc, "grouped_scaled_mm")
    return C


@_cabi.device_impl(lib, "grouped_scaled_mm_depth")
def _depth_hip(A: Tensor, B: Tensor, scale_A: Tensor, scale_B: Tensor, offs: Tensor):
    _check_scale_dtype(scale_A, "grouped_scaled_mm_depth")
    _check("grouped_scaled_mm_depth", A, B, scale_A, scale_B, offs)
    (M, T), N, E = A.shape, B.shape[1], offs.shape[0]
    C = torch.empty((E, M, N), device=A.device, dtype=scale_A.dtype)
    L, code = _cabi.load(), _cabi.DTYPE_CODE
    with _cabi.device_of(A):
        nws = L.gnk_grouped_scaled_mm_depth_workspace_bytes(A.data_ptr(), B.data_ptr(), T, M, N, *A.stride(), *B.stride())
        nws = (nws + 15) // 16 * 16 + L.gnk_grouped_scaled_mm_depth_split_bytes(T, E, M, N)
        ws = torch.empty(nws, device=A.device, dtype=torch.uint8) if nws else None
        rc = L.gnk_grouped_scaled_mm_depth(A.data_ptr(), code[A.dtype], B.data_ptr(), code[B.dtype], C.data_ptr(), code[C.dtype], scale_A.data_ptr(),
                                           scale_B.data_ptr(), code[scale_A.dtype], int(scale_B.shape[2] == 1 and N != 1), offs.data_ptr(), T, E, M, N,
                                           *A.stride(), *B.stride(), ws.data_ptr() if nws else None, nws, _cabi.stream_of(A))
    _cabi.check(rc, "grouped_scaled_mm_depth")
    return C


@_cabi.device_impl(lib, "quantize_int8_grouped")
def _quantize_hip(x: Tensor, offs: Tensor, stochastic_rounding: bool, eps: float, rng: Tensor | None = None):
    _check_scale_dtype(x, "quantize_int8_grouped")
    _check("quantize_int8_grouped", x, offs)
    (T, C), E = x.shape, offs.shape[0]
    q = torch.empty((T, C), dtype=torch.int8, device=x.device)
    scale = torch.empty((E, 1, C), dtype=x.dtype, device=x.device)
    L = _cabi.load()
    nws = L.gnk_quantize_int8_grouped_workspace_bytes(T, E, C)
    ws = torch.empty(nws, dtype=torch.uint8, device=x.device) if nws else None
    seed, offset = _sr_args(stochastic_rounding, rng)
    with _cabi.device_of(x):
        rc = L.gnk_quantize_int8_grouped(x.data_ptr(), _cabi.DTYPE_CODE[x.dtype], offs.data_ptr(), T, E, C, *x.stride(), q.data_ptr(), scale.data_ptr(), eps,
                                         int(stochastic_rounding), seed, offset, ws.data_ptr() if nws else None, nws, _cabi.stream_of(x))
    _cabi.check(rc, "quantize_int8_grouped")
    return q, scale


def linear_forward(x: Tensor, w: Tensor, offs: Tensor, sr: bool) -> Tensor:
    """y (T, N) of x (T, K) and w (E, K, N): x per row and w per (expert, n) in int8."""
    E, K, N = w.shape
    xq, xs = lib_ops.quantize_int8(x, 1, sr, 1e-12, draw_rng(sr))
    wq, ws = lib_ops.quantize_int8(w.transpose(1, 2).reshape(E * N, K), 1, sr, 1e-12, draw_rng(sr))
    return lib_ops.grouped_scaled_mm(xq, wq.view(E, N, K).transpose(1, 2), xs, ws.view(E, 1, N), offs)


def linear_backward(grad_y: Tensor, x: Tensor, w: Tensor, offs: Tensor, need_x: bool, need_w: bool, sr: bool):
    """(grad_x (T, K), grad_w (E, N, K)): grad_y per row with w per (expert, k); grad_y and x per (group, column)."""
    E, K, N = w.shape
    gx, gw = x.new_empty((0, K)), x.new_empty((0, N, K))
    if need_x:
        gq, gs = lib_ops.quantize_int8(grad_y, 1, sr, 1e-12, draw_rng(sr))
        ends = torch.arange(1, E + 1, dtype=torch.int32, device=w.device) * N      # an expert's N rows are a group
        wq, ws = lib_ops.quantize_int8_grouped(w.transpose(1, 2).reshape(E * N, K), ends, sr, 1e-12, draw_rng(sr))
        gx = lib_ops.grouped_scaled_mm(gq, wq.view(E, N, K), gs, ws, offs)
    if need_w:
        xq, xs = lib_ops.quantize_int8_grouped(x, offs, sr, 1e-12, draw_rng(sr))
        gq, gs = lib_ops.quantize_int8_grouped(grad_y, offs, sr, 1e-12, draw_rng(sr))
        gw = lib_ops.grouped_scaled_mm_depth(gq.T, xq, gs.view(E, N, 1), xs, offs)
    return gx, gw


@_cabi.device_impl(lib, "grouped_linear_int8")
def _linear_hip(x: Tensor, w: Tensor, offs: Tensor):
    return linear_forward(x, w, offs, False)


@_cabi.device_impl(lib, "grouped_linear_int8_backward")
def _linear_backward_hip(grad_y: Tensor, x: Tensor, w: Tensor, offs: Tensor, need_x: bool, need_w: bool):
    return linear_backward(grad_y, x, w, offs, need_x, need_w, False)
