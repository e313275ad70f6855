"""`orthogonalize`: Newton-Schulz orthogonalisation of matrices, the update rule of optimizers that orthogonalise their momentum.

No counterpart in the reference, whose optimizers are element-wise (its train_utils.py takes them from torch, torchao and bitsandbytes).
The three products of a step run on the 16-bit matrix cores in fp16 with power-of-two scales and fp32 sums (csrc/gnk_ortho.hip), in pairs of
fp16 parts where the result has more bits than bf16, a whole stack of matrices -- the weights of a layer of experts, or equal layers side by side -- per launch.
"""
from __future__ import annotations

import torch
from torch import Tensor

from . import _cabi
from ._lib import lib, lib_ops

lib.define("orthogonalize(Tensor G, int steps, float a, float b, float c, float eps) -> Tensor")

_FLOAT = (torch.bfloat16, torch.float16, torch.float32)


def orthogonalize(G: Tensor, *, steps: int = 5, coefficients: tuple[float, float, float] = (3.4445, -4.7750, 2.0315), eps: float = 1e-7) -> Tensor:
    """X = G / max(|G|_F, eps), then `steps` times X <- a X + b (X X^T) X + c (X X^T)^2 X, for every matrix of G (..., m, n).

    Pushes all singular values of G towards 1; bf16, fp16 or fp32, the result has G's dtype and shape and is contiguous.  For the default five
    steps the result is off by about 2e-3 of its norm in bf16 (1.7e-3 is the rounding to bf16), 2e-4 in fp16 (its rounding) and 3e-6 in fp32; fp16 and fp32 take two
    to three times as long as bf16.  The coefficients must keep the singular values below sqrt(2).  A matrix with a NaN or Inf comes out as NaN.
    Not differentiable.
    """
    assert G.ndim >= 2 and G.dtype in _FLOAT
    assert 1 <= steps <= 100 and len(coefficients) == 3 and eps >= 0
    return lib_ops.orthogonalize(G, steps, *(float(v) for v in coefficients), eps)


@torch.library.impl(lib, "orthogonalize", "Meta")
def _meta(G: Tensor, steps: int, a: float, b: float, c: float, eps: float):
    return torch.empty(G.shape, dtype=G.dtype, device=G.device)


@_cabi.device_impl(lib, "orthogonalize")
def _hip(G: Tensor, steps: int, a: float, b: float, c: float, eps: float):
    if G.dtype not in _FLOAT or G.ndim < 2:
        raise RuntimeError(f"gn_kernels::orthogonalize: unsupported input (shape {tuple(G.shape)}, dtype {G.dtype})")
    G = G.contiguous()
    rows, cols = G.shape[-2:]
    batch = G.shape[:-2].numel()
    out = torch.empty_like(G)
    L, code = _cabi.load(), _cabi.DTYPE_CODE[G.dtype]
    with _cabi.device_of(G):
        nws = L.gnk_orthogonalize_workspace_bytes_of(code, batch, rows, cols)
        ws = torch.empty(nws, dtype=torch.uint8, device=G.device) if nws else None
        rc = L.gnk_orthogonalize(G.data_ptr(), code, out.data_ptr(), code, batch, rows, cols, steps, a, b, c, eps, ws.data_ptr() if nws else None, nws,
                                 _cabi.stream_of(G))
    _cabi.check(rc, "orthogonalize")
    return out
