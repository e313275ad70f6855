"""An optimizer whose update is the orthogonalised momentum of each weight matrix (`gn_kernels.orthogonalize`).

The reference's scripts take their optimizers by name from torch, torchao and bitsandbytes (train_utils.py:14-33); this one is written here because
its inner operator is a kernel of this package.  For the matrices of the body -- Linears and stacks of experts (3-D weights: every expert's matrix by
itself); embeddings, norms and biases belong to an element-wise optimizer.  Weights may be MixedPrecisionLinearWeight.
"""
from __future__ import annotations

import torch
from torch import Tensor

from gn_kernels import orthogonalize


def _plain(t: Tensor) -> Tensor:
    return getattr(t, "_data", t) if type(t) is not Tensor else t


# What a call of `orthogonalize` takes at most, so that the memory for the momentum's copies and the operator's workspace does not grow with the number of equal
# layers.  Multiply-adds of one m x m x n product over the stack: one call for all was at most 2 % faster for bf16 2048 x 5632 (383 us a matrix for 8 matrices, 359
# for 16, 352 for 64), 2048 x 2048 and 4096 x 11008 (2 matrices, 2623; 8, 2591).  Elements: for long, narrow matrices.  65535 is the operator's own bound.
_CALL_WORK, _CALL_ELEMENTS, _CALL_MATRICES = 4.0e11, 1 << 28, 65535


def matrices_per_call(rows: int, cols: int, total: int) -> int:
    """Of `total` matrices of this shape, as many as a call of `orthogonalize` takes: calls of nearly the same size, none empty."""
    most = max(1, min(_CALL_MATRICES, int(_CALL_WORK / (min(rows, cols) * rows * cols)), _CALL_ELEMENTS // (rows * cols)))
    return -(-total // -(-total // most)) if total else 1


def _calls(counts, per):
    """Parts (weight, first, last) of weights of so many matrices each, `per` matrices to a call."""
    call, room = [], per
    for i, count in enumerate(counts):
        at = 0
        while at < count:
            n = min(room, count - at)
            call.append((i, at, at + n))
            at, room = at + n, room - n
            if not room:
                yield call
                call, room = [], per
    if call:
        yield call


class Muon(torch.optim.Optimizer):
    """m <- momentum m + g;  u = orthogonalize(g + momentum m) (nesterov) or orthogonalize(m);  p <- (1 - lr weight_decay) p - lr max(1, rows / cols)^0.5 u.

    The momentum m is held in fp32 whatever the weights' type (a bf16 sum would lose gradients below 2^-8 of it).  bf16 gradients: what is orthogonalised is
    rounded once to bf16; fp16: it stays fp32, as the sum may be 1 / (1 - momentum) times the gradients and leave fp16's range.
    Weights of one shape and type share calls of `orthogonalize`: equal layers fill the chip where one matrix does not (`matrices_per_call`)."""

    def __init__(self, params, lr: float = 0.02, *, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0, steps: int = 5,
                 coefficients: tuple[float, float, float] = (3.4445, -4.7750, 2.0315), eps: float = 1e-7):
        if lr < 0 or not 0 <= momentum < 1 or weight_decay < 0:
            raise ValueError(f"Muon: lr {lr}, momentum {momentum}, weight_decay {weight_decay}")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps, coefficients=tuple(coefficients), eps=eps))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.ndim not in (2, 3) or not p.is_floating_point() or 0 in p.shape[-2:]:
                self.param_groups.pop()
                raise ValueError(f"Muon takes matrices and stacks of matrices, not a {p.dtype} parameter of shape {tuple(p.shape)}")

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        saved = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        for i, p in zip(saved, params):          # the base class rounds floating-point state to the weight's type
            if "momentum" in state_dict["state"].get(i, {}):
                self.state[p]["momentum"] = state_dict["state"][i]["momentum"].detach().to(p.device, torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            alike: dict = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                g = _plain(p.grad)
                state = self.state[p]
                if "momentum" not in state:
                    state["momentum"] = torch.zeros_like(g, dtype=torch.float32, memory_format=torch.contiguous_format)
                state["momentum"].mul_(group["momentum"]).add_(g)
                # what is orthogonalised (u) has the gradient's type; fp16 does not hold the sum
                dtype = torch.float32 if g.dtype is torch.float16 else g.dtype
                alike.setdefault((tuple(p.shape[-2:]), dtype, g.device), []).append((_plain(p), *(t if t.ndim == 3 else t[None] for t in (g, state["momentum"]))))
            for ((rows, cols), dtype, _), weights in alike.items():
                counts = [g.shape[0] for _, g, _ in weights]
                for call in _calls(counts, matrices_per_call(rows, cols, sum(counts))):
                    u = [(torch.add(g[a:b], m[a:b], alpha=group["momentum"]) if group["nesterov"] else m[a:b]).to(dtype) for i, a, b in call for _, g, m in (weights[i],)]
                    out = orthogonalize(u[0] if len(u) == 1 else torch.cat(u), steps=group["steps"], coefficients=group["coefficients"], eps=group["eps"])
                    at, scale = 0, -group["lr"] * max(1.0, rows / cols) ** 0.5
                    for i, a, b in call:
                        w = weights[i][0] if b - a == counts[i] else weights[i][0][a:b]       # whole where it can be: not every weight class has views
                        if group["weight_decay"]:
                            w.mul_(1 - group["lr"] * group["weight_decay"])
                        w.add_(out[at:at + b - a].view(w.shape), alpha=scale)
                        at += b - a
        return loss
