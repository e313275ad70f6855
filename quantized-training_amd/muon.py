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


class Muon(torch.optim.Optimizer):
    """m <- momentum m + g;  u = orthogonalize(g + momentum m) (nesterov) or orthogonalize(m);  p <- (1 - lr weight_decay) p - lr max(1, rows / cols)^0.5 u.

    The momentum m is held in fp32 whatever the weights' type (a bf16 sum would lose gradients below 2^-8 of it).  bf16 gradients: what is orthogonalised is
    rounded once to bf16; fp16: it stays fp32, as the sum may be 1 / (1 - momentum) times the gradients and leave fp16's range.
    Weights of one shape and type share a call of `orthogonalize`: equal layers fill the chip where one matrix does not."""

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
                m = state["momentum"].mul_(group["momentum"]).add_(g)
                u = (torch.add(g, m, alpha=group["momentum"]) if group["nesterov"] else m).to(torch.float32 if g.dtype is torch.float16 else g.dtype)
                alike.setdefault((tuple(p.shape[-2:]), u.dtype, u.device), []).append((p, u))
            for (shape, _, _), pairs in alike.items():
                # one stack of all matrices of this shape; a single one goes as it is
                stack = pairs[0][1] if len(pairs) == 1 else torch.cat([u.reshape(-1, *shape) for _, u in pairs])
                out = orthogonalize(stack, steps=group["steps"], coefficients=group["coefficients"], eps=group["eps"]).reshape(-1, *shape)
                at, scale = 0, -group["lr"] * max(1.0, shape[0] / shape[1]) ** 0.5
                for p, u in pairs:
                    n = u.numel() // (shape[0] * shape[1])
                    w = _plain(p)
                    if group["weight_decay"]:
                        w.mul_(1 - group["lr"] * group["weight_decay"])
                    w.add_(out[at:at + n].view(w.shape), alpha=scale)
                    at += n
        return loss
