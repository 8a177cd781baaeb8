"""Optimisers whose updates run on liblic."""
from __future__ import annotations

import math
from typing import Iterable, List, Tuple

import torch
import torch.nn as nn

from . import functional as Fn

__all__ = ["Muon", "Together", "split_muon_params"]


def split_muon_params(module: nn.Module, params: Iterable[torch.Tensor]) -> Tuple[List[torch.Tensor], List[torch.Tensor]]:
    """(matrices, others) of ``params``: the weights of module's dense convolutions, transposed convolutions and Linears
    with at least 8 rows and columns, and everything else (biases, GDN parameters, bias tables, depthwise filters)."""
    dense = set()
    for m in module.modules():
        if isinstance(m, (nn.Conv2d, nn.ConvTranspose2d, nn.Linear)) and getattr(m, "groups", 1) == 1:
            w = m.weight
            if min(w.shape[0], w[0].numel()) >= 8:
                dense.add(id(w))
    params = list(params)
    return [p for p in params if id(p) in dense], [p for p in params if id(p) not in dense]


class Muon(torch.optim.Optimizer):
    """Momentum whose update is orthogonalised (functional.orthogonalize): every weight moves by
    lr * scale * NewtonSchulz(u), u the (Nesterov) momentum of its gradient as a matrix [shape[0], rest].

    ``adjust``: 'rms' scales by 0.2 sqrt(max(rows, cols)), an update of root mean square about 0.2 whatever the shape
    (Adam's learning rates carry over); 'shape' by sqrt(max(1, rows / cols)).  ``weight_decay`` is decoupled.  The
    momentum is fp32, all matrices of a dtype are orthogonalised in the same few launches, and the result is the same
    bits on every rank that holds the same gradients.  ``lr`` may be a device scalar: the step then captures into a
    hipGraph (after one eager step, which creates the momentum)."""

    def __init__(self, params, lr=1e-3, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                 steps: int = 5, adjust: str = "rms", eps: float = 1e-7):
        if not isinstance(lr, torch.Tensor) and not lr >= 0:
            raise ValueError(f"Muon: lr must be >= 0, got {lr}")
        if not 0 <= momentum < 1 or not weight_decay >= 0:
            raise ValueError("Muon: momentum in [0, 1), weight_decay >= 0")
        if adjust not in ("rms", "shape"):
            raise ValueError(f"Muon: adjust must be 'rms' or 'shape', got {adjust!r}")
        if not 1 <= steps <= 64 or not eps >= 0:
            raise ValueError("Muon: steps from 1 to 64, eps >= 0")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay,
                                      steps=steps, adjust=adjust, eps=eps))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        if any(p.dim() < 2 for p in self.param_groups[-1]["params"]):
            del self.param_groups[-1]
            raise ValueError("Muon: matrices and filters only (give vectors to another optimiser)")

    @staticmethod
    def _scale(adjust: str, rows: int, cols: int) -> float:
        return 0.2 * math.sqrt(max(rows, cols)) if adjust == "rms" else math.sqrt(max(1.0, rows / cols))

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # the base class casts floating state to the parameter's dtype: the momentum stays fp32
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        for i, p in zip(ids, params):
            saved = state_dict["state"].get(i, {})
            if "momentum" in saved:
                self.state[p]["momentum"] = saved["momentum"].detach().to(device=p.device, dtype=torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None and p.numel()]
            if not params:
                continue
            Fn._on_current_device("Muon", *params)
            lr, mu, wd = group["lr"], group["momentum"], group["weight_decay"]
            new = [p for p in params if "momentum" not in self.state[p]]
            if new and torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("Muon: capture after one eager step of these parameters (a graph that creates their "
                                   "momentum would set it to zero at every replay)")
            for p in new:
                self.state[p]["momentum"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            bufs = [self.state[p]["momentum"] for p in params]
            grads = [p.grad.float() for p in params]
            # m <- mu m + (1 - mu) g;  u = mu m + (1 - mu) g (Nesterov) or m
            torch._foreach_lerp_(bufs, grads, 1.0 - mu)
            ups = torch._foreach_lerp(bufs, grads, 1.0 - mu) if group["nesterov"] else bufs
            mats = [u.reshape(u.shape[0], -1) for u in ups]
            orth = Fn.orthogonalize(mats, steps=group["steps"], eps=group["eps"])
            orth = [o.view(p.shape) for o, p in zip(orth, params)]   # fp32: only the new weight is rounded to its type
            torch._foreach_mul_(orth, [self._scale(group["adjust"], *m.shape) for m in mats])
            if wd:
                # weights of other types: the decay joins the fp32 update, a multiply of its own would round it away
                exact = [p for p in params if p.dtype == torch.float32]
                if exact:
                    torch._foreach_mul_(exact, 1.0 - lr * wd)
                for p, o in zip(params, orth):
                    if p.dtype != torch.float32:
                        o.add_(p.float(), alpha=wd)
            if isinstance(lr, torch.Tensor):
                torch._foreach_mul_(orth, lr)
                torch._foreach_sub_(params, orth)
            else:
                torch._foreach_sub_(params, orth, alpha=lr)
        return loss


class Together(torch.optim.Optimizer):
    """Several optimisers as one: a GradScaler decides once whether the gradients are finite and all of them step or none,
    and one scheduler sets every learning rate.  The parameter groups are the optimisers' own, those that one of them is
    given later included."""

    def __init__(self, *optimizers: torch.optim.Optimizer):
        if not optimizers:
            raise ValueError("Together: at least one optimiser")
        super().__init__([g for o in optimizers for g in o.param_groups], {})
        self.optimizers = optimizers
        del self._at_first

    @property
    def param_groups(self):
        return [g for o in self.optimizers for g in o.param_groups] if "optimizers" in self.__dict__ else self._at_first

    @param_groups.setter
    def param_groups(self, groups):   # the base class' list while it checks the optimisers' groups against each other
        self._at_first = groups

    def __getstate__(self):   # copies and pickles: the groups are in the optimisers
        return {"defaults": self.defaults, "state": self.state, "optimizers": self.optimizers}

    def add_param_group(self, param_group):
        if "optimizers" in self.__dict__:
            raise ValueError("Together: give the group to one of its optimisers (optimizers[i].add_param_group)")
        super().add_param_group(param_group)

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for o in self.optimizers:
            o.step()
        return loss

    def state_dict(self):
        return {"optimizers": [o.state_dict() for o in self.optimizers]}

    def load_state_dict(self, state_dict):
        if len(state_dict["optimizers"]) != len(self.optimizers):
            raise ValueError("Together: a state of other optimisers")
        for o, s in zip(self.optimizers, state_dict["optimizers"]):
            o.load_state_dict(s)
