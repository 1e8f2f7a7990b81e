"""Muon: momentum with orthogonalised updates, for the matrices of a policy.

    m <- momentum m + grad;  u = grad + momentum m (nesterov) or m
    W <- (1 - lr weight_decay) W - lr sqrt(max(1, rows / cols)) orthogonalize(u)

Momentum is a running sum and is kept in fp32 whatever the parameters' type.
Matrices of one shape are orthogonalised as one batch
(:func:`nesle_b200.ops.orthogonalize`).  Vectors, embeddings and output layers
belong to another optimiser.  No counterpart in the reference.
"""
from __future__ import annotations

import torch

from . import ops

__all__ = ["Muon"]


class Muon(torch.optim.Optimizer):
    """``params``: 2-D CUDA parameters (float32, bfloat16 or float16).  ``lr`` is the spectral size of a step."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                 steps: int = 5):
        if lr < 0 or weight_decay < 0:
            raise ValueError("lr and weight_decay must not be negative")
        if not 0 <= momentum < 1:
            raise ValueError("momentum must be in [0, 1)")
        if steps < 1:
            raise ValueError("steps must be at least 1")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() != 2:
                    raise ValueError(f"Muon takes matrices, got a parameter of shape {tuple(p.shape)}")

    def load_state_dict(self, state_dict) -> None:
        super().load_state_dict(state_dict)
        # torch has cast the state to the parameters' type
        saved = [i for group in state_dict["param_groups"] for i in group["params"]]
        for i, p in zip(saved, (p for group in self.param_groups for p in group["params"])):
            momentum = state_dict["state"].get(i, {}).get("momentum")
            if momentum is not None:
                self.state[p]["momentum"] = momentum.to(device=p.device, dtype=torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            alike: dict[tuple, list[torch.Tensor]] = {}
            for p in group["params"]:
                if p.grad is not None and p.numel():
                    alike.setdefault((p.shape, p.dtype, p.device), []).append(p)
            for (shape, _, _), params in alike.items():
                grads = [p.grad for p in params]
                buffers = []
                for p in params:
                    state = self.state[p]
                    if "momentum" not in state:
                        state["momentum"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format)
                    buffers.append(state["momentum"])
                torch._foreach_mul_(buffers, group["momentum"])
                torch._foreach_add_(buffers, grads)
                updates = torch._foreach_add(grads, buffers, alpha=group["momentum"]) if group["nesterov"] else buffers
                stacked = updates[0][None] if len(updates) == 1 else torch.stack(updates)
                with torch.cuda.device(params[0].device):
                    directions = ops.orthogonalize(stacked, steps=group["steps"])
                if group["weight_decay"]:
                    torch._foreach_mul_(params, 1.0 - group["lr"] * group["weight_decay"])
                size = group["lr"] * max(1.0, shape[0] / shape[1]) ** 0.5
                torch._foreach_add_(params, [d.to(params[0].dtype) for d in directions.unbind()], alpha=-size)
        return loss
