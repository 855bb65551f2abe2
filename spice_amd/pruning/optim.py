"""Adam that clips the global gradient norm as it reads the gradients: the norm's launch, then one launch that updates
every tensor; the clipped gradients are never written and the host never waits for the norm.  The reference's fine-tune
loop steps torch's Adam without clipping (pruning/trainer.py:160-228); the trainer takes this optimiser where
`max_grad_norm` is set."""
from __future__ import annotations

from typing import Dict, Optional, Tuple

import torch

from .. import ops


# what torch.optim.Adam's groups hold beside this class's options
_ADAM_ONLY = {"amsgrad", "maximize", "foreach", "capturable", "differentiable", "fused", "decoupled_weight_decay"}


class ClippedAdam(torch.optim.Optimizer):
    """Parameters and gradients fp32 / fp16 / bf16 on one HIP device, moments fp32.  `decoupled`: weight decay as
    p *= 1 - lr * weight_decay, else added to the gradient (torch.optim.Adam's way).  max_grad_norm: the gradients of
    all groups together count as clipped to that norm; `last_grad_norm` is that norm of the last step, a device scalar."""

    def __init__(self, params, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.0, decoupled: bool = False, max_grad_norm: Optional[float] = None):
        if not lr >= 0.0 or not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError("lr, eps and weight_decay must not be negative")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"betas must lie in [0, 1), got {betas}")
        if max_grad_norm is not None and not max_grad_norm > 0.0:
            raise ValueError(f"max_grad_norm must be positive, got {max_grad_norm}")
        self.max_grad_norm = max_grad_norm
        self.last_grad_norm: Optional[torch.Tensor] = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, decoupled=decoupled))

    def __getstate__(self) -> dict:      # (the base class keeps its own three attributes alone)
        return {**super().__getstate__(), "max_grad_norm": self.max_grad_norm, "last_grad_norm": self.last_grad_norm}

    def _state_of(self, p: torch.Tensor) -> dict:
        state = self.state[p]
        if not state:
            state["step"] = 0
            for key in ("exp_avg", "exp_avg_sq"):
                state[key] = self._moment_of(p)
        return state

    @staticmethod
    def _moment_of(p: torch.Tensor) -> torch.Tensor:
        return torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format, requires_grad=False)

    def load_state_dict(self, state_dict: dict) -> None:
        """Also a state of torch.optim.Adam or AdamW, but for amsgrad's and maximize's.  The moments stay fp32 (the base
        class would cast them to their parameters' type) and take their parameters' order of axes."""
        groups = []
        for group in state_dict["param_groups"]:
            if group.get("amsgrad") or group.get("maximize"):
                raise ValueError("ClippedAdam has neither amsgrad nor maximize")
            decoupled = group.get("decoupled", group.get("decoupled_weight_decay", self.defaults["decoupled"]))
            groups.append({**{k: v for k, v in group.items() if k not in _ADAM_ONLY}, "decoupled": bool(decoupled)})
        keys = [key for group in groups for key in group["params"]]
        loaded = {}
        for key, p in zip(keys, (p for group in self.param_groups for p in group["params"])):
            saved = state_dict["state"].get(key)
            if not saved:
                continue
            if not {"step", "exp_avg", "exp_avg_sq"} <= set(saved):
                raise ValueError(f"the state of parameter {key} is not Adam's: {sorted(saved)}")
            loaded[p] = {"step": int(saved["step"])}
            for name in ("exp_avg", "exp_avg_sq"):
                if saved[name].shape != p.shape:
                    raise ValueError(f"{name} of parameter {key} has shape {tuple(saved[name].shape)}, its parameter {tuple(p.shape)}")
                loaded[p][name] = self._moment_of(p).copy_(saved[name])
        super().load_state_dict({**state_dict, "state": {}, "param_groups": groups})
        self.state.update(loaded)

    @staticmethod
    def _grad_of(p: torch.Tensor) -> torch.Tensor:
        if p.grad.is_sparse:
            raise RuntimeError("ClippedAdam takes no sparse gradients")
        # the update walks a parameter and its gradient in memory order
        return p.grad if p.grad.stride() == p.stride() or p.numel() <= 1 else torch.empty_like(p).copy_(p.grad)

    @torch.no_grad()
    def step(self, closure=None):
        on_device = any(p.is_cuda for group in self.param_groups for p in group["params"])
        if on_device and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("ClippedAdam counts its steps on the host: capture ops.adam_step with a device step count")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # parameters of a group that have taken as many steps and are of one type go in one launch
        sets: Dict[tuple, list] = {}
        for i, group in enumerate(self.param_groups):
            for p in group["params"]:
                if p.grad is not None:
                    sets.setdefault((i, self._state_of(p)["step"], p.dtype), []).append((p, self._grad_of(p)))
        if not sets:
            return loss
        norm = None
        if self.max_grad_norm is not None and len(sets) > 1:
            norm = ops.grad_norm([g for s in sets.values() for _, g in s], any_type=True)
        for (i, steps, _), members in sets.items():
            group, states = self.param_groups[i], [self.state[p] for p, _ in members]
            got = ops.adam_step([p for p, _ in members], [g for _, g in members], [s["exp_avg"] for s in states],
                                [s["exp_avg_sq"] for s in states], steps + 1, lr=float(group["lr"]), betas=group["betas"],
                                eps=group["eps"], weight_decay=group["weight_decay"], decoupled=group["decoupled"],
                                max_norm=self.max_grad_norm, norm=norm)
            for s in states:
                s["step"] = steps + 1
            self.last_grad_norm = got if norm is None else norm
        return loss
