"""Muon for the hidden matrices of a model and AdamW for everything else, as one optimizer.

One optimizer object is what :func:`init_optimizer_state`, :func:`shared_state_for`, DiLoCo's shared state and a
checkpoint take, so a run with Muon joins, resumes and retries like one with AdamW. The Muon part is
:func:`pccl_amd.ops.muon_step`: a handful of HIP launches for all matrices together, and equal bits on every peer that
has equal gradients and makes the same calls. The AdamW part is torch's.
"""
from __future__ import annotations

from typing import Any, Dict, Iterable, List, Sequence, Tuple

import torch

from ..ops.muon import COEFFICIENTS, check_muon, muon_step


class Muon(torch.optim.Optimizer):
    """``matrices``: parameters (or groups of them) that are 2-D, contiguous and whole, for Muon; ``others``: parameters
    or groups for ``torch.optim.AdamW``, whose ``betas`` and ``adamw_eps`` are given here.

    ``adjust_lr="match_rms_adamw"`` scales Muon's step so that the learning rate and weight decay of AdamW fit both
    parts; ``lr`` and ``weight_decay`` are the defaults of all groups. State of a matrix: ``momentum_buffer`` (fp32).
    Sharded parameters (DTensor) are refused: the orthogonal factor of a shard is not the shard of the factor.
    """

    def __init__(self, matrices: Iterable, others: Iterable = (), *, lr: float = 6e-4, weight_decay: float = 0.1,
                 momentum: float = 0.95, nesterov: bool = True, steps: int = 5,
                 coefficients: Sequence[float] = COEFFICIENTS, eps: float = 1e-7,
                 adjust_lr: str = "match_rms_adamw", betas: Tuple[float, float] = (0.9, 0.95),
                 adamw_eps: float = 1e-8, fused: bool = False):
        groups = [dict(g, muon=True) for g in self._groups(matrices)]
        others = self._groups(others)
        if others:
            adamw = torch.optim.AdamW(others, lr=lr, weight_decay=weight_decay, betas=betas, eps=adamw_eps,
                                      fused=fused)
            groups += [dict(g, muon=False) for g in adamw.param_groups]
        defaults = dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov, steps=steps,
                        coefficients=tuple(coefficients), eps=eps, adjust_lr=adjust_lr, muon=True)
        check_muon("Muon", lr, weight_decay, momentum, steps, tuple(coefficients), eps, adjust_lr)
        super().__init__(groups, defaults)
        self._adamw = adamw if others else None

    @staticmethod
    def _groups(params: Iterable) -> List[Dict[str, Any]]:
        params = list(params)
        return params if params and isinstance(params[0], dict) else [{"params": params}] if params else []

    def add_param_group(self, param_group: Dict[str, Any]) -> None:
        if not param_group.get("muon", True) and hasattr(self, "_adamw"):
            raise ValueError("Muon: parameters for AdamW are given to the constructor")
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            if group["muon"]:
                check_muon("Muon", *(group[k] for k in ("lr", "weight_decay", "momentum", "steps", "coefficients",
                                                        "eps", "adjust_lr")))
                for p in group["params"]:
                    if hasattr(p, "placements"):  # not isinstance: importing DTensor takes half a second
                        raise TypeError("Muon: a sharded parameter (DTensor); matrices must be whole")
                    if p.dim() != 2:
                        raise ValueError(f"Muon: a matrix has two dimensions, got a parameter of {tuple(p.shape)}")
        except Exception:
            self.param_groups.pop()
            raise

    def __setstate__(self, state: Dict[str, Any]) -> None:
        """A copy, an unpickled optimizer or one that loaded a checkpoint: the AdamW part follows from the groups."""
        super().__setstate__(state)
        others = [g for g in self.param_groups if not g["muon"]]
        self._adamw = torch.optim.AdamW(others) if others else None

    def load_state_dict(self, state_dict: Dict[str, Any]) -> None:
        super().load_state_dict(state_dict)  # casts state to the parameter's type; the momentum stays fp32
        saved = state_dict["state"]
        at = 0
        for group in self.param_groups:
            for p in group["params"]:
                buf = saved.get(at, {}).get("momentum_buffer")
                if group["muon"] and buf is not None:
                    self.state[p]["momentum_buffer"] = buf.detach().to(p.device, torch.float32).contiguous().clone()
                at += 1

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            if group["muon"]:
                self._muon(group)
        if self._adamw is not None:  # the same groups and state (both are replaced when a checkpoint is loaded)
            self._adamw.param_groups = [g for g in self.param_groups if not g["muon"]]
            self._adamw.state = self.state
            self._adamw.step()
        return loss

    def _muon(self, group: Dict[str, Any]) -> None:
        calls: Dict[tuple, Tuple[list, list, list]] = {}  # one call takes tensors of one device and type
        for p in group["params"]:
            if p.grad is None:
                continue
            if p.grad.is_sparse:
                raise RuntimeError("Muon: sparse gradients are not supported")
            state = self.state[p]
            if "momentum_buffer" not in state:
                state["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            call = calls.setdefault((p.device, p.dtype, p.grad.dtype), ([], [], []))
            for to, t in zip(call, (p, p.grad, state["momentum_buffer"])):
                to.append(t)
        for params, grads, moms in calls.values():
            muon_step(params, grads, moms, lr=float(group["lr"]), weight_decay=group["weight_decay"],
                      momentum=group["momentum"], nesterov=group["nesterov"], steps=group["steps"],
                      coefficients=group["coefficients"], eps=group["eps"], adjust_lr=group["adjust_lr"])
