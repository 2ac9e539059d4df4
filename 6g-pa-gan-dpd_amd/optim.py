"""Muon: momentum, Newton-Schulz iteration and weight update of whole matrices on the device (csrc/orthogonal.hip)."""
import ctypes
from typing import Dict, Optional

import torch

from . import _lib as L
from .utils.orthogonal import COEFFICIENTS, Coefficients, coefficient_table, wants_accurate

_PTR, _I64 = ctypes.c_void_p, ctypes.c_int64


class Muon(torch.optim.Optimizer):
    """For every weight matrix W with gradient G and momentum M (fp32):

        M <- momentum M + G;   U = G + momentum M  (nesterov)  or  M
        W <- W (1 - lr weight_decay) - lr sqrt(max(1, rows / cols)) O(U),   O = `dpd_amd.utils.orthogonalize`

    Parameters that are not matrices (biases) are updated by torch's Adam with the options in `adam`; both kinds are groups
    of this optimiser, so schedulers and state_dict() cover them.  `params`: tensors, or groups with options of their own.
    The steps of all matrices of up to 64 x 128 take one launch (24 at a time); larger ones a handful each.  Every result is
    the same in every run."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0, steps: int = 5,
                 coefficients: Coefficients = COEFFICIENTS, eps: float = 1e-7, accurate: Optional[bool] = None, adam: Optional[Dict] = None):
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f"momentum must lie in [0, 1), got {momentum}")
        if lr < 0.0 or weight_decay < 0.0 or not eps > 0.0:
            raise ValueError(f"lr and weight_decay must not be negative and eps must be positive, got {lr}, {weight_decay}, {eps}")
        coefficient_table(coefficients, steps)
        defaults = dict(kind="matrix", lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                        coefficients=coefficients, eps=eps, accurate=accurate)
        params = list(params)
        given = params if params and isinstance(params[0], dict) else [{"params": params}]
        groups, others = [], []
        for g in given:
            ps = [g["params"]] if isinstance(g["params"], torch.Tensor) else list(g["params"])
            rest = {k: v for k, v in g.items() if k != "params"}
            matrices = [p for p in ps if p.dim() == 2]
            if matrices:
                groups.append({**rest, "params": matrices, "kind": "matrix"})
            others += [p for p in ps if p.dim() != 2]
        self._adam = None
        if others:
            self._adam = torch.optim.Adam(others, **(adam if adam is not None else dict(lr=1e-4, betas=(0.0, 0.9), weight_decay=1e-5, fused=True)))
            groups += [{**g, "kind": "other"} for g in self._adam.param_groups]
        super().__init__(groups, defaults)

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # the base class casts state to the type of its parameter; the momentum is fp32 whatever that is
        for saved, group in zip(state_dict["param_groups"], self.param_groups):
            for key, p in zip(saved["params"], group["params"]):
                m = state_dict["state"].get(key, {}).get("momentum_buffer")
                if m is not None:
                    self.state[p]["momentum_buffer"] = m.detach().to(device=p.device, dtype=torch.float32, copy=True).contiguous()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        others = []
        for group in self.param_groups:
            if group["kind"] == "matrix":
                self._matrices(group)
            else:
                others.append(group)
        if others:
            self._adam.param_groups, self._adam.state = others, self.state     # the groups and the state are this optimiser's
            self._adam.step()
        return loss

    def _matrices(self, group):
        sets: Dict = {}
        for p in group["params"]:
            g = p.grad
            if g is None:
                continue
            if p.dim() != 2 or g.is_sparse:
                raise ValueError(f"a weight matrix with a dense gradient is expected, got {tuple(p.shape)}, sparse = {g.is_sparse}")
            L.need_gpu(p, g)
            if p.dtype not in L.TYPES or g.dtype != p.dtype or not p.is_contiguous():
                raise RuntimeError(f"weights must be contiguous float32, bfloat16 or float16 with gradients of their type, got {p.dtype} / {g.dtype}")
            state = self.state[p]
            m = state.get("momentum_buffer")
            if m is None:
                m = state["momentum_buffer"] = torch.zeros_like(p, dtype=torch.float32)
            elif m.dtype != torch.float32 or m.shape != p.shape or not m.is_contiguous() or m.device != p.device:
                raise RuntimeError(f"the momentum of a weight must be a contiguous float32 tensor of its shape on {p.device}, got {m.dtype} {tuple(m.shape)}")
            sets.setdefault((p.dtype, p.device), []).append((p, g.contiguous(), m))
        for (dtype, _), items in sets.items():
            n = len(items)
            ptrs = [(_PTR * n)(*(t[i].data_ptr() for t in items)) for i in range(3)]
            rows, cols = (_I64 * n)(*(t[0].shape[0] for t in items)), (_I64 * n)(*(t[0].shape[1] for t in items))
            acc, steps = wants_accurate(group["accurate"], dtype), int(group["steps"])
            coef = coefficient_table(group["coefficients"], steps)
            with L.device(items[0][0]):
                nbytes = L.lib().dpd_muon_workspace_bytes(n, rows, cols, acc)
                ws = torch.empty(nbytes, dtype=torch.uint8, device=items[0][0].device)
                L.call("dpd_muon_step", n, *ptrs, rows, cols, L.TYPES[dtype], float(group["lr"]), float(group["momentum"]), int(group["nesterov"]),
                       float(group["weight_decay"]), steps, coef, float(group["eps"]), acc, L.c_p(ws.data_ptr()), nbytes, L.stream())
            torch.autograd.graph.increment_version([t[0] for t in items])
