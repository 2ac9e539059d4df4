"""Muon: momentum, Newton-Schulz iteration and weight update of whole matrices on the device (csrc/orthogonal.hip)."""
import ctypes
from typing import Dict, Optional

import torch

from . import _lib as L
from .utils.orthogonal import COEFFICIENTS, Coefficients, coefficient_table

# autograd sees that the weights changed (the public form of the same call walks its argument as a tree first)
_bump_versions = getattr(torch._C, "_increment_version", None) or torch.autograd.graph.increment_version
_PTR, _I64 = ctypes.c_void_p, ctypes.c_int64


def wants_accurate(accurate: Optional[bool], dtype: torch.dtype) -> int:
    """Unless the caller says: fp16 factors for bf16 weights, factors in two terms for the others.  A step is a small part of
    a weight, and the weight's own rounding (2^-8 of the whole) hides what fp16 factors do to it: after a step of lr 0.02, matrices
    of 2048 and 4096 are 1.66e-3 off with either."""
    return int(dtype != torch.bfloat16 if accurate is None else bool(accurate))


_NO_WORKSPACE = 256              # what dpd_muon_workspace_bytes says when no matrix needs one


_ADAM_KEYS = frozenset(torch.optim.Adam([torch.zeros(1)]).defaults)


def _check_options(o):
    """The options of a group of matrices."""
    if not 0.0 <= o["momentum"] < 1.0:
        raise ValueError(f"momentum must lie in [0, 1), got {o['momentum']}")
    if o["lr"] < 0.0 or o["weight_decay"] < 0.0 or not o["eps"] > 0.0:
        raise ValueError(f"lr and weight_decay must not be negative and eps must be positive, got {o['lr']}, {o['weight_decay']}, {o['eps']}")
    coefficient_table(o["coefficients"], o["steps"])


def _listed(params):
    if isinstance(params, set):
        raise TypeError("parameters have to come in an order that is the same in every run; a set has none")
    return [params] if isinstance(params, torch.Tensor) else list(params)


class Muon(torch.optim.Optimizer):
    """For every weight matrix W with gradient G and momentum M (fp32):

        M <- momentum M + G;   U = G + momentum M  (nesterov)  or  M
        W <- W (1 - lr weight_decay) - lr sqrt(max(1, rows / cols)) O(U),   O = `dpd_amd.utils.orthogonalize`

    Parameters that are not matrices (biases) are updated by torch's Adam with the options in `adam`; both kinds are groups
    of this optimiser, so schedulers and state_dict() cover them.  `params`: tensors, or groups with options of their own, which
    hold for the matrices of the group and, where Adam has them (lr, betas, eps, weight_decay, ...), for its other parameters too.
    `accurate`: as for `orthogonalize`, but None means False for bf16 weights, whose own rounding hides the difference.
    The steps of all matrices of up to 64 x 128 take one launch (24 at a time), and so do those of larger ones that fit into a
    compute unit; the others go through tiled products, up to 8 of one size together.  Every result is the same in every run.  A step that is captured into a graph keeps the learning rate it was captured with."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0, steps: int = 5,
                 coefficients: Coefficients = COEFFICIENTS, eps: float = 1e-7, accurate: Optional[bool] = None, adam: Optional[Dict] = None):
        defaults = dict(kind="matrix", lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                        coefficients=coefficients, eps=eps, accurate=accurate)
        _check_options(defaults)
        self._adam_options = dict(adam if adam is not None else dict(lr=1e-4, betas=(0.0, 0.9), weight_decay=1e-5, fused=True))
        params = _listed(params)
        groups, others = [], []
        for g in params if params and isinstance(params[0], dict) else [{"params": params}]:
            ps = _listed(g["params"])
            for to, part in ((groups, [p for p in ps if p.dim() == 2]), (others, [p for p in ps if p.dim() != 2])):
                if part:
                    to.append({**g, "params": part})
        super().__init__(groups + others, defaults)

    def add_param_group(self, param_group):
        """One group for the matrices in it, with its options over the constructor's, and one for the rest, with those of its
        options that Adam knows over the constructor's `adam`."""
        ps = _listed(param_group["params"])
        known = {id(p) for g in self.param_groups for p in g["params"]}
        if len({id(p) for p in ps} | known) != len(ps) + len(known):
            raise ValueError("a parameter is given twice: its update would run twice at once")
        rest = {k: v for k, v in param_group.items() if k != "params"}
        matrices, others = [p for p in ps if p.dim() == 2], [p for p in ps if p.dim() != 2]
        if matrices:
            _check_options({**self.defaults, **rest})
        if others:
            options = {**self._adam_options, **{k: v for k, v in rest.items() if k in _ADAM_KEYS}}
            adam = {**rest, **torch.optim.Adam(others, **options).param_groups[0], "kind": "other"}
        if matrices:
            super().add_param_group({**rest, "params": matrices, "kind": "matrix"})
        if others:
            super().add_param_group(adam)

    def __getstate__(self):
        return {**super().__getstate__(), "_adam_options": self._adam_options}      # a copy takes groups too

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
        # everything is looked at before the first weight changes
        calls, others = [], []
        for group in self.param_groups:
            if group["kind"] == "matrix":
                calls += self._calls(group)
            else:
                others.append(group)
                if any(p.grad is not None and p.grad.is_sparse for p in group["params"]):
                    raise ValueError("a dense gradient is expected")
        if len(calls) > 1:
            for call in calls:
                self._launch(call, check_only=True)
        for call in calls:
            self._launch(call)
        if others:
            adam = getattr(self, "_adam", None)
            if adam is None:
                adam = self._adam = torch.optim.Adam([p for g in others for p in g["params"]])
            adam.param_groups, adam.state = others, self.state                 # the groups and the state are this optimiser's
            adam.step()
        return loss

    def _calls(self, group):
        """What the library is called with for this group's matrices: one call for each type and device."""
        sets: Dict = {}
        types, state, fp32 = L.TYPES, self.state, torch.float32
        seen = last = None
        for p in group["params"]:
            g = p.grad
            if g is None:
                continue
            shape, dtype, device = p.shape, p.dtype, p.get_device()
            if len(shape) != 2 or g.is_sparse:
                raise ValueError(f"a weight matrix with a dense gradient is expected, got {tuple(shape)}, sparse = {g.is_sparse}")
            if device < 0 or g.get_device() != device:
                L.need_gpu(p, g)
            if dtype not in types or g.dtype != dtype or not p.is_contiguous():
                raise RuntimeError(f"weights must be contiguous float32, bfloat16 or float16 with gradients of their type, got {dtype} / {g.dtype}")
            own = state[p]
            m = own.get("momentum_buffer")
            if m is None:
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("the first step of a weight makes its momentum: take one before the capture, a replay would clear it each time")
                m = own["momentum_buffer"] = torch.zeros_like(p, dtype=fp32)
            elif m.dtype != fp32 or m.shape != shape or not m.is_contiguous() or m.get_device() != device:
                raise RuntimeError(f"the momentum of a weight must be a contiguous float32 tensor of its shape on {p.device}, got {m.dtype} {tuple(m.shape)}")
            if (dtype, device) != seen:
                seen = (dtype, device)
                last = sets.get(seen)
                if last is None:
                    last = sets[seen] = ([], [], [], [], [], [], [])
            ps, gs, at_p, at_g, at_m, rows, cols = last
            if not g.is_contiguous():
                g = g.contiguous()
            ps.append(p)
            gs.append(g)                       # a copy has to live until the launch
            at_p.append(p.data_ptr())
            at_g.append(g.data_ptr())
            at_m.append(m.data_ptr())
            rows.append(shape[0])
            cols.append(shape[1])
        for ps, _, at_p, *_ in sets.values():
            if len(set(at_p)) != len(ps):
                raise ValueError("two weights share their memory: their updates would run at once")
        if not sets:
            return []
        steps = int(group["steps"])
        return [(key, lists, group, steps, coefficient_table(group["coefficients"], steps)) for key, lists in sets.items()]

    def _launch(self, call, check_only=False):
        """The call; or, with no matrices, what it says to the options."""
        (dtype, index), (ps, _, at_p, at_g, at_m, rows, cols), group, steps, coef = call
        n = 0 if check_only else len(ps)
        pointers, sizes = _PTR * n, _I64 * n
        if check_only:
            at_p = at_g = at_m = rows = cols = ()
        h_rows, h_cols = sizes(*rows), sizes(*cols)
        acc = wants_accurate(group["accurate"], dtype)
        with L.device(ps[0]):
            nbytes = L.entry("dpd_muon_workspace_bytes")(n, h_rows, h_cols, acc)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=ps[0].device) if nbytes > _NO_WORKSPACE else None
            L.check(L.entry("dpd_muon_step")(
                n, pointers(*at_p), pointers(*at_g), pointers(*at_m), h_rows, h_cols, L.TYPES[dtype], float(group["lr"]),
                float(group["momentum"]), int(group["nesterov"]), float(group["weight_decay"]), steps, coef, float(group["eps"]), acc,
                0 if ws is None else ws.data_ptr(), nbytes, L.raw_stream(index)))
        if not check_only:
            _bump_versions(ps)
