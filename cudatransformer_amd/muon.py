"""Newton-Schulz orthogonalisation and the Muon step over torch device tensors (ctattn_newton_schulz /
ctattn_muon_update_multi of include/ctattn.h)."""
from __future__ import annotations

import torch

from ._capi import _DTYPE_CODE, _check, _ptr, _ptr_table, _stream_handle, last_error, load, on_device

COEFFS = (3.4445, -4.7750, 2.0315)


def _check_mats(name, *ts):
    for t in ts:
        if t.dtype not in (torch.float32, torch.bfloat16, torch.float16) or not t.is_cuda or not t.is_contiguous():
            raise ValueError(f"{name}: tensors must be contiguous float32, bfloat16 or float16 on the GPU")
        if t.device != ts[0].device or t.dtype != ts[0].dtype:
            raise ValueError(f"{name}: dtypes or devices differ")


def _workspace_for(name, need, workspace, device):
    if workspace is None:
        return torch.empty(max(need, 1), dtype=torch.uint8, device=device)
    if not workspace.is_contiguous() or workspace.device != device:
        raise ValueError(f"{name}: workspace must be contiguous on {device}")
    return workspace


def newton_schulz_workspace_bytes(dtype, mats: int, rows: int, cols: int) -> int:
    """Bytes of the workspace of newton_schulz for `mats` matrices."""
    need = load().ctattn_newton_schulz_workspace_bytes(_DTYPE_CODE[dtype], mats, rows, cols)
    if need < 0:
        raise ValueError(last_error())
    return need


def newton_schulz(x, steps: int = 5, coeffs=COEFFS, eps: float = 1e-7, out=None, workspace=None, stream=None):
    """x [..., rows, cols] / (|x| + eps) through `steps` of X <- a X + (b X X^T + c (X X^T)^2) X, each matrix by
    itself: with the default coefficients its singular values end near one.  `out` may be `x`."""
    name = "newton_schulz"
    _check_mats(name, x, *(() if out is None else (out,)))
    if x.dim() < 2:
        raise ValueError(f"{name}: x must be [..., rows, cols], got {tuple(x.shape)}")
    if out is not None and out.shape != x.shape:
        raise ValueError(f"{name}: out must be {list(x.shape)}, got {tuple(out.shape)}")
    a, b, c = (float(v) for v in coeffs)
    rows, cols = x.shape[-2:]
    if x.numel() == 0:
        return torch.empty_like(x) if out is None else out
    mats = x.numel() // (rows * cols)
    need = newton_schulz_workspace_bytes(x.dtype, mats, rows, cols)
    with on_device(x.device, stream):
        out = torch.empty_like(x) if out is None else out
        ws = _workspace_for(name, need, workspace, x.device)
        rc = load().ctattn_newton_schulz(_DTYPE_CODE[x.dtype], _ptr(x), _ptr(out), _ptr(ws), ws.numel() * ws.element_size(),
                                         mats, rows, cols, int(steps), a, b, c, float(eps), _stream_handle(stream))
    if rc == 1:
        raise ValueError(last_error())
    _check(rc, "ctattn_newton_schulz")
    return out


def muon_update(params, grads, moments, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True,
                weight_decay: float = 0.0, scale: float | None = None, steps: int = 5, coeffs=COEFFS,
                eps: float = 1e-7, stream=None):
    """One Muon step, in place on lists of matrices [rows, cols] of one dtype and their moments (float32):
    m <- momentum m + g, u = g + momentum m (nesterov) or m, p <- (1 - lr weight_decay) p - lr scale
    newton_schulz(u).  Matrices of one shape go through the iteration together.  scale: sqrt(max(1,
    rows / cols)) if not given."""
    name = "muon_update"
    if not (len(params) == len(grads) == len(moments)):
        raise ValueError(f"{name}: list lengths differ")
    if not params:
        return
    _check_mats(name, *params, *grads)
    _check_mats(name, *moments)
    shapes = {}
    for i, (p, g, m) in enumerate(zip(params, grads, moments)):
        if p.dim() != 2 or p.shape != g.shape or p.shape != m.shape or m.dtype != torch.float32 or m.device != p.device:
            raise ValueError(f"{name}: matrix {i} needs a gradient and a float32 moment of its shape on its device")
        if p.numel() > 0:
            shapes.setdefault(tuple(p.shape), []).append(i)
    a, b, c = (float(v) for v in coeffs)
    dev, code, lib = params[0].device, _DTYPE_CODE[params[0].dtype], load()
    needs = {}
    for (rows, cols), which in shapes.items():
        needs[rows, cols] = lib.ctattn_muon_update_workspace_bytes(code, len(which), rows, cols)
        if needs[rows, cols] < 0:
            raise ValueError(last_error())
    with on_device(dev, stream):
        # One after the other on the stream, so one workspace serves all shapes.
        ws = torch.empty(max(needs.values(), default=1), dtype=torch.uint8, device=dev)
        for (rows, cols), which in shapes.items():
            s = max(1.0, rows / cols) ** 0.5 if scale is None else float(scale)
            rc = lib.ctattn_muon_update_multi(code, len(which), _ptr_table([params[i] for i in which]),
                                              _ptr_table([grads[i] for i in which]), _ptr_table([moments[i] for i in which]),
                                              _ptr(ws), ws.numel(), rows, cols, float(lr), float(momentum),
                                              int(bool(nesterov)), float(weight_decay), s, int(steps), a, b, c, float(eps),
                                              _stream_handle(stream))
            if rc == 1:
                raise ValueError(last_error())
            _check(rc, "ctattn_muon_update_multi")


class Muon(torch.optim.Optimizer):
    """Muon over matrices (2-D parameters; embeddings and vectors belong to another optimizer): muon_update of
    every parameter that has a gradient, matrices of one shape and dtype together."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, steps: int = 5):
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() != 2:
                    raise ValueError(f"Muon: parameters must be matrices, got {tuple(p.shape)}")

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # The base class gives a 16-bit parameter's state the parameter's type; moments stay float32.
        for group, saved in zip(self.param_groups, state_dict["param_groups"]):
            for p, key in zip(group["params"], saved["params"]):
                if "moment" in state_dict["state"].get(key, {}):
                    self.state[p]["moment"] = state_dict["state"][key]["moment"].to(p.device, torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            kinds = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if "moment" not in self.state[p]:
                    self.state[p]["moment"] = torch.zeros_like(p, dtype=torch.float32)
                kinds.setdefault((p.dtype, p.device), []).append(p)
            for ps in kinds.values():
                muon_update(ps, [p.grad.contiguous() for p in ps], [self.state[p]["moment"] for p in ps], lr=group["lr"],
                            momentum=group["momentum"], nesterov=group["nesterov"], weight_decay=group["weight_decay"],
                            steps=group["steps"])
        return loss


__all__ = ["Muon", "muon_update", "newton_schulz", "newton_schulz_workspace_bytes"]
