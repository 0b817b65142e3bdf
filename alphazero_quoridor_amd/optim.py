"""Orthogonalised updates: ``orthogonalize`` (Newton-Schulz products on the matrix cores) and the ``Muon`` optimiser, whose step
-- momentum, orthogonalisation, decay and the weight's update of a whole list of matrices -- is one call of the C ABI
(csrc/qz_ortho.hip: qz_orthogonalize, qz_muon_step).  There is no CPU path."""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _cabi
from .losses import DTYPES, _gpu, _Launch


def _matrix(t, name):
    """[rows, ...] -> [rows, cols] whose rows are contiguous (a view wherever there is one)."""
    _gpu(t, name)
    if t.dim() < 2:
        raise ValueError("%s: a matrix is needed, got the shape %s" % (name, tuple(t.shape)))
    if t.dim() > 2:
        t = t.reshape(t.shape[0], math.prod(t.shape[1:]))  # (no -1: a side may be zero)
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _workspace(lst, count, device):
    size = _cabi.load().qz_orthogonalize_workspace(lst, count)
    return torch.empty(max(size, 1), dtype=torch.uint8, device=device), size


@torch.no_grad()
def orthogonalize(update, steps=5):
    """The Newton-Schulz iterate of ``update`` / |update|_F after ``steps`` (1 .. 16) quintic steps: same singular vectors, singular
    values near 1.  A tensor [rows, ...] (trailing dimensions count as columns), or a list of them, which share their launches.
    float32, bfloat16 or float16; the result has the type and shape of its input."""
    many = isinstance(update, (list, tuple))
    updates = list(update) if many else [update]
    steps = int(steps)
    if not 1 <= steps <= 16:
        raise ValueError("steps = %d is not in 1 .. 16" % steps)
    mats = [_matrix(u, "update") for u in updates]
    outs = [torch.empty(u.shape, dtype=u.dtype, device=u.device) for u in updates]
    for u in updates:
        if u.dtype not in DTYPES:
            raise TypeError("update: %s is not one of float32, bfloat16, float16" % u.dtype)
    for key in dict.fromkeys((u.dtype, u.device) for u in updates):
        lst = [(m, o) for m, o, u in zip(mats, outs, updates) if (u.dtype, u.device) == key and u.numel()]
        if not lst:
            continue
        arr = (_cabi.qz_matrix * len(lst))(*[(m.shape[0], m.shape[1], m.data_ptr(), m.stride(0), o.data_ptr(), m.shape[1]) for m, o in lst])
        ws, size = _workspace(arr, len(lst), key[1])
        with _Launch(key[1]) as stream:
            _cabi.check(_cabi.load().qz_orthogonalize(arr, len(lst), DTYPES[key[0]], steps, ws.data_ptr(), size, stream))
    return outs if many else outs[0]


class Muon(torch.optim.Optimizer):
    """M <- mu M + (1 - mu) G;  U = (1 - mu) G + mu M (Nesterov) or M;  W <- W (1 - lr weight_decay) - lr scale orthogonalize(U).

    Parameters are float32 matrices or convolution weights ([out, ...] counts as [out, the rest]) on one GPU; gradients float32,
    bfloat16 or float16.  ``adjust_lr``: "original" scales a matrix by sqrt(max(1, rows / cols)), "match_rms_adamw" by
    0.2 sqrt(max(rows, cols)), which gives updates the size of Adam's.  ``lr`` may be a one-element float32 tensor on the GPU:
    a captured step follows it."""

    def __init__(self, params, lr=1e-3, momentum=0.95, nesterov=True, weight_decay=0.0, ns_steps=5, adjust_lr="original"):
        if not torch.is_tensor(lr) and not lr >= 0.0:
            raise ValueError("lr = %r" % (lr,))
        if not 0.0 <= momentum < 1.0:
            raise ValueError("momentum = %r is not in [0, 1)" % (momentum,))
        if not weight_decay >= 0.0:
            raise ValueError("weight_decay = %r" % (weight_decay,))
        if not 1 <= int(ns_steps) <= 16:
            raise ValueError("ns_steps = %r is not in 1 .. 16" % (ns_steps,))
        if adjust_lr not in ("original", "match_rms_adamw"):
            raise ValueError("adjust_lr = %r" % (adjust_lr,))
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=bool(nesterov), weight_decay=weight_decay, ns_steps=int(ns_steps),
                                      adjust_lr=adjust_lr))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() < 2 or p.dtype != torch.float32 or not p.is_contiguous():
                    raise ValueError("Muon takes contiguous float32 matrices, got %s %s" % (tuple(p.shape), p.dtype))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            batches = {}
            for p in group["params"]:
                if p.grad is None or p.numel() == 0:
                    continue
                _gpu(p, "parameter")
                if p.grad.is_sparse or p.grad.dtype not in DTYPES:
                    raise TypeError("gradient: %s is not a dense float32, bfloat16 or float16 tensor" % p.grad.dtype)
                state = self.state[p]
                if "momentum_buffer" not in state:
                    state["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                buf = state["momentum_buffer"]
                if buf.shape != p.shape or buf.dtype != torch.float32 or not buf.is_contiguous() or buf.device != p.device or not p.is_contiguous():
                    raise ValueError("a weight and its momentum must be contiguous float32 tensors of one shape and device")
                batches.setdefault((p.grad.dtype, p.device), []).append((p, _matrix(p.grad, "gradient"), buf))
            for (dtype, device), lst in batches.items():
                self._batch(group, dtype, device, lst)
        return loss

    @staticmethod
    def _batch(group, dtype, device, lst):
        lr = group["lr"]
        lr_dev = lr if torch.is_tensor(lr) and lr.is_cuda else None
        if lr_dev is not None and (lr_dev.dtype != torch.float32 or lr_dev.numel() != 1 or lr_dev.device != device):
            raise ValueError("a learning rate on the GPU must be one float32 on the parameters' device")
        adam = group["adjust_lr"] == "match_rms_adamw"
        rows = []
        for p, g, buf in lst:
            m, n = g.shape
            scale = 0.2 * math.sqrt(max(m, n)) if adam else math.sqrt(max(1.0, m / n))
            rows.append((m, n, g.data_ptr(), g.stride(0), 0, 0, buf.data_ptr(), p.data_ptr(), scale))
        arr = (_cabi.qz_matrix * len(rows))(*rows)
        opts = _cabi.qz_muon_opts(0.0 if lr_dev is not None else float(lr), group["momentum"], group["weight_decay"], int(group["nesterov"]),
                                  lr_dev.data_ptr() if lr_dev is not None else 0)
        ws, size = _workspace(arr, len(rows), device)
        with _Launch(device) as stream:
            _cabi.check(_cabi.load().qz_muon_step(arr, len(rows), DTYPES[dtype], group["ns_steps"], C.byref(opts), ws.data_ptr(), size, stream))
        torch.autograd.graph.increment_version([t for p, _, buf in lst for t in (p, buf)])


class Chained:
    """Several optimisers stepped as one (Muon for the hidden matrices, Adam for the rest)."""

    def __init__(self, *optimizers):
        self.optimizers = optimizers

    @property
    def param_groups(self):
        return [g for o in self.optimizers for g in o.param_groups]

    def zero_grad(self, set_to_none=True):
        for o in self.optimizers:
            o.zero_grad(set_to_none=set_to_none)

    def step(self):
        for o in self.optimizers:
            o.step()

    def state_dict(self):
        return {"optimizers": [o.state_dict() for o in self.optimizers]}

    def load_state_dict(self, state):
        if len(state["optimizers"]) != len(self.optimizers):
            raise ValueError("%d optimisers in the state, %d here" % (len(state["optimizers"]), len(self.optimizers)))
        for o, s in zip(self.optimizers, state["optimizers"]):
            o.load_state_dict(s)
