"""Orthogonalised updates: ``orthogonalize`` (Newton-Schulz products on the matrix cores) and the ``Muon`` optimiser, whose step
-- momentum, orthogonalisation, decay and the weight's update of a whole list of matrices -- is one call of the C ABI
(csrc/qz_ortho.hip: qz_orthogonalize, qz_muon_step).  There is no CPU path."""
from __future__ import annotations

import array
import ctypes as C
import math
import struct

import torch
from torch.autograd import forward_ad

from . import _cabi
from .losses import DTYPES, _call, _gpu, _plain


def _matrix(t, name):
    """[rows, ...] -> [rows, cols] whose rows are contiguous (a view wherever there is one)."""
    _gpu(t, name)
    if t.dim() < 2:
        raise ValueError("%s: a matrix is needed, got the shape %s" % (name, tuple(t.shape)))
    t = _plain(t)
    if t.dim() > 2:
        t = t.reshape(t.shape[0], math.prod(t.shape[1:]))  # (no -1: a side may be zero)
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


class _List:
    """qz_matrix[]: nine 8-byte words a matrix (the last one holds a float), written as one run of integers."""

    def __init__(self, words, device):
        self.words = array.array("q", words)
        self.count = len(words) // 9
        self.ptr = C.cast(self.words.buffer_info()[0], C.POINTER(_cabi.qz_matrix))
        self.size = _cabi.load().qz_orthogonalize_workspace(self.ptr, self.count)
        if self.size < 0:
            _cabi.check(self.size)
        self.ws = torch.empty(max(self.size, 1), dtype=torch.uint8, device=device)


def _float_word(v):
    return struct.unpack("q", struct.pack("fi", v, 0))[0]


def _constant(t, name):
    """The result carries no derivative: an input that asks for one is refused."""
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError("%s requires grad, but the result is a constant: detach it" % name)
    if forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError("%s: orthogonalisation has no forward-mode derivative" % name)


def orthogonalize(update, steps=5):
    """The Newton-Schulz iterate of ``update`` / |update|_F after ``steps`` (1 .. 16) quintic steps: same singular vectors, singular
    values near 1.  A tensor [rows, ...] (trailing dimensions count as columns), or a list of them, which share their launches.
    float32, bfloat16 or float16; the result has the type and shape of its input.  Not differentiable: an update that requires grad is
    refused (outside torch.no_grad()), and so is one with a forward-mode tangent."""
    many = isinstance(update, (list, tuple))
    updates = list(update) if many else [update]
    steps = int(steps)
    if not 1 <= steps <= 16:
        raise ValueError("steps = %d is not in 1 .. 16" % steps)
    outs, batches, keep = [], {}, []
    for u in updates:
        _gpu(u, "update")
        _constant(u, "update")
        m = _matrix(u, "update")
        if u.dtype not in DTYPES:
            raise TypeError("update: %s is not one of float32, bfloat16, float16" % u.dtype)
        o = torch.empty(u.shape, dtype=u.dtype, device=u.device)
        outs.append(o)
        keep.append(m)  # (may be a copy: it lives until the launches are queued)
        rows, cols = m.shape
        if rows and cols:
            batches.setdefault((u.dtype, u.device), []).extend((rows, cols, m.data_ptr(), m.stride(0), o.data_ptr(), cols, 0, 0, 0))
    for (dtype, device), words in batches.items():
        lst = _List(words, device)
        _call(device, _cabi.load().qz_orthogonalize, lst.ptr, lst.count, DTYPES[dtype], steps, lst.ws.data_ptr(), lst.size)
    return outs if many else outs[0]


class Muon(torch.optim.Optimizer):
    """M <- mu M + (1 - mu) G;  U = (1 - mu) G + mu M (Nesterov) or M;  W <- W (1 - lr weight_decay) - lr scale orthogonalize(U).

    Parameters are float32 matrices or convolution weights ([out, ...] counts as [out, the rest]) on one GPU; gradients float32,
    bfloat16 or float16.  ``adjust_lr``: "original" scales a matrix by sqrt(max(1, rows / cols)), "match_rms_adamw" by
    0.2 sqrt(max(rows, cols)), which gives updates the size of Adam's.  A step can be captured into a HIP graph once a first one has
    made the momentum buffers; ``lr`` may then be a one-element float32 tensor on the GPU, which the replays follow (a number is
    recorded as it is)."""

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

    def add_param_group(self, group):
        super().add_param_group(group)
        params = self.param_groups[-1]["params"]
        for p in params:
            if p.dim() < 2 or p.dtype != torch.float32 or not p.is_contiguous():
                raise ValueError("Muon takes contiguous float32 matrices, got %s %s" % (tuple(p.shape), p.dtype))
        if len({id(p) for p in params}) < len(params):
            raise ValueError("the same parameter twice")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            adam, batches, changed = group["adjust_lr"] == "match_rms_adamw", {}, []
            for p in group["params"]:
                g = p.grad
                if g is None or p.numel() == 0:
                    continue
                if g.layout is not torch.strided or g.dtype not in DTYPES:
                    raise TypeError("gradient: %s is not a dense float32, bfloat16 or float16 tensor" % g.dtype)
                state = self.state[p]
                buf = state.get("momentum_buffer")
                if buf is None:
                    _gpu(p, "parameter")
                    if torch.cuda.is_current_stream_capturing():
                        # (the capture would record the zeroing, and every replay forget the momentum)
                        raise RuntimeError("the first step makes the momentum buffers: take one step before the capture")
                    buf = state["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                if buf.shape != p.shape or buf.dtype is not torch.float32 or p.dtype is not torch.float32 or buf.device != p.device \
                        or not buf.is_contiguous() or not p.is_contiguous():
                    raise ValueError("a weight and its momentum must be contiguous float32 tensors of one shape and device")
                m = _matrix(g, "gradient")
                rows, cols = m.shape
                scale = 0.2 * math.sqrt(max(rows, cols)) if adam else math.sqrt(rows / cols) if rows > cols else 1.0
                words, keep = batches.setdefault((g.dtype, p.device), ([], []))
                words.extend((rows, cols, m.data_ptr(), m.stride(0), 0, 0, buf.data_ptr(), p.data_ptr(), _float_word(scale)))
                keep.append(m)
                changed += (p, buf)
            for (dtype, device), (words, _) in batches.items():
                self._batch(group, dtype, device, words)
            if changed:
                torch.autograd.graph.increment_version(changed)
        return loss

    @staticmethod
    def _batch(group, dtype, device, words):
        lr = group["lr"]
        lr_dev = lr if torch.is_tensor(lr) and lr.is_cuda else None
        if lr_dev is not None and (lr_dev.dtype != torch.float32 or lr_dev.numel() != 1 or lr_dev.device != device):
            raise ValueError("a learning rate on the GPU must be one float32 on the parameters' device")
        opts = _cabi.qz_muon_opts(0.0 if lr_dev is not None else float(lr), group["momentum"], group["weight_decay"], int(group["nesterov"]),
                                  lr_dev.data_ptr() if lr_dev is not None else 0)
        spans = sorted(zip(words[7::9], words[0::9], words[1::9]))
        if any(at + 4 * rows * cols > above[0] for (at, rows, cols), above in zip(spans, spans[1:])):
            raise ValueError("two parameters share their memory: their updates would race")
        lst = _List(words, device)
        _call(device, _cabi.load().qz_muon_step, lst.ptr, lst.count, DTYPES[dtype], group["ns_steps"], opts, lst.ws.data_ptr(), lst.size)


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
