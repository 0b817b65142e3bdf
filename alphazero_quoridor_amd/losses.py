"""Policy losses on the GPU: log-probabilities of actions under a legal-move mask, and the clipped policy loss with its KL and
entropy terms, each with its gradient (csrc/qz_policy.hip through the C ABI: qz_action_logp, qz_policy_loss; the autograd functions
over them: csrc/qz_autograd.cpp).

``logits`` are [..., A]: any number of decisions over A actions (float32, bfloat16 or float16; log-probabilities serve as
logits too).  ``legal`` is None, a mask of bytes or bools [..., A], or packed 32-bit words [..., ceil(A / 32)] -- what
``rules.movegen`` returns.  Its leading dimensions broadcast.  A decision whose action is negative, out of range, illegal or
has a logit of -inf is left out: no loss, no gradient, no entropy; its log-probability reads 0 for a negative action (padding)
and -inf otherwise.  Illegal columns may hold anything, NaN included.

Derivatives are reverse-mode and first-order: a second derivative and forward-mode tangents are refused (RuntimeError,
NotImplementedError).  There is no CPU path: tensors on another device than a GPU raise ``QzError(QZ_E_NO_DEVICE)``."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _cabi

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_BITS = (torch.int32, torch.uint32)
_BYTES = (torch.bool, torch.uint8)


class PolicyLoss(NamedTuple):
    loss: torch.Tensor     # scalar float32, the only differentiable member
    logp: torch.Tensor     # log pi(a), float32, one per decision; the same for the others
    kl: torch.Tensor       # KL term of every decision (0 without a frozen policy); which one: see clipped_policy_loss
    entropy: torch.Tensor


def _gpu(t, name):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a tensor" % name)
    if not t.is_cuda:
        raise _cabi.QzError(_cabi.E_NO_DEVICE, "%s is on %s; this package has no CPU path" % (name, t.device))


def _plain(t):
    """A lazily negated view (the imaginary part of a conjugate) as the values it stands for: its memory holds the others."""
    return t.resolve_neg() if t.is_neg() else t


def _same_device(t, device, name):
    _gpu(t, name)
    if t.device != device:
        raise ValueError("%s is on %s, the logits on %s" % (name, t.device, device))


def _rows_of(logits, name="logits"):
    """[..., A] -> [n, A] whose rows are contiguous (a view wherever there is one)."""
    _gpu(logits, name)
    if logits.dtype not in DTYPES:
        raise TypeError("%s: %s is not one of float32, bfloat16, float16" % (name, logits.dtype))
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("%s: at least one action is needed, got the shape %s" % (name, tuple(logits.shape)))
    if logits.shape[-1] > 1 << 30:
        raise ValueError("%s: %d actions, at most 2^30 are supported" % (name, logits.shape[-1]))
    logits = _plain(logits)
    return logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])


def _unit_rows(t):
    # (a row stride below the row's length is fine for an input: broadcast rows)
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _vector(t, lead, device, name):
    """A float per decision, constant for the gradient."""
    if t is None:
        return None
    _same_device(t, device, name)
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError("%s requires grad, but the loss treats it as a constant: detach it" % name)
    if not t.is_floating_point():
        raise TypeError("%s must be floating point" % name)
    if tuple(t.shape) != tuple(lead):
        raise ValueError("%s has the shape %s, %s is needed" % (name, tuple(t.shape), tuple(lead)))
    t = _plain(t)
    if t.dtype is torch.float32 and t.dim() == 1 and t.is_contiguous():
        return t
    return t.to(torch.float32).reshape(-1).contiguous()


def _actions(t, lead, device):
    _same_device(t, device, "actions")
    if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
        raise TypeError("actions must be integers")
    if tuple(t.shape) != tuple(lead):
        raise ValueError("actions have the shape %s, %s is needed" % (tuple(t.shape), tuple(lead)))
    t = _plain(t)
    if t.dtype is torch.int64 and t.dim() == 1 and t.is_contiguous():
        return t
    return t.to(torch.int64).reshape(-1).contiguous()


def _legal(t, lead, a, device):
    """-> (tensor [n, words or bytes] or None, kind)"""
    if t is None:
        return None, 0
    _same_device(t, device, "legal")
    kind, width = (1, (a + 31) // 32) if t.dtype in _BITS else (2, a) if t.dtype in _BYTES else (0, 0)
    if not kind:
        raise TypeError("legal: %s is neither packed 32-bit words nor bytes" % t.dtype)
    if t.dim() < 1 or t.shape[-1] != width:
        raise ValueError("legal has the shape %s, its last dimension must be %d" % (tuple(t.shape), width))
    if t.dim() != 2 or len(lead) != 1 or t.shape[0] != lead[0]:
        t = t.expand(tuple(lead) + (width,)).reshape(-1, width)
    return _unit_rows(t), kind


def _autograd():
    """The autograd functions (csrc/qz_autograd.cpp, built beside the library)."""
    global _ext
    if _ext is None:
        _cabi.load()
        try:
            from . import _autograd as ext
        except ImportError as e:
            raise _cabi.QzLibraryError("_autograd.so is missing or does not load (%s). Build it with `make -C %s`." % (e, _cabi.CSRC)) from e
        _ext = ext
    return _ext


_ext = None


def _checked(call, *args):
    try:
        return call(*args)
    except RuntimeError as e:
        text = str(e)
        if text.startswith("libqzero_hip error "):  # the library's own refusal, as everywhere in this package
            code, _, rest = text[len("libqzero_hip error "):].partition(": ")
            raise _cabi.QzError(int(code), rest.splitlines()[0]) from None
        raise


class _Launch:
    """The tensor's device made current (only if it is not), and its current stream."""

    def __init__(self, device):
        self.guard = torch.cuda.device(device) if torch.cuda.current_device() != device.index else None
        self.device = device

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return torch.cuda.current_stream(self.device).cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _call(device, fn, *args):
    """fn(*args, stream) of the library on the device's current stream (a raw handle: wrapping it in a Stream costs 3 us)."""
    if torch.cuda.current_device() == device.index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(device.index))
    else:
        with _Launch(device) as stream:
            rc = fn(*args, stream)
    if rc:
        _cabi.check(rc)


def _refuse_captured_leaf(logits):
    # the backward pass of a leaf runs on the stream that the leaf's gradient was first accumulated on: inside a capture that
    # may be a stream outside of it, which ends the process
    if logits.is_leaf and logits.requires_grad and torch.is_grad_enabled() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("logits that are leaves cannot be differentiated inside a graph capture: use policy_loss_and_grad, or let "
                           "the network that makes them run inside the capture too")


def action_logp(logits, actions, legal=None, entropy=False):
    """log pi(action) of every decision, float32 with the shape of ``actions``; with ``entropy=True`` a pair of that and the
    entropy of the distribution over the legal actions.  Differentiable in ``logits``."""
    lead = tuple(logits.shape[:-1]) if isinstance(logits, torch.Tensor) else ()
    z = _rows_of(logits)
    _refuse_captured_leaf(logits)
    acts = _actions(actions, lead, z.device)
    mask, kind = _legal(legal, lead, z.shape[1], z.device)
    logp, ent = _checked(_autograd().action_logp, _unit_rows(z), acts, mask, kind, bool(entropy))
    if len(lead) != 1:
        logp, ent = logp.reshape(lead), ent.reshape(lead) if entropy else None
    return (logp, ent) if entropy else logp


def _loss_arguments(logits, actions, advantages, old_logp, legal, weights, ref_logits, ref_logp, clip, kl_coef, entropy_coef):
    z = _rows_of(logits)
    lead, device = tuple(logits.shape[:-1]), z.device
    low, high = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    low, high = float(low), float(high)
    if not (0.0 <= low <= 1.0 and high >= 0.0):
        raise ValueError("clip = %r: the ratio's range is [1 - low, 1 + high] with 0 <= low <= 1 and high >= 0" % (clip,))
    if ref_logits is not None and ref_logp is not None:
        raise ValueError("ref_logits and ref_logp exclude each other")
    ref = None
    if ref_logits is not None:
        _same_device(ref_logits, device, "ref_logits")
        if ref_logits.requires_grad and torch.is_grad_enabled():
            raise ValueError("ref_logits require grad, but the loss treats them as constants: detach them")
        if ref_logits.shape != logits.shape or ref_logits.dtype != logits.dtype:
            raise ValueError("ref_logits: %s %s, the logits are %s %s" % (tuple(ref_logits.shape), ref_logits.dtype, tuple(logits.shape), logits.dtype))
        ref = _unit_rows(_rows_of(ref_logits, "ref_logits"))
    if advantages is None or old_logp is None:
        raise TypeError("advantages and old_logp are needed")
    mask, kind = _legal(legal, lead, z.shape[1], device)
    return (_unit_rows(z), _actions(actions, lead, device), mask, kind, _vector(advantages, lead, device, "advantages"),
            _vector(old_logp, lead, device, "old_logp"), _vector(ref_logp, lead, device, "ref_logp"), _vector(weights, lead, device, "weights"), ref, low, high,
            float(kl_coef), float(entropy_coef)), lead


def clipped_policy_loss(logits, actions, advantages, old_logp, legal: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None,
                        ref_logits: Optional[torch.Tensor] = None, ref_logp: Optional[torch.Tensor] = None, clip=0.2, kl_coef=0.0,
                        entropy_coef=0.0) -> PolicyLoss:
    """sum_i w_i [ -min(r A, clip(r, 1 - low, 1 + high) A) + kl_coef KL - entropy_coef H ] with r = exp(log pi(a) - old_logp).

    weights: w_i (default 1 / n each; 0 leaves a decision out of the loss).  clip: one number, or (low, high).
    The KL term with ref_logits (same shape and type as the logits): KL(frozen || pi).  With ref_logp, the frozen policy's
    log-probability of the action: e^x - 1 - x with x = ref_logp - log pi(a), which estimates the other direction, KL(pi || frozen),
    where actions are drawn from pi.  One kl_coef does not weigh the two alike.
    Differentiable in ``logits``; memory for their gradient is taken in the forward pass."""
    args, lead = _loss_arguments(logits, actions, advantages, old_logp, legal, weights, ref_logits, ref_logp, clip, kl_coef, entropy_coef)
    _refuse_captured_leaf(logits)
    loss, logp, kl, entropy, _ = _checked(_autograd().policy_loss, *args, False)
    return _result(loss, logp, kl, entropy, lead)


def _result(loss, logp, kl, entropy, lead):
    if len(lead) != 1:
        logp, kl, entropy = logp.reshape(lead), kl.reshape(lead), entropy.reshape(lead)
    return PolicyLoss(loss, logp, kl, entropy)


@torch.no_grad()
def policy_loss_and_grad(logits, actions, advantages, old_logp, legal=None, weights=None, ref_logits=None, ref_logp=None, clip=0.2, kl_coef=0.0,
                         entropy_coef=0.0):
    """(PolicyLoss, gradient of its loss in the logits) without the autograd graph: what a captured HIP graph records."""
    args, lead = _loss_arguments(logits, actions, advantages, old_logp, legal, weights, ref_logits, ref_logp, clip, kl_coef, entropy_coef)
    loss, logp, kl, entropy, grad = _checked(_autograd().policy_loss, *args, True)
    return _result(loss, logp, kl, entropy, lead), grad.reshape(logits.shape)
