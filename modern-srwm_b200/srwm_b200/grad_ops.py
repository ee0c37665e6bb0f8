"""Global gradient norm over many tensors, and clipping by it, in two launches however many tensors there are.

    clip_grad_norm_(parameters, max_norm, error_if_nonfinite=False) -> norm
        the gradients of the parameters times max_norm / (norm + 1e-6) where that is below 1, in place, norm their 2-norm before;
        the same values as torch.nn.utils.clip_grad_norm_ (a NaN among them makes all of them NaN)
    grad_norm(tensors) -> norm
        the 2-norm over all values of a list of tensors

float32 and bfloat16 tensors of one device, mixed; the sum is fp32 over 32 values and fp64 from there on, in a fixed order.  The norm
stays on the device (a 0-dimensional float32 tensor): nothing waits for it.  With several ranks the gradients are all-reduced
first (``dist.GradBucket``; ``GradBucket.clip_`` is the same for the bucket).  CUDA tensors only.
"""
from __future__ import annotations

import torch

from . import _lib as L


def grad_norm(tensors):
    tensors = [t.detach() for t in tensors]
    if not tensors:
        return torch.zeros(())
    r = L.host().grads_norm(tensors, -1.0, False)
    return _checked(tensors, -1.0) if r is NotImplemented else r


def clip_grad_norm_(parameters, max_norm, error_if_nonfinite=False):
    if type(parameters) is not list:
        parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    if not error_if_nonfinite and max_norm >= 0.0:
        r = L.host().grads_norm(parameters, max_norm, True)
        if r is not NotImplemented:
            return r
    return clip_tensors_([p.grad for p in parameters if p.grad is not None], max_norm, error_if_nonfinite)


def clip_tensors_(grads, max_norm, error_if_nonfinite=False):
    """``clip_grad_norm_`` on the gradients themselves."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    if not grads:
        return torch.zeros(())
    grads = list(grads)
    if error_if_nonfinite and not torch.isfinite(norm := grad_norm(grads)):
        raise RuntimeError(f"the norm of the gradients is not finite ({float(norm)}); they have not been scaled")
    r = L.host().grads_norm(grads, max_norm, False)
    return _checked(grads, max_norm) if r is NotImplemented else r


@torch.no_grad()
def _checked(tensors, max_norm):
    device = tensors[0].device
    for t in tensors:
        if t.device.type != "cuda":
            raise RuntimeError("srwm_b200 operators run on CUDA tensors only (no CPU implementation); "
                               f"got a gradient on {t.device}")
        if t.device != device:
            raise RuntimeError(f"gradients on {device} and {t.device}: one device a call")
        if t.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"gradients must be float32 or bfloat16, got {t.dtype}")
        if t.layout is not torch.strided:
            raise TypeError("gradients must be dense tensors")
    plain = [t.detach().as_subclass(torch.Tensor) for t in tensors]
    dense = [t.contiguous() for t in plain]      # (the same memory where it is dense already)
    r = L.host().grads_norm(dense, max_norm, False)
    if r is NotImplemented:
        raise ValueError("gradients overlap in memory (the same one twice, or views of one another)")
    if max_norm >= 0.0:
        for t, d in zip(plain, dense):
            if d is not t and d.data_ptr() != t.data_ptr():
                t.copy_(d)
    return r
