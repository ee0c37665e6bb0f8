"""Global gradient norm over many tensors, and clipping by it, in two launches for each 1024 of them.

    clip_grad_norm_(parameters, max_norm, error_if_nonfinite=False) -> norm
        the gradients of the parameters times max_norm / (norm + 1e-6) where that is below 1, in place, norm their 2-norm before;
        the same values as torch.nn.utils.clip_grad_norm_ (a NaN among them makes all of them NaN)
    grad_norm(tensors) -> norm
        the 2-norm over all values of a list of tensors (which may share memory; gradients that are clipped may not)

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
    grads = list(grads)
    if not grads:
        return torch.zeros(())
    if error_if_nonfinite and not torch.isfinite(norm := grad_norm(grads)):
        raise RuntimeError(f"the norm of the gradients is not finite ({float(norm)}); they have not been scaled")
    r = L.host().grads_norm(grads, max_norm, False)
    return _checked(grads, max_norm) if r is NotImplemented else r


def _bytes(t):
    """[(distance, count)] of a tensor's bytes, the largest distance first."""
    if t.is_contiguous():
        return [(1, t.numel() * t.element_size())]
    dims = [(st * t.element_size(), n) for st, n in zip(t.stride(), t.shape) if n > 1] + [(1, t.element_size())]
    return sorted(dims, reverse=True)


def _meet(delta, dims):
    """Whether sum_k d_k distance_k = delta for some d_k from low_k to high_k; dims: (distance, low, high), the largest distance first."""
    if not dims:
        return delta == 0
    (st, low, high), rest = dims[0], dims[1:]
    if st == 0:
        return _meet(delta, rest)
    first = max(low, -((sum(s * h for s, _, h in rest) - delta) // st))
    last = min(high, (delta - sum(s * l for s, l, _ in rest)) // st)
    return any(_meet(delta - d * st, rest) for d in range(first, last + 1))


def _overlap(tensors):
    """Whether a byte belongs to two values of these tensors (of one of them, where its dimensions are not nested, is taken to)."""
    spans = []
    for t in tensors:
        if t.numel() == 0:
            continue
        dims, extent = _bytes(t), 0
        for st, n in reversed(dims):
            if st <= extent:
                return True
            extent += st * (n - 1)
        spans.append((t.data_ptr(), t.data_ptr() + extent, dims))
    spans.sort(key=lambda s: s[:2])
    for i, (a, end, da) in enumerate(spans):
        for b, _, db in spans[i + 1:]:
            if b > end:
                break
            both = [(st, 0, n - 1) for st, n in da] + [(st, 1 - n, 0) for st, n in db]
            if _meet(b - a, sorted(both, reverse=True)):
                return True
    return False


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
    if max_norm >= 0.0 and _overlap(plain):
        raise ValueError("gradients overlap in memory (the same one twice, views of one another or an expanded one)")
    dense = [t.contiguous() for t in plain]      # (the same memory where it is dense already)
    r = L.host().grads_norm(dense, max_norm, False)
    if r is NotImplemented:
        raise RuntimeError("these gradients cannot be used")
    if max_norm >= 0.0:
        for t, d in zip(plain, dense):
            if d is not t and d.data_ptr() != t.data_ptr():
                t.copy_(d)
    return r
