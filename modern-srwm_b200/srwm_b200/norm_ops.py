"""Root-mean-square norm of the residual stream.

    rms_norm(x, weight, residual=None, eps=1e-6) -> y, or (y, stream) with a residual
        stream = x + residual (rounded to their type),  y = stream / sqrt(mean(stream^2) + eps) * weight

    rms_norm_fp8(x, weight, residual=None, eps=1e-6) -> (q, scale[, stream])
        the same without gradients, y in 8 bits: q (float8_e4m3fn) times scale [..., 1], scale = max |y| / 448 of the row

x and residual [..., D] float32 or bfloat16, rows at any equal distance, D at most 8192; weight [D] float32.  Statistics are fp32;
the norm sees the stream as it is stored.  Gradients reach x, residual and weight, once.  CUDA tensors only.
"""
from __future__ import annotations

import torch

from . import _lib as L
from .scan_ops import _declined, _empty, _like, _tensor


def rms_norm(x, weight, residual=None, eps=1e-6):
    r = L.host().rms_norm(x, weight, residual, eps, False)
    return _checked(x, weight, residual, eps, False) if r is NotImplemented else r


def rms_norm_fp8(x, weight, residual=None, eps=1e-6):
    r = L.host().rms_norm(x, weight, residual, eps, True)
    return _checked(x, weight, residual, eps, True) if r is NotImplemented else r


def _checked(x, weight, residual, eps, fp8):
    x = _tensor("x", x)
    if x.device.type != "cuda":
        raise RuntimeError("srwm_b200 operators run on CUDA tensors only (no CPU implementation); "
                           f"got x on {x.device}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"x must be float32 or bfloat16, got {x.dtype}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 8192:
        raise ValueError(f"x must be [..., D] with D from 1 to 8192, got {tuple(x.shape)}")
    weight = _like("weight", weight, x.shape[-1:], torch.float32, x.device)
    residual = None if residual is None else _like("residual", residual, x.shape, x.dtype, x.device)
    if fp8 and torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise ValueError("rms_norm_fp8 has no gradient: call it under torch.no_grad()")
    if x.numel() == 0:
        y = (torch.empty_like(x, dtype=torch.float8_e4m3fn), x.new_empty((*x.shape[:-1], 1), dtype=torch.float32)) if fp8 \
            else (_empty(torch.empty_like(x.detach()), x, weight, residual),)
        y += () if residual is None else (_empty(torch.empty_like(x.detach()), x, residual),)
        return y if len(y) > 1 else y[0]
    r = L.host().rms_norm(x.contiguous(), weight.contiguous(), None if residual is None else residual.contiguous(), eps, fp8)
    return _declined("rms_norm") if r is NotImplemented else r
