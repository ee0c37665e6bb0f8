"""Selective state-space scan and the short causal convolution in front of it: a third recurrence beside the SRWM and the
delta rule, with the same uses -- training on whole sequences, the learner's unroll with episode resets, prompts, and single tokens
with the state carried (no reference operator corresponds; the call conventions are those of ``srwm_layer``).

    selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, state=None, done=None,
                   delta_softplus=True, inplace_state=False) -> (y, state)

        Delta = softplus(delta + delta_bias)            (``delta_softplus=False``: as given)
        h_t   = exp(Delta_t A) h_{t-1} + (Delta_t u_t) B_t
        y_t   = (C_t . h_t + D u_t) silu(z_t)           (without ``z``: ungated)

    u, delta, z [N, L, D] float32 or bfloat16; B, C [N, L, S] or, in G groups of D / G neighbouring channels,
    [N, L, G, S], the same type; A [D, S], D, delta_bias [D], state [N, D, S] float32; S is 8, 16, 32 or 64.
    ``done`` [N, L] (bool): the state in front of step t is zero (an episode, or the next of several packed sequences, begins).

    causal_conv(x, weight, bias=None, state=None, done=None, silu=True, inplace_state=False) -> (y, state)

        y_t = silu(bias + sum_i weight[:, K-1-i] x_{t-i})

    x [N, L, D]; weight [D, K] float32, K = 2, 3 or 4; bias [D] float32; state [N, K-1, D] in x's type: the last K - 1
    inputs of the call before.  Nothing is read across an episode's start.

Rows may be any strided views with a dense last dimension (a time-major ``[L, N, D]`` activation as its transposed view, a slice of
a wider projection); outputs follow their input's memory order.  Gradients reach every floating argument, the state included, once
(as with the other recurrences).  ``inplace_state`` (calls without gradients): the new state is written over the given one (not over an expanded view).
Sums and states are fp32.  CUDA tensors only; there is no CPU implementation.
"""
from __future__ import annotations

import torch

from . import _lib as L


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, state=None, done=None, delta_softplus=True,
                   inplace_state=False):
    r = L.host().selective_scan(u, delta, A, B, C, D, z, delta_bias, state, done, delta_softplus, inplace_state)
    if r is not NotImplemented:
        return r
    return _scan(u, delta, A, B, C, D, z, delta_bias, state, done, delta_softplus, inplace_state)


def causal_conv(x, weight, bias=None, state=None, done=None, silu=True, inplace_state=False):
    r = L.host().causal_conv(x, weight, bias, state, done, silu, inplace_state)
    if r is not NotImplemented:
        return r
    return _conv(x, weight, bias, state, done, silu, inplace_state)


# ---------------------------------------------------------------------------------------
# what the native path has declined: errors are raised, anything else is brought into a form that it takes
# ---------------------------------------------------------------------------------------

def _tensor(name, t):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    return t if type(t) in (torch.Tensor, torch.nn.Parameter) else t.as_subclass(torch.Tensor)


def _like(name, t, shape, dtype, device):
    t = _tensor(name, t)
    if t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, expected {device}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t


def _activation(name, t, dims=3):
    t = _tensor(name, t)
    if t.device.type != "cuda":
        raise RuntimeError("srwm_b200 operators run on CUDA tensors only (no CPU implementation); "
                           f"got {name} on {t.device}")
    if t.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"{name} must be float32 or bfloat16, got {t.dtype}")
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got {tuple(t.shape)}")
    return t


def _rows(t):
    return t if t is None or t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def _dense(t):
    if t is None:
        return None
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _flags(done, N, Ln, device):
    if done is None:
        return None
    done = _tensor("done", done)
    if tuple(done.shape) != (N, Ln):
        raise ValueError(f"done must be [N, L] = {(N, Ln)}, got {tuple(done.shape)}")
    if done.device != device:
        raise RuntimeError(f"done is on {done.device}, expected {device}")
    return done if done.dtype in (torch.bool, torch.uint8) else done != 0


def _inplace(state, tensors):
    if state is None:
        raise ValueError("inplace_state needs a state")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError("inplace_state is for calls without gradients")


def _apart(rows):
    """Whether no two of the rows [N, L, D] share a value."""
    (far, n), (near, l) = sorted(((rows.stride(i), rows.shape[i]) for i in (0, 1)), reverse=True)
    width = rows.shape[2]
    return (l == 1 or near >= width) and (n == 1 or far >= (0 if l == 1 else near * (l - 1)) + width)


def _empty(out, *tensors):
    """An output without values: all of ``tensors`` have a gradient through it, zeros."""
    for t in tensors:
        if torch.is_grad_enabled() and t is not None and t.requires_grad:
            out = out + 0 * t.sum().to(out.dtype)
    return out


def _declined(what):
    raise RuntimeError(f"{what}: these tensors cannot be used (forward-mode AD, or a size beyond 2^31)")


def _scan(u, delta, A, B, C, D, z, delta_bias, state, done, delta_softplus, inplace_state):
    u = _activation("u", u)
    dev, dt = u.device, u.dtype
    N, Ln, Dn = u.shape
    delta = _like("delta", delta, u.shape, dt, dev)
    A = _tensor("A", A)
    if A.dim() != 2 or A.shape[1] not in (8, 16, 32, 64):
        raise ValueError(f"A must be [D, S] with 8, 16, 32 or 64 states, got {tuple(A.shape)}")
    S = A.shape[1]
    A = _like("A", A, (Dn, S), torch.float32, dev)
    B = _tensor("B", B)
    shape = (N, Ln, S)
    if B.dim() == 4:
        if B.shape[2] == 0 or Dn % B.shape[2]:
            raise ValueError(f"{B.shape[2]} groups of B and C do not divide {Dn} channels")
        shape = (N, Ln, B.shape[2], S)
    B, C = _like("B", B, shape, dt, dev), _like("C", C, shape, dt, dev)
    z = None if z is None else _like("z", z, u.shape, dt, dev)
    D = None if D is None else _like("D", D, (Dn,), torch.float32, dev)
    delta_bias = None if delta_bias is None else _like("delta_bias", delta_bias, (Dn,), torch.float32, dev)
    state = None if state is None else _like("state", state, (N, Dn, S), torch.float32, dev)
    done = _flags(done, N, Ln, dev)
    if inplace_state:
        _inplace(state, (u, delta, A, B, C, D, z, delta_bias, state))
        if not state.is_contiguous() or state.data_ptr() % 16:
            raise ValueError("inplace_state needs a dense state on a 16-byte boundary")
    if u.numel() == 0:      # nothing to run: the state is carried through unchanged
        y = _empty(torch.empty_like(u.detach()), u, delta, A, B, C, D, z, delta_bias, state)
        if state is None:
            return y, torch.zeros(N, Dn, S, device=dev)
        return y, state if inplace_state else state.clone()
    r = L.host().selective_scan(_rows(u), _rows(delta), _dense(A), _rows(B), _rows(C), _dense(D), _rows(z), _dense(delta_bias),
                                state if inplace_state else _dense(state), done, delta_softplus, inplace_state)
    return _declined("selective_scan") if r is NotImplemented else r


def _conv(x, weight, bias, state, done, silu, inplace_state):
    x = _activation("x", x)
    dev, dt = x.device, x.dtype
    N, Ln, Dn = x.shape
    weight = _tensor("weight", weight)
    if weight.dim() != 2 or weight.shape[1] not in (2, 3, 4):
        raise ValueError(f"weight must be [D, K] with 2, 3 or 4 taps, got {tuple(weight.shape)}")
    K = weight.shape[1]
    weight = _like("weight", weight, (Dn, K), torch.float32, dev)
    bias = None if bias is None else _like("bias", bias, (Dn,), torch.float32, dev)
    state = None if state is None else _like("state", state, (N, K - 1, Dn), dt, dev)
    done = _flags(done, N, Ln, dev)
    if inplace_state:
        _inplace(state, (x, weight, bias, state))
        if _rows(state) is not state:
            raise ValueError("inplace_state needs a state whose rows are dense")
        if not _apart(state):
            raise ValueError("inplace_state needs a state whose rows do not overlap (an expanded view is not written to)")
    if x.numel() == 0:
        y = _empty(torch.empty_like(x.detach()), x, weight, bias, state)
        if state is None:
            return y, torch.zeros(N, K - 1, Dn, device=dev, dtype=dt)
        return y, state if inplace_state else state.clone()
    r = L.host().causal_conv(_rows(x), _dense(weight), _dense(bias), _rows(state), done, silu, inplace_state)
    return _declined("causal_conv") if r is NotImplemented else r
