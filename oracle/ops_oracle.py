"""Step-by-step float64 definitions of the selective scan, the causal convolution, the root-mean-square norm and clipping by
the gradients' norm; differentiable by autograd.  Test infrastructure; runs on any device."""
import torch


def scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, state=None, done=None, softplus=True):
    """-> y [N, L, D], state [N, D, S]"""
    N, L, Dn = u.shape
    S = A.shape[1]
    G = B.shape[2] if B.dim() == 4 else 1
    group = torch.arange(Dn, device=u.device) // (Dn // G)
    B, C = B.reshape(N, L, G, S), C.reshape(N, L, G, S)
    raw = delta if delta_bias is None else delta + delta_bias
    step = torch.nn.functional.softplus(raw, threshold=40) if softplus else raw
    h = u.new_zeros(N, Dn, S) if state is None else state
    ys = []
    for t in range(L):
        if done is not None:
            h = torch.where(done[:, t, None, None].bool(), torch.zeros_like(h), h)
        h = torch.exp(step[:, t, :, None] * A) * h + (step[:, t] * u[:, t])[..., None] * B[:, t][:, group]
        y = (h * C[:, t][:, group]).sum(-1)
        ys.append(y if D is None else y + D * u[:, t])
    y = torch.stack(ys, 1) if ys else torch.empty_like(u)
    return (y if z is None else y * z * torch.sigmoid(z)), h


def conv(x, w, bias=None, state=None, done=None, silu=True):
    """-> y [N, L, D], state [N, K - 1, D]"""
    N, L, D = x.shape
    K = w.shape[1]
    win = x.new_zeros(N, K - 1, D) if state is None else state
    ys = []
    for t in range(L):
        if done is not None:
            win = torch.where(done[:, t, None, None].bool(), torch.zeros_like(win), win)
        win = torch.cat([win, x[:, t:t + 1]], 1)
        y = (win * w.t()).sum(1)
        ys.append(y if bias is None else y + bias)
        win = win[:, 1:]
    y = torch.stack(ys, 1) if ys else torch.empty_like(x)
    return (y * torch.sigmoid(y) if silu else y), win


def rms(x, w, residual=None, eps=1e-6, dtype=None):
    """-> y, stream; dtype: the type that the stream is rounded to (its gradient passes through)"""
    s = x if residual is None else x + residual
    if residual is not None and dtype is not None:
        s = s + (s.detach().to(dtype).double() - s.detach())
    return s * torch.rsqrt((s * s).mean(-1, keepdim=True) + eps) * w, s


def clip(tensors, max_norm):
    """-> norm, scaled tensors (float64)"""
    ts = [t.double() for t in tensors]
    norm = sum((t * t).sum() for t in ts).sqrt()
    return norm, [t * torch.clamp(max_norm / (norm + 1e-6), max=1.0) for t in ts]
