"""The selective scan and the causal convolution against their step-by-step definitions in float64.

Tolerances.  With steps Delta >= 0.05 and decays A <= -0.5 a state remembers 1 / (1 - exp(-0.025)) = 40 steps; each adds at most 2^-22 of
the exponential and two roundings of 2^-24 to the state's relative error: 40 x 1.5 x 2^-22 = 1.5e-5 of the largest value, FWD.  A
gradient has the state's and its own carry's error and a product's, 3 FWD, and sums over at most 300 steps and 160 channels in
fp32, 460 x 2^-24 = 2.7e-5: GRAD = 7.5e-5.  A bfloat16 output is off by half a step more, 2^-8 of its value.
"""
import pytest
import torch

import ops_oracle as orc
import srwm_b200 as sb

pytestmark = pytest.mark.gpu
FWD, GRAD = 1.5e-5, 7.5e-5
NAMES = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state")


def _near(got, want, tol, what=""):
    want = want.to(got.device)
    err = (got.double() - want).abs()
    bound = tol * float(want.abs().max()) + (2.0 ** -8 * want.abs() if got.dtype == torch.bfloat16 else 0.0) + 1e-30
    assert bool((err <= bound).all()), (what, float((err / bound).max()))


def _inputs(N, L, D, S, G, dtype, seed=0, done=False, gate=True, state=True, time_major=False):
    g = torch.Generator(device="cuda").manual_seed(seed + N + 7 * L + 13 * D + S)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731

    def rows(t):      # time-major rows as their transposed view
        return t.transpose(0, 1).contiguous().transpose(0, 1) if time_major else t
    bc = (N, L, S) if G == 1 else (N, L, G, S)
    x = {"u": rows(r(N, L, D)).to(dtype), "delta": rows(r(N, L, D) * 0.5).to(dtype), "A": -(0.5 + 2 * torch.rand(D, S, device="cuda", generator=g)),
         "B": rows(r(*bc)).to(dtype), "C": rows(r(*bc)).to(dtype), "D": r(D), "z": rows(r(N, L, D)).to(dtype) if gate else None,
         "delta_bias": -0.5 + 0.5 * torch.rand(D, device="cuda", generator=g), "state": r(N, D, S) if state else None}
    x["delta"].clamp_(min=-2.0)       # softplus(-2 - 0.5) = 0.079
    flags = torch.rand(N, L, device="cuda", generator=g) < (3.0 / max(L, 1)) if done else None
    return x, flags, r(N, L, D).to(dtype), r(N, D, S)


def _scan_case(N, L, D, S, G=1, dtype=torch.float32, softplus=True, **kw):
    x, done, gy, gs = _inputs(N, L, D, S, G, dtype, **kw)
    if not softplus:
        x["delta"] = torch.nn.functional.softplus(x["delta"].float()).to(dtype)
        x["delta_bias"] = None
    names = [k for k in NAMES if x[k] is not None]
    ref = {k: (v.detach().double().requires_grad_() if v is not None else None) for k, v in x.items()}
    yr, hr = orc.scan(**ref, done=done, softplus=softplus)
    gr = torch.autograd.grad([yr, hr], [ref[k] for k in names], [gy.double(), gs.double()])
    args = {k: (v.detach().requires_grad_() if v is not None else None) for k, v in x.items()}
    y, h = sb.selective_scan(**args, done=done, delta_softplus=softplus)
    assert y.dtype == dtype and h.dtype == torch.float32 and y.stride() == x["u"].stride()
    _near(y.detach(), yr.detach(), FWD, "y")
    _near(h.detach(), hr.detach(), FWD, "state")
    got = torch.autograd.grad([y, h], [args[k] for k in names], [gy, gs])
    for k, a, b in zip(names, got, gr):
        assert a.dtype == x[k].dtype and a.shape == x[k].shape
        _near(a, b, GRAD, k)
    with torch.no_grad():
        y2, h2 = sb.selective_scan(**x, done=done, delta_softplus=softplus)
        _near(y2, yr.detach(), FWD, "y without gradients")
        _near(h2, hr.detach(), FWD, "state without gradients")
        if x["state"] is not None:
            st = x["state"].clone()
            y3, h3 = sb.selective_scan(**{**x, "state": st}, done=done, delta_softplus=softplus, inplace_state=True)
            assert h3 is st or h3.data_ptr() == st.data_ptr()
            assert torch.equal(y3, y2) and torch.equal(st, h2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S", [8, 16, 32, 64])
@pytest.mark.parametrize("N,L,D", [(1, 1, 1), (2, 4, 33), (3, 5, 32), (2, 16, 64), (1, 17, 31), (2, 33, 100)])
def test_scan_sizes(N, L, D, S, dtype):
    _scan_case(N, L, D, S, dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,L,D,S,G", [(2, 70, 96, 16, 2), (1, 300, 160, 16, 1), (3, 45, 66, 8, 3), (2, 130, 40, 64, 2), (1, 257, 36, 32, 1)])
def test_scan_resets_groups_and_pieces_of_time(N, L, D, S, G, dtype):
    _scan_case(N, L, D, S, G, dtype, done=True)
    _scan_case(N, L, D, S, G, dtype, seed=3, gate=False, state=False)
    _scan_case(N, L, D, S, G, dtype, seed=4, done=True, time_major=True, softplus=False)


@pytest.mark.parametrize("N,L,D,S,G,dtype", [(40, 35, 250, 16, 1, torch.float32), (40, 35, 256, 16, 2, torch.bfloat16), (40, 21, 256, 32, 1, torch.float32),
                                             (40, 37, 250, 32, 2, torch.bfloat16), (38, 20, 256, 64, 1, torch.float32), (40, 19, 250, 64, 2, torch.bfloat16),
                                             (40, 35, 300, 8, 1, torch.float32), (2, 1200, 512, 16, 1, torch.float32), (37, 300, 64, 64, 1, torch.float32),
                                             (2, 1100, 576, 32, 1, torch.bfloat16)])
def test_scan_grids_that_fill_the_gpu(N, L, D, S, G, dtype):
    """Two channels a thread; the last three cut into pieces of the time axis as well (no sum has more than 300 terms in a row then either:
    a piece's steps, the pieces and sequences, the channels of a block, the blocks)."""
    _scan_case(N, L, D, S, G, dtype, done=True)
    _scan_case(N, L, D, S, G, dtype, seed=2, gate=False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S", [8, 16, 32, 64])
@pytest.mark.parametrize("N,L,D,G", [(303, 1, 1000, 1), (301, 3, 1028, 2)])
def test_tokens_of_many_sequences(N, L, D, G, S, dtype):
    """Four sequences a thread, the last group not whole."""
    x, done, _, _ = _inputs(N, L, D, S, G, dtype, seed=21, done=True)
    with torch.no_grad():
        yr, hr = orc.scan(**{k: v.double() for k, v in x.items()}, done=done)
        st = x["state"].clone()
        y, h = sb.selective_scan(**{**x, "state": st}, done=done, inplace_state=True)
        _near(y, yr, FWD, "y")
        _near(st, hr, FWD, "state")
        y, h = sb.selective_scan(**{**x, "z": None, "state": None, "D": None, "delta_bias": None})
        yr, hr = orc.scan(**{k: (v.double() if v is not None else None) for k, v in {**x, "z": None, "state": None, "D": None, "delta_bias": None}.items()})
        _near(y, yr, FWD, "y")
        _near(h, hr, FWD, "state")


def test_scan_reset_at_every_step_and_at_the_first():
    for fill in (lambda d: d.fill_(True), lambda d: d.index_fill_(1, torch.tensor([0], device="cuda"), True),
                 lambda d: d[:, -1].fill_(True)):
        x, _, gy, gs = _inputs(2, 150, 40, 16, 1, torch.float32, seed=9)
        done = torch.zeros(2, 150, dtype=torch.uint8, device="cuda")
        fill(done)
        names = [k for k in NAMES]
        ref = {k: v.detach().double().requires_grad_() for k, v in x.items()}
        yr, hr = orc.scan(**ref, done=done)
        gr = torch.autograd.grad([yr, hr], [ref[k] for k in names], [gy.double(), gs.double()], allow_unused=True)
        args = {k: v.detach().requires_grad_() for k, v in x.items()}
        y, h = sb.selective_scan(**args, done=done)
        _near(y.detach(), yr.detach(), FWD)
        for k, a, b in zip(names, torch.autograd.grad([y, h], [args[k] for k in names], [gy, gs]), gr):
            _near(a, torch.zeros_like(a, dtype=torch.float64) if b is None else b, GRAD, k)


def test_scan_state_across_calls_is_one_call():
    """A sequence in three parts with the state carried, gradients through it, is the whole sequence."""
    x, _, gy, gs = _inputs(2, 90, 48, 16, 1, torch.float32, seed=5)
    whole = {k: v.detach().requires_grad_() for k, v in x.items()}
    y, h = sb.selective_scan(**whole)
    want = torch.autograd.grad([y, h], list(whole.values()), [gy, gs])
    parts = {k: v.detach().requires_grad_() for k, v in x.items()}
    st, ys = parts["state"], []
    for a, b in ((0, 3), (3, 52), (52, 90)):
        sl = {k: (v[:, a:b] if k in ("u", "delta", "B", "C", "z") else v) for k, v in parts.items()}
        yp, st = sb.selective_scan(**{**sl, "state": st})
        ys.append(yp)
    got = torch.autograd.grad([torch.cat(ys, 1), st], list(parts.values()), [gy, gs])
    _near(torch.cat(ys, 1).detach(), y.detach().double(), 2 * FWD)
    for a, b in zip(got, want):
        _near(a, b.double(), 2 * GRAD)


def test_scan_views_broadcasts_and_unaligned_rows():
    """Slices of wider rows at odd offsets, B shared by all sequences, a state that is a transposed view."""
    N, L, D, S = 2, 37, 52, 16
    x, _, gy, gs = _inputs(N, L, D, S, 1, torch.bfloat16, seed=6)
    wide = torch.randn(N, L, 2 * D + 2 * S + 3, device="cuda").to(torch.bfloat16)
    x["u"], x["z"] = wide[..., 1:1 + D], wide[..., 1 + D:1 + 2 * D]
    x["C"] = wide[..., 2 * D + 3:2 * D + 3 + S]
    x["B"] = x["B"][:1].expand(N, L, S)
    x["state"] = x["state"].transpose(1, 2).contiguous().transpose(1, 2)
    x["A"] = x["A"].t().contiguous().t()
    ref = {k: v.detach().double().requires_grad_() for k, v in x.items()}
    yr, hr = orc.scan(**ref)
    gr = torch.autograd.grad([yr, hr], list(ref.values()), [gy.double(), gs.double()])
    args = {k: v.detach().requires_grad_() for k, v in x.items()}
    y, h = sb.selective_scan(**args)
    _near(y.detach(), yr.detach(), FWD)
    for k, a, b in zip(args, torch.autograd.grad([y, h], list(args.values()), [gy, gs]), gr):
        _near(a, b, GRAD, k)
    base = torch.randn(L, S, device="cuda").to(torch.bfloat16).requires_grad_()      # one leaf for all sequences: its gradient is their sum
    y, h = sb.selective_scan(**{**x, "B": base.expand(N, L, S)})
    got = torch.autograd.grad(y, base, gy)[0]
    b64 = base.detach().double().requires_grad_()
    r64 = {k: v.detach().double() for k, v in x.items()}
    want = torch.autograd.grad(orc.scan(**{**r64, "B": b64.expand(N, L, S)})[0], b64, gy.double())[0]
    assert float((got.double() - want).abs().max()) <= 3 * 2.0 ** -8 * float(want.abs().max())      # (N rounded gradients and their rounded sum)


def test_scan_one_gradient_at_a_time():
    x, _, gy, gs = _inputs(2, 20, 32, 16, 1, torch.float32, seed=7)
    for k in NAMES:
        ref = {n: (v.double().requires_grad_() if n == k else v.double()) for n, v in x.items()}
        args = {n: (v.detach().requires_grad_() if n == k else v) for n, v in x.items()}
        for out in (0, 1):
            if out == 1 and k in ("C", "D", "z"):
                continue
            go = gs if out else gy
            want = torch.autograd.grad(orc.scan(**ref)[out], ref[k], go.double())[0]
            _near(torch.autograd.grad(sb.selective_scan(**args)[out], args[k], go)[0], want, GRAD, k)


def test_scan_gradient_is_the_function_s_difference():
    x, _, gy, _ = _inputs(1, 24, 32, 16, 1, torch.float32, seed=8)
    args = {k: v.detach().requires_grad_() for k, v in x.items()}
    grads = torch.autograd.grad(sb.selective_scan(**args)[0], list(args.values()), gy)
    for k, g in zip(args, grads):
        d = torch.randn_like(x[k])
        eps = 1e-2 * float(x[k].abs().mean()) / float(d.abs().mean())
        f = lambda s: (orc.scan(**{**{n: v.double() for n, v in x.items()}, k: x[k].double() + s * eps * d.double()})[0] * gy.double()).sum()  # noqa: E731
        want = (8 * (f(1) - f(-1)) - (f(2) - f(-2))) / (12 * eps)       # fourth order: off by eps^4
        scale = float((g.double() * d.double()).abs().sum())
        assert abs(float((g.double() * d.double()).sum() - want)) < 1e-4 * scale, k


def test_scan_masked_and_infinite_values_stay_where_they_belong():
    """NaN and infinities in front of a reset, in another sequence or another channel, do not reach past it."""
    x, _, _, _ = _inputs(2, 64, 64, 16, 1, torch.float32, seed=10)
    done = torch.zeros(2, 64, dtype=torch.bool, device="cuda")
    done[0, 20] = True
    clean = sb.selective_scan(**x, done=done)[0]
    bad = {k: (v.clone() if v is not None else None) for k, v in x.items()}
    bad["u"][0, 7, :] = float("nan")
    bad["u"][0, 9, 5] = float("inf")
    bad["state"][0, 3] = float("inf")
    y, h = sb.selective_scan(**bad, done=done)
    assert torch.equal(y[0, 20:], clean[0, 20:]) and torch.equal(y[1], clean[1])
    assert bool(y[0, 7:20].isnan().all()) and bool(torch.isfinite(h).all())
    bad["u"] = x["u"].clone()
    bad["state"] = x["state"].clone()
    bad["delta"][:, 11, 40] = float("-inf")      # a step of zero: the state stays
    y, h = sb.selective_scan(**{**bad, "delta_bias": None}, done=done)
    assert bool(torch.isfinite(y).all())
    keep = [c for c in range(64) if c != 40]
    assert torch.equal(y[:, :, keep], sb.selective_scan(**{**x, "delta_bias": None}, done=done)[0][:, :, keep])


@pytest.mark.parametrize("D", [1, 33])
def test_scan_infinite_b_and_c(D):
    """An infinite B or C reaches the gradients that it has a part in, and the channels that a block has room for beyond D none."""
    for name in ("B", "C"):
        x, _, gy, gs = _inputs(1, 20, D, 16, 1, torch.float32, seed=12)
        x[name][0, 13, 5] = float("inf")
        ref = {k: v.detach().double().requires_grad_() for k, v in x.items()}
        want = torch.autograd.grad(list(orc.scan(**ref)), [ref["B"], ref["C"]], [gy.double(), gs.double()])
        args = {k: v.detach().requires_grad_() for k, v in x.items()}
        got = torch.autograd.grad(list(sb.selective_scan(**args)), [args["B"], args["C"]], [gy, gs])
        for a, b in zip(got, want):
            assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.isposinf(), b.isposinf()) and torch.equal(a.isneginf(), b.isneginf())
            fine = torch.isfinite(b)
            _near(torch.where(fine, a, torch.zeros_like(a)), torch.where(fine, b, torch.zeros_like(b)), GRAD, name)


def test_rows_beyond_32_bit_offsets():
    """Sequences more than 2^31 elements apart, and a tensor of more than 2^31 values."""
    far = (1 << 31) + 64
    buf = torch.zeros(far + 40 * 96, device="cuda", dtype=torch.bfloat16)
    view = lambda w, at=0: buf.as_strided((2, 40, w), (far, 96, 1), at)  # noqa: E731
    x, _, gy, _ = _inputs(2, 40, 32, 16, 1, torch.bfloat16, seed=13)
    for k, at in (("u", 0), ("z", 32), ("C", 64)):
        view(x[k].shape[-1], at).copy_(x[k])
    near, far_ = [{k: v.detach().clone().requires_grad_() for k, v in x.items()} for _ in range(2)]
    for k, at in (("u", 0), ("z", 32), ("C", 64)):
        far_[k] = view(x[k].shape[-1], at).detach().requires_grad_()
    a, b = sb.selective_scan(**near), sb.selective_scan(**far_)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for g, h in zip(torch.autograd.grad(a[0], list(near.values()), gy), torch.autograd.grad(b[0], list(far_.values()), gy)):
        assert torch.equal(g, h)
    w = torch.randn(32, 4, device="cuda")
    near_u = x["u"].clone().requires_grad_()
    c, d = sb.causal_conv(near_u, w), sb.causal_conv(far_["u"], w)
    assert torch.equal(c[0], d[0]) and torch.equal(torch.autograd.grad(c[0].sum(), near_u)[0], torch.autograd.grad(d[0].sum(), far_["u"])[0])
    n = torch.ones(32, device="cuda")
    assert torch.equal(sb.rms_norm(x["u"][:, 3], n), sb.rms_norm(view(32)[:, 3], n))
    want = float(buf[:4096].double().square().sum() + buf[-4096:].double().square().sum()) ** 0.5      # (zeros between)
    assert abs(float(sb.grad_norm([buf])) / want - 1) < 1e-6
    sb.grad_ops.clip_tensors_([buf], want / 2)
    assert abs(float(sb.grad_norm([buf])) / (want / 2) - 1) < 2e-3


def test_scan_small_steps_keep_their_precision():
    """Steps of 1e-3 and slow decays: 1000 steps of memory; the state's relative error is a random walk of half-steps of the decay,
    2^-24 sqrt(1000) = 2e-6, and at most the sum of the exponentials' bias: 1e-5 asked."""
    N, L, D, S = 2, 2048, 64, 16
    x, _, _, _ = _inputs(N, L, D, S, 1, torch.float32, seed=11)
    x["delta"] = x["delta"] * 0.3
    x["delta_bias"] = torch.full((D,), -6.9, device="cuda")
    x["A"] = -torch.arange(1, S + 1, device="cuda").float().expand(D, S).contiguous()
    with torch.no_grad():
        yr, hr = orc.scan(**{k: v.double() for k, v in x.items()})
        y, h = sb.selective_scan(**x)
    assert float((y.double() - yr).norm() / yr.norm()) < 1e-5 and float((h.double() - hr).norm() / hr.norm()) < 1e-5


def test_scan_empty_and_refused():
    x, done, _, _ = _inputs(2, 6, 32, 16, 1, torch.float32, done=True)
    for k in ("u", "delta", "B", "C", "z"):
        x[k] = x[k][:, :0]
    y, h = sb.selective_scan(**x)
    assert y.shape == (2, 0, 32) and torch.equal(h, x["state"])
    assert not bool(sb.selective_scan(**{**x, "state": None})[1].any())
    x, done, _, _ = _inputs(2, 6, 32, 16, 1, torch.float32, done=True)
    bad = [({"A": x["A"][:, :12]}, ValueError), ({"A": x["A"].double()}, TypeError), ({"delta": x["delta"][:, :5]}, ValueError),
           ({"B": x["B"].to(torch.bfloat16)}, TypeError), ({"C": x["C"][:, :, :8]}, ValueError), ({"u": x["u"].half()}, TypeError),
           ({"done": done[:, :4]}, ValueError), ({"state": x["state"].cpu()}, RuntimeError), ({"D": x["D"][:3]}, ValueError),
           ({"B": x["B"].unsqueeze(2).expand(-1, -1, 5, -1)}, ValueError), ({"state": None, "inplace_state": True}, ValueError),
           ({"state": x["state"].transpose(1, 2).contiguous().transpose(1, 2), "inplace_state": True}, ValueError),
           ({"u": x["u"].clone().requires_grad_(), "inplace_state": True}, ValueError)]
    for change, error in bad:
        with pytest.raises(error):
            sb.selective_scan(**{**x, **change})
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError):
        sb.selective_scan(**{**x, "u": torch.autograd.forward_ad.make_dual(x["u"], torch.ones_like(x["u"]))})


# ---- causal convolution ----

def _conv_case(N, L, D, K, dtype, done=False, bias=True, state=True, silu=True, view=None):
    g = torch.Generator(device="cuda").manual_seed(N + 3 * L + 5 * D + K)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x = r(N, L, D).to(dtype)
    if view == "time":
        x = x.transpose(0, 1).contiguous().transpose(0, 1)
    if view == "slice":
        x = r(N, L, 2 * D + 1).to(dtype)[..., 1:1 + D]
    w, b = r(D, K) * K ** -0.5, r(D) if bias else None
    st = r(N, K - 1, D).to(dtype) if state else None
    flags = torch.rand(N, L, device="cuda", generator=g) < 0.2 if done else None
    gy, gs = r(N, L, D).to(dtype), r(N, K - 1, D).to(dtype)
    leaves = [t for t in (x, w, b, st) if t is not None]
    ref = [t.detach().double().requires_grad_() if t is not None else None for t in (x, w, b, st)]
    yr, sr = orc.conv(*ref, done=flags, silu=silu)
    gr = torch.autograd.grad([yr, sr], [t for t in ref if t is not None], [gy.double(), gs.double()])
    args = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b, st)]
    y, s = sb.causal_conv(*args, done=flags, silu=silu)
    # a few products and a sigmoid of 2^-22: 3e-6; sums over N L values in fp32, at most 600 x 2^-24 = 3.6e-5
    _near(y.detach(), yr.detach(), 3e-6, "y")
    assert s.dtype == dtype and torch.equal(s.double(), sr)
    assert y.stride() == x.stride() or view == "slice"
    for k, a, b_ in zip(leaves, torch.autograd.grad([y, s], [t for t in args if t is not None], [gy, gs]), gr):
        assert a.dtype == k.dtype
        _near(a, b_, 4e-5)
    with torch.no_grad():
        y2, s2 = sb.causal_conv(x, w, b, st, flags, silu)
        assert torch.equal(y2, y) and torch.equal(s2, s)
        if state:
            st2 = st.clone()
            y3, s3 = sb.causal_conv(x, w, b, st2, flags, silu, inplace_state=True)
            assert s3.data_ptr() == st2.data_ptr() and torch.equal(y3, y) and torch.equal(st2, s)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [2, 3, 4])
@pytest.mark.parametrize("N,L,D", [(1, 1, 1), (2, 1, 64), (3, 2, 37), (2, 3, 128), (1, 15, 5), (2, 16, 130), (2, 17, 64), (3, 100, 36), (1, 200, 512)])
def test_conv_sizes(N, L, D, K, dtype):
    _conv_case(N, L, D, K, dtype)


@pytest.mark.parametrize("K", [2, 4])
@pytest.mark.parametrize("L", [1, 2, 3, 17, 50])
def test_conv_resets_views_and_options(L, K):
    _conv_case(3, L, 40, K, torch.float32, done=True)
    _conv_case(3, L, 40, K, torch.bfloat16, done=True, view="time", state=False)
    _conv_case(2, L, 33, K, torch.float32, view="slice", bias=False)
    _conv_case(2, L, 36, K, torch.bfloat16, silu=False, done=True)


def test_conv_refused_and_empty():
    x, w = torch.randn(2, 5, 8, device="cuda"), torch.randn(8, 4, device="cuda")
    for args, error in (((x, w[:, :1]), ValueError), ((x, w[:7]), ValueError), ((x, w.double()), TypeError), ((x.half(), w), TypeError),
                        ((x, w.cpu()), RuntimeError), ((x[0], w), ValueError), ((x, w, w), ValueError), ((x, w, None, x), ValueError)):
        with pytest.raises(error):
            sb.causal_conv(*args)
    with pytest.raises(ValueError):
        sb.causal_conv(x, w, inplace_state=True)
    st = torch.randn(2, 3, 8, device="cuda")
    y, s = sb.causal_conv(x[:, :0], w, state=st)
    assert y.shape == (2, 0, 8) and torch.equal(s, st)


def test_conv_state_in_place_is_not_an_expanded_view():
    x, w = torch.randn(4, 3, 64, device="cuda"), torch.randn(64, 4, device="cuda")
    with torch.no_grad():
        for state in (torch.zeros(1, 3, 64, device="cuda").expand(4, -1, -1), torch.zeros(4, 1, 64, device="cuda").expand(-1, 3, -1),
                      torch.zeros(4 * 64 + 128, device="cuda").as_strided((4, 3, 64), (64, 64, 1))):
            with pytest.raises(ValueError):
                sb.causal_conv(x, w, None, state, inplace_state=True)
            assert not state.any()
        # rows of a wider buffer, time-major and not, are written, and nothing between them
        for buf, view in ((torch.randn(4, 5, 96, device="cuda"), lambda b: b[:, 1:4, 16:80]), (torch.randn(3, 6, 64, device="cuda"), lambda b: b[:, 1:5].transpose(0, 1))):
            y, st = sb.causal_conv(x, w, None, view(buf).clone())
            got = buf.clone()
            y2, _ = sb.causal_conv(x, w, None, view(got), inplace_state=True)
            view(buf).copy_(st)
            assert torch.equal(y, y2) and torch.equal(got, buf)


@pytest.mark.parametrize("S", [8, 16, 32, 64])
@pytest.mark.parametrize("L,D", [(1, 96), (37, 96), (2000, 36)])
def test_steps_of_no_length_leave_the_state(S, L, D):
    """Delta of zero (a padded step) keeps every bit of the state and of its gradient, in one piece of the time axis or several."""
    g = torch.Generator(device="cuda").manual_seed(S + L)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)      # noqa: E731
    u, B, C, A = rand(2, L, D), rand(2, L, S), rand(2, L, S), -torch.rand(D, S, device="cuda", generator=g) * S
    state, go = rand(2, D, S).requires_grad_(), rand(2, D, S)
    with torch.no_grad():
        assert torch.equal(sb.selective_scan(u, torch.zeros_like(u), A, B, C, state=state, delta_softplus=False)[1], state)
    _, last = sb.selective_scan(u, torch.zeros_like(u), A, B, C, state=state, delta_softplus=False)
    assert torch.equal(last, state)
    assert torch.equal(torch.autograd.grad(last, state, go)[0], go)


# ---- values that are not finite, and a time axis that is cut into pieces ----

def _pieces(L, D, S):
    """The case's time axis is cut into three pieces at least: the forward's scratch is (2 pieces - 1) states."""
    from srwm_b200 import _lib
    return (_lib.load().srwm_b200_scan_scratch_bytes(2, L, D, S, 1) // (4 * 2 * D * S) + 1) // 2


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("S", [8, 16, 32, 64])
@pytest.mark.parametrize("L,D,at,reset", [(1000, 64, 300, 700), (512, 33, 10, 500)])
def test_scan_bad_values_do_not_pass_a_reset_in_another_piece(L, D, at, reset, S, bad):
    """NaN and infinities of an episode, pieces in front of the next one's start, leave every bit of what follows."""
    assert _pieces(L, D, S) >= 3
    x, _, _, _ = _inputs(2, L, D, S, 1, torch.float32, seed=30)
    done = torch.zeros(2, L, dtype=torch.bool, device="cuda")
    done[0, reset] = True
    spoilt = {**x, "u": x["u"].clone()}
    spoilt["u"][0, at] = bad
    first = done.clone()
    first[0, 0] = True
    recycled = {**x, "state": x["state"].clone()}
    recycled["state"][0] = bad
    for grad in (False, True):      # (the second keeps states for a backward)
        with torch.set_grad_enabled(grad):
            clean = sb.selective_scan(**{**x, "A": x["A"].detach().requires_grad_(grad)}, done=done)
            y, h = sb.selective_scan(**{**spoilt, "A": x["A"].detach().requires_grad_(grad)}, done=done)
            assert torch.equal(y[0, :at], clean[0][0, :at]) and not bool(torch.isfinite(y[0, at]).any())
            assert torch.equal(y[0, reset:], clean[0][0, reset:]) and torch.equal(y[1], clean[0][1]) and torch.equal(h, clean[1])
            clean = sb.selective_scan(**{**x, "A": x["A"].detach().requires_grad_(grad)}, done=first)
            y, h = sb.selective_scan(**{**recycled, "A": x["A"].detach().requires_grad_(grad)}, done=first)
            assert torch.equal(y, clean[0]) and torch.equal(h, clean[1])


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("S", [8, 16, 32, 64])
@pytest.mark.parametrize("L,D,at,reset", [(1000, 64, 900, 400), (512, 33, 500, 100)])
def test_scan_bad_gradients_do_not_pass_a_reset_in_another_piece(L, D, at, reset, S, bad):
    """A gradient of an output or of the last state that is NaN or infinite, and inputs that are, leave every bit of the rows' gradients
    in the episodes in front (behind)."""
    assert _pieces(L, D, S) >= 3
    x, _, gy, gs = _inputs(2, L, D, S, 1, torch.float32, seed=31)
    done = torch.zeros(2, L, dtype=torch.bool, device="cuda")
    done[0, reset] = True
    rows = ("u", "delta", "B", "C", "z")

    def grads(gy, gs, **change):
        args = {k: v.detach().requires_grad_() for k, v in {**x, **change}.items()}
        return dict(zip(NAMES, torch.autograd.grad(list(sb.selective_scan(**args, done=done)), [args[k] for k in NAMES], [gy, gs])))
    clean = grads(gy, gs)
    assert all(bool(torch.isfinite(v).all()) for v in clean.values())
    gy_bad, gs_bad, u_bad = gy.clone(), gs.clone(), x["u"].clone()
    gy_bad[0, at] = bad
    gs_bad[0] = bad
    for got in (grads(gy_bad, gs), grads(gy, gs_bad)):
        for k in rows:
            assert torch.equal(got[k][0, :reset], clean[k][0, :reset]) and torch.equal(got[k][1], clean[k][1]), k
        assert torch.equal(got["state"], clean["state"]) and not bool(torch.isfinite(got["B"][0, at]).any())
    u_bad[0, reset // 2] = bad
    got = grads(gy, gs, u=u_bad)
    for k in rows:
        assert torch.equal(got[k][0, reset:], clean[k][0, reset:]) and torch.equal(got[k][1], clean[k][1]), k
    assert torch.equal(got["state"], clean["state"])


@pytest.mark.parametrize("S", [8, 16, 32, 64])
def test_scan_growth_that_a_float_does_not_hold_over_a_piece(S):
    """Steps as given may be negative, and a state grow.  A state of zero stays zero however much a whole piece grows, and a small one comes
    to what its steps make of it, as long as these are finite; its gradient likewise.  Of the largest value: 140 steps of growth and
    decay, 1.5 x 2^-22 each, 5e-5, and three times that for gradients.  A piece's product has its steps' sum in fp32 as well, here up to
    98 in 70 additions, half-steps of 2^-18 for 24 of them, 2^-19 for 23, 2^-20 for 11 and less: 1.5e-4 in all."""
    N, L, D = 2, 1000, 64
    assert _pieces(L, D, S) == 13      # of 80 steps
    x, _, gy, gs = _inputs(N, L, D, S, 1, torch.float32, seed=32)
    x["delta_bias"] = None
    x["delta"] = torch.full((N, L, D), 1.4, device="cuda")
    x["A"] = torch.full((D, S), -1.0, device="cuda")

    def both(x, gy, gs):
        names = [k for k in NAMES if x[k] is not None]
        ref = {k: (v if v is None else v.detach().double().requires_grad_()) for k, v in x.items()}
        args = {k: (v if v is None else v.detach().requires_grad_()) for k, v in x.items()}
        want, got = orc.scan(**ref, softplus=False), sb.selective_scan(**args, delta_softplus=False)
        gw = torch.autograd.grad(list(want), [ref[k] for k in names], [gy.double(), gs.double()])
        gg = torch.autograd.grad(list(got), [args[k] for k in names], [gy, gs])
        return [(a.detach(), b.detach()) for a, b in zip(got, want)], {k: (a, b) for k, a, b in zip(names, gg, gw)}

    # nothing in front of step 400, and growth beyond every float: 2^323 in each of the pieces from 160 to 320
    empty = {**x, "state": None, "u": x["u"].clone(), "delta": x["delta"].clone()}
    empty["u"][:, :400] = 0.0
    empty["delta"][:, 160:320] = -2.8
    out, grads = both(empty, gy * (torch.arange(L, device="cuda") >= 400)[:, None], gs)
    for a, b in out:
        _near(a, b, 5e-5)
    for k in ("B", "C", "z"):      # (of u and delta, those of the steps in front of the growth are beyond a float themselves)
        _near(grads[k][0][:, 400:], grads[k][1][:, 400:], 1.5e-4, k)
    # a small state through 98 e-folds inside one piece, and as many back
    small = {**x, "state": 1e-30 * x["state"], "u": torch.zeros_like(x["u"]), "delta": x["delta"].clone()}
    small["delta"][:, :160] = 0.0
    small["delta"][:, 160:230] = -1.4
    small["delta"][:, 230:330] = 0.0
    out, _ = both(small, gy, gs)
    _near(*out[0], 2e-4)
    _near(out[0][0][:, 240:330], out[0][1][:, 240:330], 2e-4)
    assert 1e11 < float(out[0][1].abs().max()) < 1e16
    # a small gradient, the same way back
    last = {**x, "u": x["u"].clone(), "delta": x["delta"].clone()}
    last["u"][:, 500:] = 0.0
    last["delta"][:, 800:870] = -1.4
    last["delta"][:, 870:] = 0.0
    last["delta"][:, 700:800] = 1e-3
    out, grads = both(last, gy * (torch.arange(L, device="cuda") < 500)[:, None], 1e-30 * gs)
    for a, b in out:
        _near(a, b, 5e-5)
    for k in ("u", "state"):
        _near(*grads[k], 3e-4, k)
    _near(grads["u"][0][:, 700:800], grads["u"][1][:, 700:800], 3e-4, "in front of the growth")
    assert 1e11 < float(grads["u"][1][:, 500:].abs().max()) < 1e16


def test_conv_of_more_than_2_31_weights_and_biases():
    """The sums of dw and dbias, D (K + 1) values, beyond 32 bits: one step of one sequence, every value a product."""
    D, K = 860_000_004, 4
    if torch.cuda.get_device_properties(0).total_memory < 100e9:
        pytest.skip("100 GB of memory")
    torch.cuda.empty_cache()
    x, w = torch.empty(1, 1, D, device="cuda", dtype=torch.bfloat16).normal_().requires_grad_(), torch.full((D, K), 0.5, device="cuda").requires_grad_()
    bias, gy = torch.zeros(D, device="cuda").requires_grad_(), torch.empty(1, 1, D, device="cuda", dtype=torch.bfloat16).normal_()
    y, _ = sb.causal_conv(x, w, bias, silu=False)
    dx, dw, db = torch.autograd.grad(y, [x, w, bias], gy)
    for a in (0, D // 2, D - 1000):
        at = slice(a, a + 1000)
        g, v = gy[0, 0, at].float(), x[0, 0, at].detach().float()
        assert torch.equal(y[0, 0, at].detach(), (0.5 * v).bfloat16()) and torch.equal(dx[0, 0, at], (0.5 * g).bfloat16())
        assert torch.equal(db[at], g) and torch.equal(dw[at, K - 1], g * v) and not bool(dw[at, :K - 1].any())
    del x, w, bias, gy, y, dx, dw, db
    torch.cuda.empty_cache()


def test_scan_refuses_b_and_c_of_other_dimensions():
    x, _, _, _ = _inputs(2, 6, 32, 16, 1, torch.float32)
    for k in ("B", "C"):
        for t in (torch.ones((), device="cuda"), torch.ones(16, device="cuda"), torch.ones(2, 6, 1, 1, 16, device="cuda"), torch.ones(2, 6, device="cuda")):
            with pytest.raises(ValueError):
                sb.selective_scan(**{**x, k: t})


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("K", [2, 3, 4])
@pytest.mark.parametrize("L,reset", [(9, 4), (100, 16), (100, 33), (300, 150)])
def test_conv_bad_values_do_not_pass_a_reset(L, reset, K, bad):
    """Inputs, states and gradients of one episode that are NaN or infinite leave every bit of the other's, at the edges of the chunks of
    the time axis too."""
    g = torch.Generator(device="cuda").manual_seed(L + K)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x, w, b, st, gy, gs = r(2, L, 40), r(40, K), r(40), r(2, K - 1, 40), r(2, L, 40), r(2, K - 1, 40)
    done = torch.zeros(2, L, dtype=torch.bool, device="cuda")
    done[0, reset] = True

    def both(x, st, gy):
        args = [t.detach().requires_grad_() for t in (x, st)]
        y, s = sb.causal_conv(args[0], w, b, args[1], done)
        return [y.detach(), s.detach(), *torch.autograd.grad([y, s], args, [gy, gs])]
    y, s, dx, ds = both(x, st, gy)
    for at in range(max(0, reset - K), reset):
        spoilt, recycled = x.clone(), st.clone()
        spoilt[0, at], recycled[0] = bad, bad
        got = both(spoilt, recycled, gy)
        assert torch.equal(got[0][0, reset:], y[0, reset:]) and torch.equal(got[1], s) and torch.equal(got[2][0, reset:], dx[0, reset:])
        assert torch.equal(got[0][1], y[1]) and torch.equal(got[2][1], dx[1]) and not bool(torch.isfinite(got[0][0, at]).any())
    for at in range(reset, min(L, reset + K)):
        gy_bad, spoilt = gy.clone(), x.clone()
        gy_bad[0, at], spoilt[0, at] = bad, bad
        got = both(spoilt, st, gy_bad)
        assert torch.equal(got[0][0, :reset], y[0, :reset]) and torch.equal(got[2][0, :reset], dx[0, :reset]) and torch.equal(got[3], ds)
