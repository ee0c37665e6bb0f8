"""The root-mean-square norm (with the residual's addition, 8-bit output) and clipping by the gradients' norm against float64.

Tolerances.  A row's sum of D <= 8192 squares by 32 or 256 threads has at most 8192 / 32 + 8 additions in a chain, and rstd half of its error
and 2^-22: (64 + 8) x 2^-24 / 2 + 2^-22 < 3e-6 for y; the backward has that twice and another row sum: 1e-5.  dw adds rows in fp32: 1e-5
up to 2000 rows a block.  dx = rstd (dy w - xh mean(dy w xh)) is a difference, whose terms are off by 2^-24 each however small it
is (at D = 1 it is eps-sized): its error is relative to rstd |dy w| too.  A bfloat16 output is off by 2^-8 of its value more, an e4m3 one by 2^-4 of it or half its smallest
step of 2^-9 scale.
"""
import pytest
import torch

import ops_oracle as orc
import srwm_b200 as sb
from srwm_b200.dist import GradBucket

pytestmark = pytest.mark.gpu


def _near(got, want, tol, what="", terms=0.0):
    err = (got.double() - want).abs()
    bound = tol * max(float(want.abs().max()), terms) + (2.0 ** -8 * want.abs() if got.dtype == torch.bfloat16 else 0.0) + 1e-30
    assert bool((err <= bound).all()), (what, float((err / bound).max()))


def _rand(*s, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(s))
    return torch.randn(*s, device="cuda", generator=g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 5), (7, 64), (9, 130), (33, 256), (48, 257), (5, 512), (17, 1000), (12, 1024), (6, 1030),
                                    (5, 2048), (3, 4001), (4, 8192), (5000, 96)])
def test_rms_norm(rows, D, residual, dtype):
    x, w = _rand(rows, D).to(dtype), 1 + 0.3 * _rand(D, seed=1)
    res = (3 * _rand(rows, D, seed=2)).to(dtype) if residual else None
    gy, gs = _rand(rows, D, seed=3).to(dtype), _rand(rows, D, seed=4).to(dtype)
    ref = [t.double().requires_grad_() if t is not None else None for t in (x, w, res)]
    yr, sr = orc.rms(*ref, dtype=dtype)
    args = [t.clone().requires_grad_() if t is not None else None for t in (x, w, res)]
    leaves, rleaves = [t for t in args if t is not None], [t for t in ref if t is not None]
    if residual:
        y, s = sb.rms_norm(args[0], args[1], residual=args[2])
        assert torch.equal(s.double(), sr)
        got, want = torch.autograd.grad([y, s], leaves, [gy, gs]), torch.autograd.grad([yr, sr], rleaves, [gy.double(), gs.double()])
    else:
        y = sb.rms_norm(args[0], args[1])
        got, want = torch.autograd.grad(y, leaves, gy), torch.autograd.grad(yr, rleaves, gy.double())
    _near(y.detach(), yr.detach(), 3e-6, "y")
    terms = float((torch.rsqrt((sr.detach() ** 2).mean(-1, keepdim=True) + 1e-6) * (gy.double() * w.double()).abs()).max())
    for a, b, t in zip(got, want, leaves):
        assert a.dtype == t.dtype
        _near(a, b, 1e-5, terms=0.0 if t is args[1] else terms)
    with torch.no_grad():
        r = sb.rms_norm_fp8(x, w, residual=res)
        q, scale = r[0], r[1]
        assert q.dtype == torch.float8_e4m3fn and scale.shape == (rows, 1) and len(r) == (3 if residual else 2)
        if residual:
            assert torch.equal(r[2].double(), sr)
        yd = yr.detach()
        _near(scale, yd.abs().amax(-1, keepdim=True) / 448, 4e-6)
        assert bool(((q.double() * scale.double() - yd).abs() <= 2.0 ** -4 * yd.abs() * 1.001 + 2.0 ** -10 * 1.001 * scale.double()).all())
        assert float(q.float().abs().amax()) == 448.0


def test_rms_rows_of_other_strides():
    wide = _rand(6, 7, 100).to(torch.bfloat16)
    for x in (wide[..., 3:67], wide[:, 1, :64], wide.transpose(0, 1)[..., :64], wide[:, :, :100:2], wide[2, 3, :64]):
        w = 1 + 0.3 * _rand(x.shape[-1])
        a, b = x.detach().clone().requires_grad_(), x.double().requires_grad_()
        y, yr = sb.rms_norm(x, w), orc.rms(b, w.double())[0]
        assert y.shape == x.shape
        _near(y, yr.detach(), 3e-6)
        y, s = sb.rms_norm(x, w, residual=x)
        _near(s, 2 * x.double(), 1e-30)
        go = _rand(*x.shape, seed=5).to(torch.bfloat16)
        view = x.detach().requires_grad_()
        _near(torch.autograd.grad(sb.rms_norm(view, w), view, go)[0], torch.autograd.grad(yr, b, go.double())[0], 1e-5)
        expanded = torch.ones(1, device="cuda", dtype=torch.bfloat16).expand(x.shape)
        _near(torch.autograd.grad(sb.rms_norm(a, w), a, expanded)[0], torch.autograd.grad(orc.rms(b, w.double())[0], b, expanded.double())[0], 1e-5)


def test_rms_rows_that_are_zero_infinite_or_nan():
    x, w = _rand(5, 40), torch.ones(40, device="cuda")
    x[1] = 0.0
    x[2, 7] = float("inf")
    x[3, 9] = float("nan")
    x[4] *= 1e-30
    y = sb.rms_norm(x, w)
    want = orc.rms(x.double(), w.double())[0]
    _near(y[[0, 1, 4]], want[[0, 1, 4]], 3e-6)
    assert not bool(y[1].any()) and bool(y[2, 7].isnan()) and not bool(y[2, :7].any()) and bool(y[3].isnan().all())
    with torch.no_grad():
        q, scale = sb.rms_norm_fp8(x, w)
    assert not bool(q[1].float().any()) and float(scale[1]) == 2.0 ** -126 and bool(q[3].float().isnan().all())
    assert not bool(q[4].float().isnan().any()) and bool(scale[3].isnan())


def test_rms_refused():
    x, w = _rand(4, 64), _rand(64)
    for args, kw, error in (((x, w[:60]), {}, ValueError), ((x.half(), w), {}, TypeError), ((x, w.double()), {}, TypeError),
                            ((x, w), {"residual": x[:3]}, ValueError), ((x, w), {"residual": x.cpu()}, RuntimeError),
                            ((_rand(2, 8200), _rand(8200)), {}, ValueError), ((x, w.cpu()), {}, RuntimeError)):
        with pytest.raises(error):
            sb.rms_norm(*args, **kw)
    with pytest.raises(ValueError):
        sb.rms_norm_fp8(x.clone().requires_grad_(), w)
    y, s = sb.rms_norm(x[:0], w, residual=x[:0])
    assert y.shape == (0, 64) and s.shape == (0, 64)


# ---- gradients ----
# squares over 32 values a thread in fp32: 32 x 2^-24 of the sum, half of it in the norm: 1e-6; a scaled value has that and two roundings

def _params(shapes, dtypes, seed=0, scale=1.0):
    out = []
    for i, s in enumerate(shapes):
        p = torch.nn.Parameter(torch.empty(s, device="cuda", dtype=dtypes[i % len(dtypes)]))
        p.grad = (_rand(*s, seed=seed + i) * scale).to(p.dtype)
        out.append(p)
    return out


@pytest.mark.parametrize("shapes,dtypes", [
    ([(1,)], [torch.float32]), ([(3,), (0,), (17, 5)], [torch.float32]), ([(8191,), (8192,), (8193,), (2, 3, 4)], [torch.float32, torch.bfloat16]),
    ([(300, 301)] * 3 + [(7,)] * 61, [torch.bfloat16]), ([(31,)] * 65, [torch.float32, torch.bfloat16]), ([(5,)] * 2100, [torch.float32]),
    ([(3000, 1000), (1 << 20,)], [torch.float32])])
def test_clip(shapes, dtypes):
    for max_norm in (0.5, 1e9):
        ps = _params(shapes, dtypes)
        norm, want = orc.clip([p.grad for p in ps], max_norm)
        assert abs(float(sb.grad_norm([p.grad for p in ps])) / float(norm) - 1) < 1e-6
        before = [p.grad.clone() for p in ps]
        version = [p.grad._version for p in ps]
        got = sb.clip_grad_norm_(ps, max_norm)
        assert got.shape == () and got.dtype == torch.float32 and abs(float(got) / float(norm) - 1) < 1e-6
        for p, w, b, v in zip(ps, want, before, version):
            assert p.grad._version > v
            if max_norm > 1e6:
                assert torch.equal(p.grad, b)
            elif p.numel():
                _near(p.grad, w, 1.5e-6)
    again = _params(shapes, dtypes)
    sb.clip_grad_norm_(again, 0.5)
    ps = _params(shapes, dtypes)
    sb.clip_grad_norm_(ps, 0.5)
    assert all(torch.equal(a.grad, b.grad) for a, b in zip(again, ps))      # the sums have one order


def test_clip_views_and_torch_s_values():
    ps = _params([(64, 33), (40, 20), (6, 4, 8, 2)], [torch.float32])
    ps[0].grad = torch.randn(33, 64, device="cuda").t()
    ps[1].grad = torch.randn(40, 41, device="cuda")[:, 1:21]
    ps[2].grad = ps[2].grad.contiguous(memory_format=torch.channels_last)
    odd = torch.randn(1001, device="cuda")
    p = torch.nn.Parameter(torch.empty(1000, device="cuda"))
    p.grad = odd[1:]                        # not on a 16-byte boundary
    ps.append(p)
    other = [torch.nn.Parameter(q.detach().clone()) for q in ps]
    for a, b in zip(other, ps):
        a.grad = b.grad.clone()
    first = float(odd[0])
    n1, n2 = sb.clip_grad_norm_(iter(ps), 0.7), torch.nn.utils.clip_grad_norm_(other, 0.7)
    assert abs(float(n1) / float(n2) - 1) < 2e-6 and float(odd[0]) == first
    for a, b in zip(ps, other):
        _near(a.grad, b.grad.double(), 2e-6)


def test_clip_values_that_are_not_finite():
    for bad, norm in ((float("nan"), "nan"), (float("inf"), "inf")):
        ps, other = _params([(50,), (70,)], [torch.float32]), _params([(50,), (70,)], [torch.float32])
        for q in (ps, other):
            q[0].grad[3] = bad
        assert str(float(sb.clip_grad_norm_(ps, 1.0))) == norm
        torch.nn.utils.clip_grad_norm_(other, 1.0, foreach=False)
        for a, b in zip(ps, other):
            assert torch.equal(a.grad.isnan(), b.grad.isnan()) and torch.equal(a.grad.nan_to_num(5.0), b.grad.nan_to_num(5.0))
        ps = _params([(50,), (70,)], [torch.float32])
        ps[1].grad[0] = bad
        keep = ps[0].grad.clone()
        with pytest.raises(RuntimeError):
            sb.clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)
        assert torch.equal(ps[0].grad, keep)


def test_clip_refused_and_the_bucket():
    ps = _params([(50,), (70,)], [torch.float32])
    flat = torch.randn(100, device="cuda")
    for grads, error in (([flat, flat], ValueError), ([flat[:60], flat[50:]], ValueError), ([flat.half()], TypeError),
                         ([flat, torch.zeros(3)], RuntimeError), ([flat.double()], TypeError)):
        keep = flat.clone()
        with pytest.raises(error):
            sb.grad_ops.clip_tensors_(grads, 1.0)
        assert torch.equal(flat, keep)
    b = GradBucket([(2, 3), (5,)], "cuda")
    b.view(0).fill_(3.0)
    b.view(1).fill_(-4.0)
    assert abs(float(b.clip_(2.0)) - (9.0 * 6 + 16.0 * 5) ** 0.5) < 1e-5 and abs(float(b.flat.norm()) - 2.0) < 1e-5


def test_clip_of_views_that_share_values():
    """Views with gaps that overlap are refused before anything is scaled; those side by side in one buffer are scaled."""
    wide, dense = torch.randn(40, 41, device="cuda"), torch.randn(50, device="cuda")
    for grads in ([dense, wide[:, 1:20], wide[:, 1:20]], [wide[:, :20], wide[:, 19:], dense], [wide[:, 3], wide], [dense, wide[:1].expand(3, -1)]):
        keep, rest = wide.clone(), dense.clone()
        with pytest.raises(ValueError, match="overlap"):
            sb.grad_ops.clip_tensors_(grads, 1.0)
        ps = [torch.nn.Parameter(torch.empty(g.shape, device="cuda")) for g in grads]
        for p, g in zip(ps, grads):
            p.grad = g
        with pytest.raises(ValueError, match="overlap"):
            sb.clip_grad_norm_(ps, 1.0)
        assert torch.equal(wide, keep) and torch.equal(dense, rest)
    norm, want = orc.clip([wide], 0.5)
    got = sb.grad_ops.clip_tensors_([wide[:, 20:], wide[:, :20:2], wide[:, 1:20:2]], 0.5)
    assert abs(float(got) / float(norm) - 1) < 1e-6
    _near(wide, want[0], 1.5e-6)


def test_norm_of_tensors_that_share_values():
    """Nothing is written: a tensor counts as often as it is there, views and expanded ones among them."""
    wide = torch.randn(40, 41, device="cuda")
    for ts in ([wide, wide], [wide, wide[3:9]], [wide[:, 2:30], wide[:, 2:30], wide[:, 3]], [wide[:1].expand(7, -1), wide.to(torch.bfloat16)]):
        norm, _ = orc.clip(ts, 1.0)
        assert abs(float(sb.grad_norm(ts)) / float(norm) - 1) < 1e-6
