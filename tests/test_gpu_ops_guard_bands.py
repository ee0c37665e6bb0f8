"""Every tensor that the scan, convolution, norm and clipping kernels write lies between guard bands in a buffer of 0xFF bytes, working
memory included: the bands stay as they were, no byte pattern of the fill (a NaN) is left inside, and the results are those of the
ordinary path.  Odd sizes, several pieces of the time axis, channels that end inside a block."""
import ctypes as C

import pytest
import torch

import srwm_b200 as sb
from srwm_b200 import _lib as L
from srwm_b200.ops import _stream

pytestmark = pytest.mark.gpu
BAND = 512


class Banded:
    def __init__(self, *shape, dtype=torch.float32, filled=True):
        self.filled = filled
        n = 1
        for s in shape:
            n *= s
        self.bytes = n * torch.empty((), dtype=dtype).element_size()
        room = (self.bytes + 15) // 16 * 16
        self.raw = torch.full((room + 2 * BAND,), 255, dtype=torch.uint8, device="cuda")
        self.t = self.raw[BAND:BAND + self.bytes].view(dtype).view(shape)

    def ptr(self):
        return self.t.data_ptr()

    def check(self):
        assert bool((self.raw[:BAND] == 255).all()) and bool((self.raw[BAND + self.bytes:] == 255).all())
        if self.filled:
            assert not bool(self.t.float().isnan().any())


def _rows(b):
    t = b.t if isinstance(b, Banded) else b
    return L.Rows(t.data_ptr(), t.stride(0), t.stride(1))


def _bc(b):
    t = b.t if isinstance(b, Banded) else b
    return L.Seq(t.data_ptr(), t.stride(0), t.stride(2), t.stride(1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,Ln,D,S,G", [(2, 13, 33, 16, 1), (1, 300, 66, 8, 3), (3, 37, 70, 32, 2), (1, 260, 30, 64, 1), (2, 9, 130, 16, 1), (1, 3, 5, 16, 1)])
def test_scan(N, Ln, D, S, G, dtype):
    g = torch.Generator(device="cuda").manual_seed(Ln + D)
    r = lambda *s, dt=dtype: torch.randn(*s, device="cuda", generator=g).to(dt)  # noqa: E731
    u, delta, z, Bm, Cm, dy = r(N, Ln, D), r(N, Ln, D), r(N, Ln, D), r(N, Ln, G, S), r(N, Ln, G, S), r(N, Ln, D)
    A, skip, bias, h0, dh = -torch.rand(D, S, device="cuda", generator=g) - 0.2, *(r(*s, dt=torch.float32) for s in ((D,), (D,), (N, D, S), (N, D, S)))
    done = (torch.rand(N, Ln, device="cuda", generator=g) < 0.1).to(torch.uint8)
    lib = L.load()
    a = L.ScanArgs()
    a.N, a.L, a.D, a.S, a.G, a.io_dtype, a.softplus = N, Ln, D, S, G, L.BF16 if dtype == torch.bfloat16 else L.F32, 1
    a.u, a.delta, a.z, a.B, a.C = _rows(u), _rows(delta), _rows(z), _bc(Bm), _bc(Cm)
    a.A, a.skip, a.delta_bias, a.state_in, a.done = A.data_ptr(), skip.data_ptr(), bias.data_ptr(), h0.data_ptr(), done.data_ptr()
    a.done_stride_n, a.done_stride_l = Ln, 1
    need = lib.srwm_b200_scan_scratch_bytes(N, Ln, D, S, G)
    y, hT, ck = Banded(N, Ln, D, dtype=dtype), Banded(N, D, S), Banded(lib.srwm_b200_scan_checkpoint_floats(N, Ln, D, S))
    work = Banded(max(need, 16) // 4, filled=False)
    a.y, a.state_out, a.checkpoints, a.scratch, a.scratch_bytes = _rows(y), hT.ptr(), ck.ptr(), work.ptr(), need
    L.check(lib.srwm_b200_scan_forward(C.byref(a), _stream(u)), "scan")
    for b in (y, hT, ck, work):
        b.check()
    shape = (N, Ln, S) if G == 1 else (N, Ln, G, S)
    leaves = [t.requires_grad_() for t in (u, delta, A, Bm, Cm, skip, z, bias, h0)]
    want = sb.selective_scan(u, delta, A, Bm.view(shape), Cm.view(shape), skip, z, bias, h0, done)
    assert torch.equal(y.t, want[0]) and torch.equal(hT.t, want[1])
    grads = torch.autograd.grad(list(want), leaves, [dy, dh])
    need = lib.srwm_b200_scan_backward_scratch_bytes(N, Ln, D, S, G)
    work = Banded(need // 4, filled=False)
    a.scratch, a.scratch_bytes = work.ptr(), need
    outs = [Banded(*t.shape, dtype=t.dtype) for t in leaves]
    o = L.ScanGrads()
    o.dy, o.dstate_out = _rows(dy), dh.data_ptr()
    o.du, o.ddelta, o.dA, o.dB, o.dC, o.dskip, o.dz, o.ddelta_bias, o.dstate_in = (
        _rows(outs[0]), _rows(outs[1]), outs[2].ptr(), _bc(outs[3]), _bc(outs[4]), outs[5].ptr(), _rows(outs[6]), outs[7].ptr(), outs[8].ptr())
    L.check(lib.srwm_b200_scan_backward(C.byref(a), C.byref(o), _stream(u)), "scan")
    for b, w in zip(outs, grads):
        b.check()
        assert torch.equal(b.t, w)
    work.check()
    ck.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,Ln,D,K", [(2, 1, 5, 4), (3, 2, 33, 3), (2, 50, 130, 4), (1, 400, 36, 2)])
def test_conv(N, Ln, D, K, dtype):
    g = torch.Generator(device="cuda").manual_seed(Ln + D)
    r = lambda *s, dt=dtype: torch.randn(*s, device="cuda", generator=g).to(dt)  # noqa: E731
    x, s0, dy, ds = r(N, Ln, D), r(N, K - 1, D), r(N, Ln, D), r(N, K - 1, D)
    w, b = r(D, K, dt=torch.float32), r(D, dt=torch.float32)
    lib = L.load()
    a = L.ConvArgs()
    a.N, a.L, a.D, a.K, a.io_dtype, a.silu = N, Ln, D, K, L.BF16 if dtype == torch.bfloat16 else L.F32, 1
    a.x, a.w, a.bias, a.state_in = _rows(x), w.data_ptr(), b.data_ptr(), _rows(s0)
    y, sT = Banded(N, Ln, D, dtype=dtype), Banded(N, K - 1, D, dtype=dtype)
    a.y, a.state_out = _rows(y), _rows(sT)
    L.check(lib.srwm_b200_conv_forward(C.byref(a), _stream(x)), "conv")
    leaves = [t.requires_grad_() for t in (x, w, b, s0)]
    want = sb.causal_conv(x, w, b, s0)
    for o, v in zip((y, sT), want):
        o.check()
        assert torch.equal(o.t, v)
    need = lib.srwm_b200_conv_scratch_bytes(N, Ln, D, K)
    outs, work = [Banded(*t.shape, dtype=t.dtype) for t in leaves], Banded(need // 4, filled=False)
    o = L.ConvGrads()
    o.dy, o.dstate_out, o.dx, o.dw, o.dbias, o.dstate_in = _rows(dy), _rows(ds), _rows(outs[0]), outs[1].ptr(), outs[2].ptr(), _rows(outs[3])
    o.scratch, o.scratch_bytes = work.ptr(), need
    L.check(lib.srwm_b200_conv_backward(C.byref(a), C.byref(o), _stream(x)), "conv")
    for v, k in zip(torch.autograd.grad(list(want), leaves, [dy, ds]), outs):
        k.check()
        assert torch.equal(k.t, v)
    work.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,D", [(1, 3), (9, 130), (33, 1024), (5, 1500), (700, 64)])
def test_rms(rows, D, dtype):
    x, res, dy, ds = (torch.randn(rows, D, device="cuda").to(dtype) for _ in range(4))
    w = torch.rand(D, device="cuda")
    lib = L.load()
    for fp8 in (False, True):
        a = L.RmsArgs()
        a.rows, a.D, a.io_dtype, a.eps = rows, D, L.BF16 if dtype == torch.bfloat16 else L.F32, 1e-6
        a.x, a.residual, a.x_stride, a.residual_stride, a.w = x.data_ptr(), res.data_ptr(), D, D, w.data_ptr()
        y = Banded(rows, D, dtype=torch.float8_e4m3fn if fp8 else dtype)
        s, rstd, scale = Banded(rows, D, dtype=dtype), Banded(rows), Banded(rows)
        a.y, a.sum, a.rstd, a.scale = y.ptr(), s.ptr(), rstd.ptr(), scale.ptr() if fp8 else None
        L.check(lib.srwm_b200_rms_forward(C.byref(a), _stream(x)), "rms")
        for b in (y, s, rstd) + ((scale,) if fp8 else ()):
            b.check()
        with torch.no_grad():
            want = (sb.rms_norm_fp8 if fp8 else sb.rms_norm)(x, w, residual=res)
        assert torch.equal(y.t.float(), want[0].float()) and torch.equal(s.t, want[-1])
    dx, dw, need = Banded(rows, D, dtype=dtype), Banded(D), lib.srwm_b200_rms_scratch_bytes(rows, D)
    work = Banded(need // 4, filled=False)
    o = L.RmsGrads(rows, D, a.io_dtype, s.ptr(), dy.data_ptr(), ds.data_ptr(), D, D, D, w.data_ptr(), rstd.ptr(), dx.ptr(), dw.ptr(), work.ptr(), need)
    L.check(lib.srwm_b200_rms_backward(C.byref(o), _stream(x)), "rms")
    for b in (dx, dw, work, s, rstd):
        b.check()


def test_clip():
    sizes = [1, 7, 8191, 8193, 40000]
    for dtype in (torch.float32, torch.bfloat16):
        ts = [Banded(n, dtype=dtype) for n in sizes]
        for b in ts:
            b.t.normal_()
        want = [b.t.double() for b in ts]
        norm = sum((v * v).sum() for v in want).sqrt()
        lib = L.load()
        list_ = (L.TensorDesc * len(ts))(*[L.TensorDesc(b.ptr(), b.t.numel(), L.BF16 if dtype == torch.bfloat16 else L.F32, 0) for b in ts])
        need = lib.srwm_b200_grads_scratch_bytes(list_, len(ts))
        out, work = Banded(1), Banded(need // 4, filled=False)
        L.check(lib.srwm_b200_grads_clip(list_, len(ts), 0.5, out.ptr(), work.ptr(), need, _stream(ts[0].t)), "clip")
        for b, v in zip(ts, want):
            b.check()
            assert float((b.t.double() - v * 0.5 / norm).abs().max()) <= (2.0 ** -8 + 2e-6) * float((v * 0.5 / norm).abs().max())
        out.check()
        work.check()
        assert abs(float(out.t) / float(norm) - 1) < 1e-6
