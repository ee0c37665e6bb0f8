"""CPU tests of the scan, convolution, norm and gradient entry points: structure layouts, refusals at the C ABI before any
CUDA call, refusals and host logic in Python."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest
import torch

import srwm_b200 as sb
from conftest import ROOT
from srwm_b200 import _lib as L
from srwm_b200.dist import GradBucket

PAIRS = {"srwm_b200_rows": L.Rows, "srwm_b200_scan_args": L.ScanArgs, "srwm_b200_scan_grads": L.ScanGrads, "srwm_b200_conv_args": L.ConvArgs,
         "srwm_b200_conv_grads": L.ConvGrads, "srwm_b200_rms_args": L.RmsArgs, "srwm_b200_rms_grads": L.RmsGrads, "srwm_b200_tensor": L.TensorDesc}


def test_structures_match_the_header():
    lines = []
    for name, cls in PAIRS.items():
        lines.append(f'printf("%zu ", sizeof({name}));')
        lines += [f'printf("%zu ", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "srwm_b200.h"\nint main(void) {' + "\n".join(lines) + "return 0;}"
    with tempfile.TemporaryDirectory() as td:
        with open(os.path.join(td, "t.c"), "w") as fh:
            fh.write(src)
        subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), os.path.join(td, "t.c"), "-o", os.path.join(td, "t")])
        got = [int(v) for v in subprocess.check_output([os.path.join(td, "t")], text=True).split()]
    want = []
    for cls in PAIRS.values():
        want.append(C.sizeof(cls))
        want += [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want


def _scan_args(**kw):
    a = L.ScanArgs()
    a.N, a.L, a.D, a.S, a.G, a.io_dtype, a.softplus = 2, 20, 64, 16, 1, L.F32, 1
    a.u = a.delta = a.y = L.Rows(0x1000, 1280, 64)
    a.B = a.C = L.Seq(0x1000, 320, 0, 16)
    a.A = 0x1000
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_scan_refusals():
    f = L.load().srwm_b200_scan_forward
    assert f(None, None) == L.ERR_NULL
    assert f(C.byref(_scan_args(N=-1)), None) == L.ERR_SHAPE
    assert f(C.byref(_scan_args(G=0)), None) == L.ERR_SHAPE
    assert f(C.byref(_scan_args(G=3)), None) == L.ERR_SHAPE
    assert f(C.byref(_scan_args(S=12)), None) == L.ERR_HEAD_DIM
    assert f(C.byref(_scan_args(io_dtype=5)), None) == L.ERR_DTYPE
    assert f(C.byref(_scan_args(A=None)), None) == L.ERR_NULL
    assert f(C.byref(_scan_args(u=L.Rows(None, 0, 0))), None) == L.ERR_NULL
    assert f(C.byref(_scan_args(y=L.Rows(None, 0, 0))), None) == L.ERR_NULL
    assert f(C.byref(_scan_args(A=0x1004)), None) == L.ERR_ALIGN
    assert f(C.byref(_scan_args(u=L.Rows(0x1002, 1280, 64))), None) == L.ERR_ALIGN
    assert f(C.byref(_scan_args(state_out=0x1008)), None) == L.ERR_ALIGN
    assert f(C.byref(_scan_args(N=1 << 20, D=1 << 20)), None) == L.ERR_SHAPE
    assert f(C.byref(_scan_args(N=1, L=(1 << 30) + 5)), None) == L.ERR_SHAPE
    assert f(C.byref(_scan_args(N=0)), None) == 0 and f(C.byref(_scan_args(D=0)), None) == 0
    # a long time axis of few channels is cut into pieces, which need scratch
    assert L.load().srwm_b200_scan_scratch_bytes(1, 4096, 64, 16, 1) > 0
    assert L.load().srwm_b200_scan_scratch_bytes(64, 4096, 2048, 16, 2) == 0
    assert f(C.byref(_scan_args(N=1, L=4096)), None) == L.ERR_NULL
    g, grads = L.load().srwm_b200_scan_backward, L.ScanGrads()
    assert g(C.byref(_scan_args()), None, None) == L.ERR_NULL
    assert g(C.byref(_scan_args()), C.byref(grads), None) == L.ERR_NULL
    assert g(C.byref(_scan_args(L=0)), C.byref(grads), None) == L.ERR_SHAPE
    assert L.load().srwm_b200_scan_checkpoint_floats(2, 17, 10, 8) == 2 * 3 * 10 * 8
    assert L.load().srwm_b200_scan_backward_scratch_bytes(2, 17, 12, 8, 5) == 0       # no such call


def _conv_args(**kw):
    a = L.ConvArgs()
    a.N, a.L, a.D, a.K, a.io_dtype, a.silu = 2, 20, 64, 4, L.F32, 1
    a.x = a.y = L.Rows(0x1000, 1280, 64)
    a.w = 0x1000
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_conv_refusals():
    f = L.load().srwm_b200_conv_forward
    assert f(None, None) == L.ERR_NULL
    assert f(C.byref(_conv_args(K=1)), None) == L.ERR_SHAPE and f(C.byref(_conv_args(K=5)), None) == L.ERR_SHAPE
    assert f(C.byref(_conv_args(L=-1)), None) == L.ERR_SHAPE
    assert f(C.byref(_conv_args(io_dtype=9)), None) == L.ERR_DTYPE
    assert f(C.byref(_conv_args(w=None)), None) == L.ERR_NULL and f(C.byref(_conv_args(x=L.Rows(None, 0, 0))), None) == L.ERR_NULL
    assert f(C.byref(_conv_args(x=L.Rows(0x1001, 1280, 64))), None) == L.ERR_ALIGN
    s = L.Rows(0x2000, 192, 64)
    assert f(C.byref(_conv_args(state_in=s, state_out=s)), None) == L.ERR_UNSUPPORTED     # in place, longer than a thread's steps
    assert f(C.byref(_conv_args(N=0)), None) == 0
    g = L.load().srwm_b200_conv_backward
    assert g(C.byref(_conv_args()), None, None) == L.ERR_NULL
    assert g(C.byref(_conv_args()), C.byref(L.ConvGrads()), None) == L.ERR_NULL


def test_rms_and_gradient_refusals():
    lib = L.load()
    a = L.RmsArgs()
    a.rows, a.D, a.io_dtype, a.x, a.w, a.y = 4, 9000, L.F32, 0x1000, 0x1000, 0x1000
    assert lib.srwm_b200_rms_forward(C.byref(a), None) == L.ERR_SHAPE
    a.D, a.w = 64, None
    assert lib.srwm_b200_rms_forward(C.byref(a), None) == L.ERR_NULL
    a.w, a.x = 0x1000, 0x1002
    assert lib.srwm_b200_rms_forward(C.byref(a), None) == L.ERR_ALIGN
    a.rows = 0
    assert lib.srwm_b200_rms_forward(C.byref(a), None) == 0
    assert lib.srwm_b200_rms_backward(C.byref(L.RmsGrads()), None) == L.ERR_SHAPE
    t = (L.TensorDesc * 2)(L.TensorDesc(0x1000, 8, L.F32, 0), L.TensorDesc(None, 8, L.F32, 0))
    assert lib.srwm_b200_grads_norm(t, -1, None, None, 0, None) == L.ERR_SHAPE
    assert lib.srwm_b200_grads_norm(t, 2, 0x1000, 0x1000, 1 << 20, None) == L.ERR_NULL
    assert lib.srwm_b200_grads_norm(t, 1, None, 0x1000, 1 << 20, None) == L.ERR_NULL
    assert lib.srwm_b200_grads_norm(t, 1, 0x1000, 0x1000, 0, None) == L.ERR_NULL
    assert lib.srwm_b200_grads_clip(t, 1, -1.0, 0x1000, 0x1000, 1 << 20, None) == L.ERR_SHAPE
    assert lib.srwm_b200_grads_clip(t, 1, float("nan"), 0x1000, 0x1000, 1 << 20, None) == L.ERR_SHAPE
    t[0].io_dtype = 3
    assert lib.srwm_b200_grads_norm(t, 1, 0x1000, 0x1000, 1 << 20, None) == L.ERR_DTYPE


def test_cpu_tensors_raise():
    x = torch.zeros(1, 2, 4)
    for call in (lambda: sb.selective_scan(x, x, torch.zeros(4, 8), torch.zeros(1, 2, 8), torch.zeros(1, 2, 8)),
                 lambda: sb.causal_conv(x, torch.zeros(4, 3)), lambda: sb.rms_norm(x, torch.ones(4)),
                 lambda: sb.rms_norm_fp8(x, torch.ones(4)), lambda: sb.grad_norm([x])):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        sb.clip_grad_norm_([p], 1.0)
    with pytest.raises(ValueError):
        sb.clip_grad_norm_([p], -1.0)
    p.grad = None
    assert float(sb.clip_grad_norm_([p], 1.0)) == 0.0 and float(sb.grad_norm([])) == 0.0
    with pytest.raises(TypeError):
        sb.selective_scan(None, x, x, x, x)


def test_bucket_clips_on_the_cpu():
    b = GradBucket([(2, 3), (5,)], "cpu")
    b.view(0).fill_(3.0)
    b.view(1).fill_(-4.0)
    want = (9.0 * 6 + 16.0 * 5) ** 0.5
    assert abs(float(b.clip_(2.0)) - want) < 1e-5
    assert abs(float(b.flat.norm()) - 2.0) < 1e-5
    assert abs(float(b.clip_(3.0)) - 2.0) < 1e-5 and abs(float(b.flat.norm()) - 2.0) < 1e-5


def test_rows_that_share_values():
    """What an in-place state must not be, against counting the addresses."""
    from srwm_b200.scan_ops import _apart
    base = torch.zeros(4096)
    seen = set()
    for n, l, d in ((1, 1, 5), (3, 1, 5), (1, 3, 5), (2, 3, 5), (4, 2, 8)):
        for sn in (0, 1, 4, 5, 8, 10, 15, 16, 20, 64):
            for sl in (0, 1, 4, 5, 8, 10, 12, 20, 32):
                rows = base.as_strided((n, l, d), (sn, sl, 1))
                where = [i * sn + j * sl + k for i in range(n) for j in range(l) for k in range(d)]
                apart = len(set(where)) == len(where)
                seen.add(apart)
                assert not _apart(rows) or apart, (n, l, d, sn, sl)              # never a race
                if sn % max(sl, 1) == 0 or sl % max(sn, 1) == 0:                 # and every nested order that there is
                    assert _apart(rows) == apart or (min(sn, sl) < d and n > 1 and l > 1), (n, l, d, sn, sl)
    assert seen == {True, False}


def test_gradients_that_share_values():
    """What clipping must not be given, against counting the bytes: no overlap is missed, and only a tensor whose own dimensions are not
    nested is taken to overlap without one."""
    import random
    from srwm_b200.grad_ops import _overlap
    base, rng, found = torch.zeros(4096), random.Random(1), 0
    for _ in range(2000):
        ts, where = [], []
        for _ in range(rng.choice((1, 2, 2, 3))):
            d, dtype = rng.choice((0, 1, 2, 3)), rng.choice((torch.float32, torch.bfloat16))
            shape, strides = [rng.choice((1, 2, 3, 4)) for _ in range(d)], [rng.choice((0, 1, 1, 2, 3, 4, 6, 8, 12, 24, 48)) for _ in range(d)]
            t = base.view(dtype).as_strided(shape, strides, rng.randrange(0, 60))
            ts.append(t)
            offsets = [t.storage_offset()]
            for n, st in zip(shape, strides):
                offsets = [o + i * st for o in offsets for i in range(n)]
            where += [o * t.element_size() + j for o in offsets for j in range(t.element_size())]
        shared = len(set(where)) != len(where)
        found += shared
        assert _overlap(ts) or not shared, ts
        assert shared or not _overlap(ts) or any(_overlap([t]) for t in ts), ts
    assert 500 < found < 1500
    wide = torch.zeros(40, 41)
    assert not _overlap([wide[:, :20], wide[:, 20:], torch.zeros(0)]) and not _overlap([wide[:, ::2], wide[:, 1::2]]) and not _overlap([wide[3:5].t(), wide[5:]])
    assert _overlap([wide[:, :20], wide[:, 19:]]) and _overlap([wide[:, ::2], wide[:, ::2]]) and _overlap([wide[:, 3], wide])
    assert _overlap([torch.zeros(1).expand(5)])


@pytest.mark.parametrize("D", [1 << 30, (1 << 31) - 1])
def test_channels_whose_blocks_are_not_counted_in_32_bits(D):
    lib = L.load()
    assert lib.srwm_b200_scan_forward(C.byref(_scan_args(N=1, L=1, D=D)), None) == L.ERR_SHAPE
    assert lib.srwm_b200_scan_scratch_bytes(1, 1, D, 16, 1) == 0 and lib.srwm_b200_scan_backward_scratch_bytes(1, 1, D, 16, 1) == 0
    assert lib.srwm_b200_conv_forward(C.byref(_conv_args(N=1, L=1, D=D)), None) == L.ERR_SHAPE
    assert lib.srwm_b200_conv_backward(C.byref(_conv_args(N=1, L=1, D=D)), C.byref(L.ConvGrads()), None) == L.ERR_SHAPE
    assert lib.srwm_b200_conv_scratch_bytes(1, 1, D, 4) == 0


def test_options_without_a_truth_value():
    x, several = torch.zeros(1, 2, 4), torch.ones(2)
    for call in (lambda: sb.selective_scan(x, x, torch.zeros(4, 8), x, x, delta_softplus=several), lambda: sb.causal_conv(x, torch.zeros(4, 3), silu=several),
                 lambda: sb.selective_scan(x, x, torch.zeros(4, 8), x, x, inplace_state=several),
                 lambda: sb.causal_conv(x, torch.zeros(4, 3), inplace_state=several)):
        with pytest.raises(RuntimeError, match="ambiguous"):
            call()


def test_clipping_an_iterator_that_is_empty():
    assert float(sb.grad_ops.clip_tensors_(iter(()), 1.0)) == 0.0 and float(sb.grad_norm(iter(()))) == 0.0
    assert float(sb.clip_grad_norm_(iter(()), 1.0)) == 0.0


def test_bucket_refuses_a_negative_norm_on_the_cpu():
    b = GradBucket([(4,)], "cpu")
    b.view(0).fill_(3.0)
    for most in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            b.clip_(most)
    assert bool((b.flat == 3.0).all())
