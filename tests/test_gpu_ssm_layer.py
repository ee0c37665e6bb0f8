"""The state-space layer and its operators as they are used together: a stack in training (scan, convolution, norm with the
residual's addition, clipping), state carried between calls and steps, episode resets, captured graphs, other streams.

Tolerances: the layer is five linear maps (3e-6 each, tests/test_gpu_linear.py) around operators of 1.5e-5 (y) and 7.5e-5 (gradients,
tests/test_gpu_scan.py); two layers in a row double it: 1e-4 and 5e-4 of the largest value.
"""
import pytest
import torch

import ops_oracle as orc
import srwm_b200 as sb
from srwm_b200.layers import SSMlayer

pytestmark = pytest.mark.gpu
FWD, GRAD = 1e-4, 5e-4


def _near(got, want, tol, what=""):
    err = float((got.double() - want).abs().max())
    assert err <= tol * float(want.abs().max()) + 1e-30, (what, err, float(want.abs().max()))


def _layer(in_dim, seed, **kw):
    torch.manual_seed(seed)
    layer = SSMlayer(in_dim, **kw).cuda()
    with torch.no_grad():
        layer.step_bias.add_(2.0)      # steps of 0.007 to 0.5: memories that end
    return layer


def _oracle(layer, p, h, state, done, residual=None):
    """The layer's lines in float64 on the step-by-step definitions; p: its parameters."""
    x, s = orc.rms(h, p["norm_weight"], residual, layer.norm_eps, dtype=torch.float32)
    conv, scan = (None, None) if state is None else state
    done = None if done is None else done.t()
    xz = (x @ p["in_linear.weight"].t()).transpose(0, 1)
    x, z = xz.split(layer.inner, -1)
    x, conv = orc.conv(x, p["conv_weight"], p["conv_bias"], conv, done)
    rows = x @ p["x_linear.weight"].t()
    step, B, C = rows.split([layer.rank, layer.state_dim, layer.state_dim], -1)
    y, scan = orc.scan(x, step @ p["step_linear.weight"].t(), -torch.exp(p["A_log"]), B, C, p["D"], z, p["step_bias"], scan, done)
    return s + y.transpose(0, 1) @ p["out_linear.weight"].t(), (conv, scan)


@pytest.mark.parametrize("L,B,dim,S,done,carried", [(20, 3, 32, 16, True, True), (33, 2, 64, 8, False, False), (100, 2, 48, 32, True, False), (5, 4, 256, 16, True, True)])
def test_layer_against_its_lines(L, B, dim, S, done, carried):
    layer = _layer(dim, L, state_dim=S)
    g = torch.Generator(device="cuda").manual_seed(L + B)
    h, res, go = (torch.randn(L, B, dim, device="cuda", generator=g) for _ in range(3))
    flags = torch.rand(L, B, device="cuda", generator=g) < 0.1 if done else None
    state = tuple(torch.randn(t.shape, device="cuda", generator=g) * 0.3 for t in layer.init_state(B)) if carried else None
    p = {k: v.detach().double().requires_grad_() for k, v in layer.named_parameters()}
    h64, r64 = h.double().requires_grad_(), res.double().requires_grad_()
    s64 = None if state is None else tuple(t.double().requires_grad_() for t in state)
    ref, ref_state = _oracle(layer, p, h64, s64, flags, r64)
    want = torch.autograd.grad(ref, [h64, r64, *p.values()] + list(s64 or ()), go.double())
    h1, r1 = h.clone().requires_grad_(), res.clone().requires_grad_()
    s1 = None if state is None else tuple(t.clone().requires_grad_() for t in state)
    out, st = layer(h1, s1, flags, get_state=True, residual=r1)
    got = torch.autograd.grad(out, [h1, r1, *layer.parameters()] + list(s1 or ()), go)
    _near(out.detach(), ref.detach(), FWD)
    for a, b in zip(st, ref_state):
        _near(a.detach(), b.detach(), FWD)
    for a, b, k in zip(got, want, ["h", "residual", *p] + ["conv state", "scan state"]):
        _near(a, b, GRAD, k)


def test_training_steps_of_a_stack():
    """Two layers, the second adding the first's output to the stream; three steps with clipping and plain gradient descent follow the
    same steps in float64."""
    layers = [_layer(64, k) for k in (1, 2)]
    g = torch.Generator(device="cuda").manual_seed(5)
    h, go = torch.randn(40, 3, 64, device="cuda", generator=g), torch.randn(40, 3, 64, device="cuda", generator=g)
    done = torch.rand(40, 3, device="cuda", generator=g) < 0.05
    params = [p for layer in layers for p in layer.parameters()]
    ref = [{k: v.detach().double().requires_grad_() for k, v in layer.named_parameters()} for layer in layers]
    for step in range(3):
        a = layers[0](h, done=done)
        out = layers[1](a, done=done, residual=h)
        grads = torch.autograd.grad(out, params, go)
        a64, _ = _oracle(layers[0], ref[0], h.double(), None, done)
        out64, _ = _oracle(layers[1], ref[1], a64, None, done, h.double())
        flat = [v for r in ref for v in r.values()]
        norm64, want = orc.clip(torch.autograd.grad(out64, flat, go.double()), 1.0)
        _near(out.detach(), out64.detach(), 2 * FWD)
        for p, v in zip(params, grads):
            p.grad = v.contiguous()
        norm = sb.clip_grad_norm_(params, 1.0)
        assert abs(float(norm) / float(norm64) - 1) < GRAD
        for p, w in zip(params, want):
            _near(p.grad, w, 2 * GRAD + 1e-3 * step)      # (the weights themselves have come apart by then)
        with torch.no_grad():
            for p, v, w in zip(params, flat, want):
                p -= 0.1 * p.grad
                v -= 0.1 * w


def test_steps_of_an_actor_are_the_sequence():
    """A sequence whole, in two parts and a token at a time with the state advanced in place, resets among them."""
    layer = _layer(64, 7, state_dim=16)
    g = torch.Generator(device="cuda").manual_seed(1)
    h = torch.randn(12, 5, 64, device="cuda", generator=g)
    done = torch.rand(12, 5, device="cuda", generator=g) < 0.2
    with torch.no_grad():
        whole, last = layer(h, layer.init_state(5), done, get_state=True)
        a, st = layer(h[:5], layer.init_state(5), done[:5], get_state=True)
        b, st = layer(h[5:], st, done[5:], get_state=True)
        _near(torch.cat([a, b]), whole.double(), 1e-5)
        state = layer.init_state(5)
        for t in range(12):
            out, st = layer(h[t:t + 1], state, done[t:t + 1], get_state=True, inplace_state=True)
            assert st[0] is state[0] or st[0].data_ptr() == state[0].data_ptr()
            _near(out, whole[t:t + 1].double(), 1e-5, t)
        for x, y in zip(state, last):
            _near(x, y.double(), 1e-5)


def test_captured_step_and_two_graphs():
    """Actor steps as graphs: replays advance the state; two captured graphs and eager calls in turn do not disturb one another."""
    layer = _layer(128, 3)
    hs = torch.randn(6, 1, 7, 128, device="cuda")
    with torch.no_grad():
        state = layer.init_state(7)
        want = [layer(h, state, inplace_state=True) for h in hs]
        graphs = []
        for k in range(2):
            buf, st = hs[0].clone(), layer.init_state(7)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                layer(buf, tuple(t.clone() for t in st), inplace_state=True)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = layer(buf, st, inplace_state=True)
            graphs.append((graph, buf, st, out))
        eager = layer.init_state(7)
        for t, h in enumerate(hs):
            for graph, buf, _, _ in graphs:
                buf.copy_(h)
                graph.replay()
            o = layer(h, eager, inplace_state=True)
            for r in (o, graphs[0][3], graphs[1][3]):
                assert torch.equal(r, want[t])
        assert torch.equal(graphs[0][2][1], eager[1]) and torch.equal(graphs[1][2][0], eager[0])


def test_captured_training_step():
    """Forward, backward and clipping of the operators in one graph give what they give outside."""
    layer = _layer(64, 9)
    h, go = torch.randn(30, 2, 64, device="cuda"), torch.randn(30, 2, 64, device="cuda")
    params = list(layer.parameters())

    def step():
        grads = torch.autograd.grad(layer(h), params, go)
        grads = [g.contiguous() for g in grads]
        return sb.grad_ops.clip_tensors_(grads, 1.0), grads
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        norm, grads = step()
    torch.cuda.current_stream().wait_stream(side)
    want = [norm.clone()] + [g.clone() for g in grads]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n2, g2 = step()
    for _ in range(3):
        graph.replay()
    for a, b in zip([n2] + g2, want):
        assert torch.equal(a, b)


def test_operators_on_another_stream():
    """Calls on a side stream, beside the same calls on the current one."""
    u, delta, z = (torch.randn(2, 300, 256, device="cuda") for _ in range(3))
    A, B, C = -torch.rand(256, 16, device="cuda") - 0.5, torch.randn(2, 300, 16, device="cuda"), torch.randn(2, 300, 16, device="cuda")
    w, cw = torch.rand(256, device="cuda"), torch.randn(256, 4, device="cuda")

    def calls():
        y, st = sb.selective_scan(u, delta, A, B, C, z=z)
        c, _ = sb.causal_conv(y, cw)
        return sb.rms_norm(c, w, residual=u), st, sb.grad_norm([c, y])
    want = calls()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = [calls() for _ in range(3)]
    b = [calls() for _ in range(3)]
    torch.cuda.synchronize()
    for r in a + b:
        assert torch.equal(r[0][0], want[0][0]) and torch.equal(r[0][1], want[0][1]) and torch.equal(r[1], want[1]) and torch.equal(r[2], want[2])


def test_bfloat16_layer_runs():
    layer = _layer(64, 4).to(torch.bfloat16)
    h = torch.randn(21, 2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    out, st = layer(h, layer.init_state(2), get_state=True)
    assert out.dtype == torch.bfloat16 and st[0].dtype == torch.bfloat16 and st[1].dtype == torch.float32
    grads = torch.autograd.grad(out.float().square().sum(), [h, *layer.parameters()])
    assert all(bool(torch.isfinite(g).all()) for g in grads)


def test_capture_beside_a_living_graph_is_refused():
    """A training step whose leaves belong to a living graph of the default stream is refused while its forward pass is captured; once
    that graph is gone the step is captured."""
    u = torch.randn(2, 9, 64, device="cuda")
    leaves = [torch.randn(64, 4, device="cuda", requires_grad=True), (-torch.rand(64, 16, device="cuda")).requires_grad_(),
              torch.rand(64, device="cuda").requires_grad_()]
    B, C = torch.randn(2, 9, 16, device="cuda"), torch.randn(2, 9, 16, device="cuda")
    ops = [lambda: sb.causal_conv(u, leaves[0])[0], lambda: sb.selective_scan(u, u, leaves[1], B, C)[0], lambda: sb.rms_norm(u, leaves[2])]
    for leaf, op in zip(leaves, ops):
        alive = op()
        want = torch.autograd.grad(alive, leaf, u, retain_graph=True)[0]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match="still alive"):
                op()
            keep = u * 2      # (a graph is not empty)
        del alive, graph, keep
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = torch.autograd.grad(op(), leaf, u)[0]
        graph.replay()
        assert torch.equal(got, want)
        del graph


def test_layer_under_autocast():
    """Projections in bfloat16, the norm and the states' types as they are: the carried state of one call fits the next."""
    layer = _layer(64, 6)
    h = torch.randn(12, 2, 64, device="cuda")
    with torch.no_grad():
        whole = layer(h)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            a, st = layer(h[:5], layer.init_state(2), get_state=True)
            b, st = layer(h[5:], st, get_state=True)
    assert st[1].dtype == torch.float32
    got = torch.cat([a, b]).double()
    # six results rounded to bf16 in a row (projection, convolution, two projections, scan, projection), half a step of 2^-8 each, and the
    # products' operands as much again: 12 x 2^-8 of the largest output
    _near(got, whole.double(), 12 * 2.0 ** -8)


def test_states_in_inference_mode():
    layer = _layer(64, 8)
    h = torch.randn(4, 3, 64, device="cuda")
    with torch.no_grad():
        state = layer.init_state(3)
        want = [layer(x[None], state, inplace_state=True) for x in h]
    with torch.inference_mode():
        state = layer.init_state(3)
        got = [layer(x[None], state, inplace_state=True) for x in h]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("N,L", [(0, 5), (3, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_calls_without_values_have_gradients(N, L, dtype):
    """A rank without sequences, an unroll without steps: every argument has a gradient, zeros, and a state its output's."""
    rows = lambda w: torch.randn(N, L, w, device="cuda", dtype=dtype, requires_grad=True)      # noqa: E731
    par = lambda *s: torch.randn(*s, device="cuda", requires_grad=True)      # noqa: E731
    u, delta, z, B, C, state = rows(32), rows(32), rows(32), rows(16), rows(16), par(N, 32, 16)
    leaves = [u, delta, par(32, 16), B, C, par(32), z, par(32), state]
    with torch.no_grad():
        leaves[2][0, 0] = float("inf")
    y, h = sb.selective_scan(*leaves)
    gs = torch.randn_like(h)
    grads = torch.autograd.grad([y, h], leaves, [torch.empty_like(y), gs])
    assert y.shape == (N, L, 32) and all(g.shape == t.shape and not bool(g.any()) for g, t in zip(grads[:-1], leaves)) and torch.equal(grads[-1], gs)
    y = sb.selective_scan(*leaves[:5])[0]
    assert all(not bool(g.any()) for g in torch.autograd.grad(y, leaves[:5], torch.empty_like(y)))
    window = torch.randn(N, 3, 32, device="cuda", dtype=dtype, requires_grad=True)
    leaves = [u, par(32, 4), par(32), window]
    y, h = sb.causal_conv(*leaves)
    gs = torch.randn_like(h)
    grads = torch.autograd.grad([y, h], leaves, [torch.empty_like(y), gs])
    assert y.shape == (N, L, 32) and not any(bool(g.any()) for g in grads[:-1]) and torch.equal(grads[-1], gs)
    w = par(32)
    y, s = sb.rms_norm(u, w, residual=z)
    assert not any(bool(g.any()) for g in torch.autograd.grad([y, s], [u, z, w], [torch.empty_like(y), torch.empty_like(s)]))
    y = sb.rms_norm(u, w)
    assert y.requires_grad and not bool(torch.autograd.grad(y, w, torch.empty_like(y))[0].any())
    with torch.no_grad():
        assert not sb.rms_norm(u, w).requires_grad and not sb.selective_scan(u, delta, leaves[1].new_zeros(32, 16), B, C)[0].requires_grad
    layer = _layer(32, 4).to(dtype)
    h = torch.randn(L, N, 32, device="cuda", dtype=dtype, requires_grad=True)
    out, st = layer(h, layer.init_state(N), torch.zeros(L, N, dtype=torch.bool, device="cuda"), get_state=True, residual=h)
    assert out.shape == (L, N, 32) and st[0].shape == (N, 3, 64) and st[1].shape == (N, 64, 16)
    assert not any(bool(g.any()) for g in torch.autograd.grad(out.sum(), [h, *layer.parameters()]))


def test_capture_of_a_layer_beside_a_living_graph_is_refused():
    """The same where the operators see casts and products of the leaves, not the leaves themselves; a graph that another stream has
    built is no obstacle."""
    layer = _layer(64, 11).to(torch.bfloat16)
    h = torch.randn(9, 2, 64, device="cuda", dtype=torch.bfloat16)
    params = list(layer.parameters())
    go = torch.randn_like(h)
    alive = layer(h)
    want = torch.autograd.grad(alive, params, go, retain_graph=True)
    weight = torch.randn(64, 64, device="cuda", requires_grad=True)
    other = (weight * 2).sum()
    for call in (lambda: layer(h), lambda: sb.rms_norm(torch.nn.functional.linear(h.float(), weight), torch.ones(64, device="cuda"))):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match="still alive"):
                call()
            keep = h * 2      # (a graph is not empty)
    del alive, other, graph, keep, call
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = layer(h)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(layer(h), params, go)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad(), torch.cuda.graph(torch.cuda.CUDAGraph()):
        layer(h)
