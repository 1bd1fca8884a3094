"""The row operators together, as the layer around the filter uses them: under
autograd, in a chain against the float64 definitions with the filter's own
calls in between, and the feature gradient from 8-bit checkpoints."""
import numpy as np
import pytest
import torch

import rows_reference as ref
from rows_reference import U, f64, half_step, worst

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


@pytest.fixture
def P():
    import plattice_pytorch_b200 as P
    yield P
    P.PLOO.set_checkpoint_precision("fp32")


def _randn(shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_linear_function_is_the_calls(dev, P, dtype, eight, act):
    R = P.rows
    leaf = lambda *s, seed: _randn(s, seed, dtype).to(dev).requires_grad_(True)  # noqa: E731
    x, w, b, r = leaf(6, 9, 64, seed=1), leaf(40, 64, seed=2), leaf(40, seed=3), leaf(6, 9, 40, seed=4)
    gy = _randn((6, 9, 40), 5, dtype).to(dev)
    y = P.RowLinearFunction.apply(x, w, b, r, act, eight)
    y.backward(gy)
    with torch.no_grad():
        ye, z = R.linear(x, w, b, act=act, residual=r, keep=None if act == "none" else "8bit" if eight else "full")
        kept = R.pack8(x) if eight and dtype != torch.float16 else x.detach()
        gx, gw, gb = R.linear_backward(gy, kept, w.detach(), z, act=act)
    for got, want in ((y, ye), (x.grad, gx), (w.grad, gw), (b.grad, gb), (r.grad, gy)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("split,act,residual", [(5, "none", False), (0, "silu", True)])
def test_norm_linear_function_is_the_calls(dev, P, dtype, split, act, residual):
    R = P.rows
    leaf = lambda *s, seed: _randn(s, seed, dtype).to(dev).requires_grad_(True)  # noqa: E731
    x, gain, w, b = leaf(50, 64, seed=1), leaf(64, seed=2), leaf(8, 64, seed=3), leaf(8, seed=4)
    r = leaf(50, 64, seed=5) if residual else None
    out = P.RowNormLinearFunction.apply(x, r, gain, w, b, 1e-6, act, split)
    out = out if isinstance(out, tuple) else (out,)
    gs = [_randn(tuple(o.shape), 6 + i, dtype).to(dev) for i, o in enumerate(out)]
    torch.autograd.backward(out, gs)
    with torch.no_grad():
        eight = dtype != torch.float16
        n, h, rstd = R.rms_norm(x, gain, r, pack=eight)
        y, z = R.linear(n, w, b, act=act, split=split, keep=None if act == "none" else "8bit" if eight else "full")
        g = (gs[0], gs[1]) if split else gs[0]
        gn, gw, gb = R.linear_backward(g, n, w.detach(), z, act=act)
        gx, gg = R.rms_norm_backward(gn, h.detach(), rstd, gain.detach(), gs[-1] if residual else None)
    for got, want in zip(out, (*(y if split else (y,)), *((h,) if residual else ()))):
        assert torch.equal(got, want)
    for got, want in ((x.grad, gx), (gain.grad, gg), (w.grad, gw), (b.grad, gb)):
        assert torch.equal(got, want)
    assert r is None or torch.equal(r.grad, gx)


def test_functions_give_only_the_wanted_gradients(dev, P):
    x, w = _randn((20, 64), 1).to(dev), _randn((8, 64), 2).to(dev)
    xg = x.clone().requires_grad_(True)
    P.RowLinearFunction.apply(xg, w, None, None).sum().backward()
    assert worst(f64(xg.grad), np.ones((20, 8)) @ f64(w), 20 * U * (np.ones((20, 8)) @ np.abs(f64(w)))) <= 1
    wg = w.clone().requires_grad_(True)
    P.RowLinearFunction.apply(x, wg, None, None, "relu").sum().backward()
    assert wg.grad.shape == w.shape
    gain = torch.ones(64, device=dev, requires_grad=True)
    f, v = P.RowNormLinearFunction.apply(x, None, gain, w, None, 1e-6, "none", 5)
    f.sum().backward()   # v's gradient is zeros
    assert gain.grad is not None


@pytest.mark.parametrize("shape,pd,vd,channels,act", [((13, 29), 5, 3, 64, "none"), ((24, 20), 2, 4, 50, "gelu"),
                                                      ((1, 7), 16, 8, 96, "silu")])
def test_layer_forward_and_gradients(dev, P, shape, pd, vd, channels, act):
    """float32 without 8-bit checkpoints: each operator's gradient against its
    definition in float64, from the values that the layer computed."""
    R, PLOO = P.rows, P.PLOO
    torch.manual_seed(0)
    m = P.PermutoLatticeLayer(channels, pd, vd, act=act, checkpoint8=False, device=dev)
    x = _randn(shape + (channels,), 7).to(dev).requires_grad_(True)
    gy = _randn(shape + (channels,), 8).to(dev)
    y = m(x)
    y.backward(gy)
    rows = shape[0] * shape[1]
    flat = lambda t: f64(t).reshape(rows, -1)  # noqa: E731
    with torch.no_grad():
        n, _, rstd = R.rms_norm(x, m.gain)
        (f, v), _ = R.linear(n, m.w_in, m.b_in, split=pd, out_dtype=torch.float32)
        weight, o, lat = PLOO.lattice_forward(f, v)
    ne, _, re_ = ref.rms_norm(flat(x), f64(m.gain))
    assert worst(flat(n), ne, 65 * U * np.abs(ne)) <= 1
    fe, _ = ref.linear(flat(n), f64(m.w_in), f64(m.b_in))
    tol = 2 * U * (channels + 8) * (np.abs(flat(n)) @ np.abs(f64(m.w_in)).T) + U * np.abs(fe)
    assert worst(np.concatenate([flat(f), flat(v)], 1), fe, tol) <= 1
    # the lattice sums of two calls differ in the order of their additions (1e-5 relative + 5e-6, as for the filter)
    ye, ze = ref.linear(flat(o), f64(m.w_out), f64(m.b_out), act, flat(x))
    tol = 2 * (1e-5 * np.abs(flat(o)) + 5e-6) @ np.abs(f64(m.w_out)).T + 2.0 ** -18 * (np.abs(ze) + np.abs(ye)) + 1e-6
    assert worst(flat(y), ye, tol) <= 1
    # gradients: through the filter's own backward calls
    with torch.no_grad():
        _, z = R.linear(o, m.w_out, m.b_out, act=act, keep=None if act == "none" else "full")
        go, gwo, gbo = R.linear_backward(gy, o, m.w_out, z, act=act)
        gf = PLOO.feature_grad(lat, f, v, go, weight, o)
        gv = PLOO.lattice_backward(f, go, weight, lat)
        gn, gwi, gbi = R.linear_backward((gf, gv), n, m.w_in)
        gx, gg = R.rms_norm_backward(gn, x.detach(), rstd, m.gain, gy)
    for got, want in ((m.w_out.grad, gwo), (m.b_out.grad, gbo), (m.w_in.grad, gwi), (m.b_in.grad, gbi),
                      (m.gain.grad, gg), (x.grad, gx)):
        # atomics in the filter's splat: the two passes differ by their order
        scale = float(want.abs().max())
        assert float((got - want).abs().max()) <= 2e-4 * scale


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_layer_with_checkpoints_in_8_bits(dev, P, dtype):
    torch.manual_seed(1)
    m = P.PermutoLatticeLayer(64, 5, 3, act="silu", dtype=dtype, device=dev)
    x = _randn((16, 24, 64), 9, dtype).to(dev).requires_grad_(True)
    for precision in ("fp32", "8bit"):
        P.PLOO.set_checkpoint_precision(precision)
        y = m(x)
        assert y.shape == x.shape and y.dtype == dtype
        grads = torch.autograd.grad(y.float().square().mean(), [x, *m.parameters()])
        for g, p in zip(grads, [x, *m.parameters()]):
            assert g.shape == p.shape and g.dtype == p.dtype and bool(torch.isfinite(g).all()) and bool(g.any())


@pytest.mark.parametrize("shape,pd,vd", [((16, 24), 5, 3), ((13, 29), 2, 8), ((1, 7), 3, 1)])
def test_feature_gradient_from_8_bit_checkpoints(dev, P, shape, pd, vd):
    """Exactly the feature gradient of the rounded values and results; the
    forward and the value gradient as without."""
    f = _randn(shape + (pd,), 10).to(dev).requires_grad_(True)
    v = _randn(shape + (vd,), 11).to(dev).requires_grad_(True)
    g = _randn(shape + (vd,), 12).to(dev)
    P.PLOO.set_checkpoint_precision("8bit")
    assert P.PLOO.get_checkpoint_precision() == "8bit"
    out = P.PermutoLatticeFeatureFunction.apply(f, v)
    gf, gv = torch.autograd.grad(out, [f, v], g)
    R, PLOO = P.rows, P.PLOO
    with torch.no_grad():
        weight, oe, lat = PLOO.lattice_forward(f, v)
        round8 = lambda t: R.unpack8(R.pack8(t.view(-1))).view(t.shape)  # noqa: E731
        gfe = PLOO.feature_grad(lat, f, round8(v), g, weight, round8(out))
        gve = PLOO.lattice_backward(f, g, weight, lat)
    close = lambda a, b: float((a - b).detach().abs().max()) <= 2e-5 * float(b.detach().abs().max()) + 5e-6  # noqa: E731
    assert close(out, oe) and close(gv, gve) and close(gf, gfe)


def test_feature_checkpoints_are_smaller(dev, P):
    f = _randn((256, 256, 5), 13).to(dev).requires_grad_(True)
    v = _randn((256, 256, 8), 14).to(dev)

    def kept(precision):
        P.PLOO.set_checkpoint_precision(precision)
        out = P.PermutoLatticeFeatureFunction.apply(f, v.clone())
        names = [t.numel() * t.element_size() for t in out.grad_fn.saved_tensors]
        return sum(names)
    n = 256 * 256 * 8
    assert kept("fp32") - kept("8bit") == 2 * (4 * n - n - n // 32)


def test_checkpoint_precision_setting(P):
    with pytest.raises(RuntimeError, match="checkpoint precision"):
        P.PLOO.set_checkpoint_precision("int8")
    assert P.PLOO.get_checkpoint_precision() == "fp32"


def test_layer_step_captured_and_replayed(dev, P):
    """Forward and gradients of the layer in a CUDA graph, replayed on new inputs."""
    torch.manual_seed(2)
    m = P.PermutoLatticeLayer(64, 5, 3, act="gelu", dtype=torch.bfloat16, device=dev)
    x = _randn((24, 20, 64), 20, torch.bfloat16).to(dev).requires_grad_(True)
    gy = _randn((24, 20, 64), 21, torch.bfloat16).to(dev)
    leaves = [x, *m.parameters()]

    def step():
        y = m(x)
        return [y, *torch.autograd.grad(y, leaves, gy)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (22, 23):
        with torch.no_grad():
            x.copy_(_randn((24, 20, 64), seed, torch.bfloat16).to(dev))
        graph.replay()
        got_now = [g.detach().float().clone() for g in got]
        for g, e in zip(got_now, step()):
            # the splat's atomics add in another order, and bfloat16 then rounds the other way now and then:
            # at most a step (2^-7) of a value near the largest
            e = e.detach().float()
            assert float((g - e).abs().max()) <= 2.0 ** -7 * float(e.abs().max())


def test_layer_on_another_stream_and_twice_at_once(dev, P):
    torch.manual_seed(3)
    m = P.PermutoLatticeLayer(40, 3, 4, act="silu", device=dev)
    xs = [_randn((17, 23, 40), 30 + i).to(dev) for i in range(2)]
    with torch.no_grad():
        want = [m(x) for x in xs]
        streams = [torch.cuda.Stream() for _ in xs]
        torch.cuda.synchronize()
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(m(x))
        torch.cuda.synchronize()
    for g, e in zip(got, want):
        # lattice sums differ by their order: 1e-5 relative + 5e-6 each, through a product of 4 weights below 1
        assert float((g - e).abs().max()) <= 1e-4
