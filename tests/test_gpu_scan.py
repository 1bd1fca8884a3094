"""The recurrence along lines against its float64 definition: types, lengths from none to
long ones, odd channels, both directions, states carried in and out, and its gradients."""
import numpy as np
import pytest
import torch

import labels_reference as ref
from rows_reference import f64, half_step, worst

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def R():
    from plattice_pytorch_b200 import rows
    return rows


def _inputs(lead, t, c, dtype, seed, gates="sigmoid"):
    g = torch.Generator().manual_seed(seed)
    shape = lead + (t, c)
    x = torch.randn(*shape, generator=g).to(dtype)
    a = torch.randn(*shape, generator=g)
    if gates == "sigmoid":
        a = torch.sigmoid(1.5 * a + 2.0)
        a[torch.rand(lead + (t, 1), generator=g).expand(shape) < 0.02] = 0.0
    elif gates == "ones":
        a = torch.ones(shape)
    elif gates == "signed":
        a = torch.tanh(a)
    return x, a.to(dtype), torch.randn(*lead, c, generator=g), torch.randn(*shape, generator=g).to(dtype), torch.randn(
        *lead, c, generator=g)


SIZES = [((1,), 1, 1), ((), 1, 4096), ((3,), 2, 5), ((2, 3), 15, 8), ((2,), 16, 33), ((5,), 17, 2), ((1,), 100, 7), ((40,), 64, 64),
         ((3,), 129, 130), ((1,), 5000, 3), ((2,), 2049, 16), ((1,), 20011, 2), ((300,), 33, 24), ((0,), 5, 4), ((2,), 0, 6),
         ((1,), 9001, 1), ((3,), 1600, 1), ((2,), 1008, 2), ((5,), 48, 1)]


def _rounded(dtype, value):
    half = half_step(dtype)
    return half * np.abs(value) + ref.tiny(half)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lead,t,c", SIZES)
def test_scan(dev, R, dtype, lead, t, c):
    for k, (blend, reverse, state) in enumerate([(False, False, True), (True, False, False), (False, True, False), (True, True, True)]):
        x, a, s, gy, gl = _inputs(lead, t, c, dtype, 10 + k)
        h, eh, last, el = ref.scan(f64(x), f64(a), f64(s) if state else None, blend, reverse)
        st = s.to(dev) if state else None
        got, glast, states = R.scan(x.to(dev), a.to(dev), st, blend=blend, reverse=reverse, keep=True)
        assert got.dtype == dtype and got.shape == x.shape and glast.shape == s.shape
        assert worst(f64(got), h, eh + _rounded(dtype, h)) <= 1
        assert worst(f64(glast), last, el + 2.0 ** -149) <= 1
        again, last2, none = R.scan(x.to(dev), a.to(dev), st, blend=blend, reverse=reverse)
        assert none is None and torch.equal(again, got) and torch.equal(last2, glast)
        want, bound = ref.scan_backward(f64(gy), f64(x), f64(a), f64(s) if state else None, f64(gl) if state else None, blend, reverse)
        grads = R.scan_backward(gy.to(dev), x.to(dev), a.to(dev), states, gl.to(dev) if state else None, blend=blend, reverse=reverse)
        for name, g, w, b, type_ in zip("x gate state".split(), grads, want, bound, (dtype, dtype, torch.float32)):
            assert g.dtype == type_
            assert worst(f64(g), w, b + _rounded(type_, w)) <= 1, (name, blend, reverse)


@pytest.mark.parametrize("gates", ["ones", "signed"])
@pytest.mark.parametrize("lead,t,c", [((2,), 300, 6), ((1,), 20000, 4)])
def test_other_gates(dev, R, gates, lead, t, c):
    x, a, s, gy, gl = _inputs(lead, t, c, torch.float32, 20, gates)
    h, eh, last, el = ref.scan(f64(x), f64(a), f64(s))
    got, glast, states = R.scan(x.to(dev), a.to(dev), s.to(dev), keep=True)
    assert worst(f64(got), h, eh + _rounded(torch.float32, h)) <= 1 and worst(f64(glast), last, el) <= 1
    want, bound = ref.scan_backward(f64(gy), f64(x), f64(a), f64(s), f64(gl))
    for g, w, b in zip(R.scan_backward(gy.to(dev), x.to(dev), a.to(dev), states, gl.to(dev)), want, bound):
        assert worst(f64(g), w, b + _rounded(torch.float32, w)) <= 1


def test_a_step_at_a_time_is_the_whole(dev, R):
    x, a, s, _, _ = _inputs((3,), 21, 40, torch.bfloat16, 30)
    x, a, s = x.to(dev), a.to(dev), s.to(dev)
    whole, last, _ = R.scan(x, a, s)
    state = s
    for t in range(21):
        h, state, _ = R.scan(x[:, t:t + 1].contiguous(), a[:, t:t + 1].contiguous(), state)
        assert torch.equal(h[:, 0], whole[:, t])
    assert torch.equal(state, last)


def test_a_zero_gate_starts_afresh(dev, R):
    """Two segments behind one another are each its own scan."""
    x, a, _, _, _ = _inputs((1,), 5000, 3, torch.float32, 31)
    a[:, 1777] = 0.0
    h, last, _ = R.scan(x.to(dev), a.to(dev))
    b, last_b, _ = R.scan(x[:, 1777:].contiguous().to(dev), a[:, 1777:].contiguous().to(dev))
    _, eh, _, el = ref.scan(f64(x[:, 1777:]), f64(a[:, 1777:]))
    assert worst(f64(h[:, 1777:]), f64(b), 2 * eh + _rounded(torch.float32, f64(b))) <= 1
    assert worst(f64(last), f64(last_b), 2 * el + 2.0 ** -149) <= 1


def test_what_is_not_finite_stays_behind_a_later_step(dev, R):
    """An infinity or NaN reaches the steps behind it and none before it."""
    for t in (300, 20000):
        for bad in (float("inf"), float("nan")):
            x, a, _, _, _ = _inputs((1,), t, 2, torch.float32, 32)
            a.clamp_(0.5, 0.9)
            x[0, t // 2, 0] = bad
            h, last, _ = R.scan(x.to(dev), a.to(dev))
            assert torch.isfinite(h[0, :, 1]).all() and torch.isfinite(h[0, :t // 2, 0]).all()
            assert not torch.isfinite(h[0, t // 2:, 0]).any() and not torch.isfinite(last[0, 0])


def test_gates_beyond_one_where_nothing_is(dev, R):
    """Products of the gates pass float32 while the state is 0; a gate of 0 and what comes
    behind it are as if they had not."""
    for t in (400, 5000, 30000):
        x, a = torch.zeros(1, t, 3), torch.full((1, t, 3), 2.0)
        half = t // 2 + 5
        a[:, half], a[:, half + 1:] = 0.0, 0.75
        x[:, half:] = torch.randn(1, t - half, 3, generator=torch.Generator().manual_seed(37))
        h, eh, last, el = ref.scan(f64(x), f64(a))
        got, glast, states = R.scan(x.to(dev), a.to(dev), keep=True)
        assert worst(f64(got), h, eh + _rounded(torch.float32, h)) <= 1 and worst(f64(glast), last, el + 2.0 ** -149) <= 1
        g = torch.zeros(1, t, 3)   # and backwards: gradients only before the large gates
        g[:, :20] = 1.0
        a2 = torch.full((1, t, 3), 0.5)
        a2[:, 40:] = 2.0
        _, _, states = R.scan(torch.zeros_like(x).to(dev), a2.to(dev), keep=True)
        want, bound = ref.scan_backward(f64(g), np.zeros(x.shape), f64(a2))
        for v, w, b in zip(R.scan_backward(g.to(dev), torch.zeros_like(x).to(dev), a2.to(dev), states), want, bound):
            assert worst(f64(v), w, b + _rounded(torch.float32, w)) <= 1


def test_unaligned_lines(dev, R):
    for dtype in TYPES:
        x, a, s, gy, gl = (v.to(dev) for v in _inputs((3,), 70, 16, dtype, 33))
        moved = [torch.empty(1 + v.numel(), dtype=dtype, device=dev)[1:].view(v.shape).copy_(v) for v in (x, a, gy)]
        h, last, states = R.scan(x, a, s, keep=True)
        h2, last2, states2 = R.scan(*moved[:2], s, keep=True)
        assert torch.equal(h, h2) and torch.equal(last, last2) and torch.equal(states, states2)
        for g, w in zip(R.scan_backward(moved[2], *moved[:2], states, gl), R.scan_backward(gy, x, a, states, gl)):
            assert torch.equal(g, w)


def test_gradients_are_differences(dev, R):
    """Of sum(h w) + sum(last v) by each input: central differences of the float64
    definition, which is linear in x and state (exact but for rounding) and polynomial
    of degree 1 in each single gate."""
    x, a, s, w, v = _inputs((2,), 19, 3, torch.float32, 34)
    for blend in (False, True):
        def loss(x, a, s):
            h, _, last, _ = ref.scan(x, a, s, blend)
            return (h * f64(w)).sum() + (last * f64(v)).sum()
        base = [f64(t) for t in (x, a, s)]
        _, _, states = R.scan(x.to(dev), a.to(dev), s.to(dev), blend=blend, keep=True)
        grads = R.scan_backward(w.to(dev), x.to(dev), a.to(dev), states, v.to(dev), blend=blend)
        rng = np.random.default_rng(35)
        for k, g in enumerate(grads):
            g = f64(g)
            for _ in range(25):
                at = tuple(rng.integers(0, n) for n in g.shape)
                up, down = [b.copy() for b in base], [b.copy() for b in base]
                up[k][at] += 1e-3
                down[k][at] -= 1e-3
                assert abs((loss(*up) - loss(*down)) / 2e-3 - g[at]) <= 1e-5 * (1 + abs(g[at]))


def test_scan_function(dev, R):
    import plattice_pytorch_b200 as P
    x, a, s, gy, gl = (v.to(dev) for v in _inputs((4,), 50, 12, torch.float32, 36))
    leaves = [v.clone().requires_grad_(True) for v in (x, a, s)]
    h, last = P.RowScanFunction.apply(*leaves, True, False)
    ((h * gy).sum() + (last * gl).sum()).backward()
    _, _, states = R.scan(x, a, s, blend=True, keep=True)
    for leaf, want in zip(leaves, R.scan_backward(gy, x, a, states, gl, blend=True)):
        assert torch.equal(leaf.grad, want)
    leaf = x.clone().requires_grad_(True)   # only the state is used, no state came in
    P.RowScanFunction.apply(leaf, a, None, False, True)[1].sum().backward()
    _, _, states = R.scan(x, a, reverse=True, keep=True)
    assert torch.equal(leaf.grad, R.scan_backward(torch.zeros_like(x), x, a, states, torch.ones_like(gl), reverse=True)[0])
