"""The recurrence along lines whose products of gates leave float32: few lines, which are cut
into pieces, and many, which are not, hold the same recurrence.  The bounds of
labels_reference.scan are relative to the recurrence of the magnitudes, however long."""
import numpy as np
import pytest
import torch

import labels_reference as ref
from rows_reference import U, f64, half_step, worst

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
WHOLE = 28416   # threads from which no line is cut; of 16-bit rows a thread takes two channels


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def R():
    from plattice_pytorch_b200 import rows
    return rows


def _check(dev, R, x, a, s, gy, gl, copies, blend, reverse):
    """Forward and back of [1, t, c], the line `copies` times; gradients too large for the
    type of the rows are left out."""
    def many(v):
        return v.repeat(copies, *[1] * (v.dim() - 1)).to(dev)

    rows = sorted({0, copies // 2, copies - 1})

    def check(name, got, want, bound):
        half, got = half_step(got.dtype), f64(got[rows])
        fits = np.abs(want) < 3e4 if half == half_step(torch.float16) else np.abs(want) < 1e38
        bound = bound + half * np.abs(want) + ref.tiny(half)
        for line in got:
            assert worst(line[fits[0]], want[fits], bound[fits]) <= 1, name
    h, eh, last, el = ref.scan(f64(x), f64(a), f64(s), blend, reverse)
    got, glast, states = R.scan(many(x), many(a), many(s), blend=blend, reverse=reverse, keep=True)
    check("h", got, h, eh)
    check("last", glast, last, el)
    want, bound = ref.scan_backward(f64(gy), f64(x), f64(a), f64(s), f64(gl), blend, reverse)
    grads = R.scan_backward(many(gy), many(x), many(a), states, many(gl), blend=blend, reverse=reverse)
    for name, g, w, b in zip("x gate state".split(), grads, want, bound):
        check(name, g, w, b)


def _scaled(level, dtype, seed):
    """Inputs of the size of h (2^level after a step) and gradients of the size of its inverse."""
    g = torch.Generator().manual_seed(seed)
    size = torch.exp2(level.double())
    x = (0.1 * torch.randn(level.shape, generator=g).double() * size).to(dtype)
    gy = 0.1 * torch.randn(level.shape, generator=g).double() / size
    gy[gy.abs() > torch.finfo(dtype).max] = 0.0
    return x, gy.to(dtype)


@pytest.mark.parametrize("copies", [1, WHOLE // 2 + 1])
@pytest.mark.parametrize("blend,reverse", [(False, False), (True, True)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t", [320, 2500])
def test_products_that_float32_does_not_hold(dev, R, t, dtype, blend, reverse, copies):
    """Gates of 1/2 and 2 take a state of 1 down to 2^-112 and up again, to 2^88 (float16:
    2^14): the products of later gates alone are up to 2^200."""
    low, high = -112, 14 if dtype == torch.float16 else 88
    a, level, way, levels = [], 0, -1, []
    for _ in range(t):
        level += way
        a.append(2.0 ** way)
        levels.append(float(level))
        if level in (low, high):
            way = -way
    a, level = torch.tensor(a), torch.tensor(levels)
    if reverse:
        a, level = a.flip(0), level.flip(0)
    level = level[None, :, None].expand(1, t, 4).contiguous()
    x, gy = _scaled(level, dtype, 1)
    s = torch.tensor([[1.0, -1.0, 0.75, 0.0]])
    gl = torch.exp2(-level[:, 0 if reverse else -1])
    _check(dev, R, x, a[None, :, None].expand(1, t, 4).contiguous().to(dtype), s, gy, gl, copies, blend, reverse)


@pytest.mark.parametrize("copies", [1, WHOLE // 2 + 1])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,spread", [(333, 60.0), (2500, 60.0), (2500, 12.0), (2500, 5.0)])
def test_gates_of_any_size(dev, R, t, spread, dtype, copies):
    """Gates, of either sign, that throw the state about between 2^-spread and 2^spread."""
    g = torch.Generator().manual_seed(2)
    if dtype == torch.float16:
        spread = min(spread, 7.0)
    level = (2 * torch.rand(1, t, 4, generator=g) - 1) * spread
    before = torch.cat([torch.zeros(1, 1, 4), level[:, :-1]], 1)
    a = torch.exp2(level - before) * torch.where(torch.rand(1, t, 4, generator=g) < 0.5, -1.0, 1.0)
    a = a.to(dtype)
    # the rounded gates' own product is where h is: followed, so that rounding does not add up
    for k in range(1, t):
        size = torch.exp2(level[:, k].double()) / torch.exp2(level[:, k - 1].double())
        a[:, k] = (size * torch.sign(a[:, k].double())).to(dtype)
        level[:, k] = level[:, k - 1] + torch.log2(a[:, k].double().abs()).float()
    x, gy = _scaled(level, dtype, 3)
    s = torch.tensor([[1.0, -1.0, 0.75, 0.0]])
    _check(dev, R, x, a, s, gy, torch.exp2(-level[:, -1]), copies, False, False)


def _walk(x, a, s):
    """Step by step in float32: h of every step."""
    h, out = s.copy(), []
    with np.errstate(all="ignore"):
        for t in range(len(x)):
            h = (a[t] * h + x[t]).astype(np.float32)
            out.append(h)
    return np.array(out)


@pytest.mark.parametrize("copies", [1, WHOLE // 2 + 1])
@pytest.mark.parametrize("t", [300, 3000])
def test_what_is_infinite_stays(dev, R, t, copies):
    """An infinite state or input stays one, whatever the product of the gates behind it comes
    to; only a gate of 0 makes it NaN.  A state that is finite and cut off by a gate of 0 leaves
    nothing, however large the gates behind that are."""
    inf = float("inf")
    x, a, s = np.zeros((t, 4), np.float32), np.full((t, 4), 0.25, np.float32), np.zeros(4, np.float32)
    x[10, 0] = inf
    s[1] = -inf
    a[t // 3, 1] = -0.25
    s[2] = inf
    a[t // 2, 2] = 0.0
    s[3] = 1e30
    a[50, 3] = 0.0
    a[51:, 3] = 2.0
    a[60:70, 3] = 1e20   # whose own products are infinite
    want = _walk(x, a, s)
    assert np.isposinf(want[-1, 0]) and np.isposinf(want[-1, 1]) and np.isnan(want[-1, 2]) and want[-1, 3] == 0
    many = lambda v: torch.from_numpy(v)[None].repeat(copies, *[1] * v.ndim).to(dev)  # noqa: E731
    h, last, _ = R.scan(many(x), many(a), many(s))
    for k in (0, copies - 1):
        assert np.array_equal(h[k].cpu().numpy(), want, equal_nan=True)
        assert np.array_equal(last[k].cpu().numpy(), want[-1], equal_nan=True)
    # and backwards: what an infinite gradient behind the last step becomes
    gl = np.array([inf, inf, -inf, 0.0], np.float32)
    b = a[::-1].copy()
    walk = _walk(np.zeros_like(b), b, gl)   # a[t] G[t], from the last step on
    _, _, states = R.scan(many(np.zeros_like(a)), many(a), many(np.zeros(4, np.float32)), keep=True)
    gx, _, gs = R.scan_backward(many(np.zeros_like(a)), many(np.zeros_like(a)), many(a), states, many(gl))
    for k in (0, copies - 1):
        assert np.array_equal(gs[k].cpu().numpy(), walk[-1], equal_nan=True)
        assert np.array_equal(gx[k].flip(0)[1:].cpu().numpy(), walk[:-1], equal_nan=True)


def test_growth_past_float32(dev, R):
    """A state that doubles a step is 2^t, then infinite, in cut lines as in whole ones."""
    t = 1000
    for copies in (1, WHOLE // 2 + 1):
        x, a, s = torch.zeros(copies, t, 4), torch.full((copies, t, 4), 2.0), torch.ones(copies, 4)
        h, last, _ = R.scan(x.to(dev), a.to(dev), s.to(dev))
        want = torch.exp2(torch.arange(1.0, t + 1).double()).float()
        assert torch.isinf(want[-1]) and torch.equal(h[0, :, 1].cpu(), want) and torch.isposinf(last).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [2.0 ** 23, 2.0 ** 25, 1e30])
def test_states_of_any_size(dev, R, size, dtype):
    """Large states that decay, with nothing added, and what is added later.  Beside the
    recurrence's rounding: its own smallest steps (2^-146 for the few that add up), and
    where all maps are tame (states up to 2^24) the factors' smallest steps, each product
    within 2^-150 of a state of 2^23: 250 blocks of 16 steps are 250 maps at most, each in
    two products at most, 500 2^-127 < 2^-118."""
    g = torch.Generator().manual_seed(4)
    for t in (300, 4000):
        a = (0.3 + 0.6 * torch.rand(1, t, 4, generator=g)).to(dtype)
        x = torch.zeros(1, t, 4)
        x[:, t - 20:] = 1e-6
        x = x.to(dtype)
        s = size * torch.tensor([[1.0, -1.0, 0.1, 1e-3]])
        h, eh, last, el = ref.scan(f64(x), f64(a), f64(s))
        got, glast, _ = R.scan(x.to(dev), a.to(dev), s.to(dev))
        half, fits = half_step(dtype), np.abs(h) < torch.finfo(dtype).max
        bound = eh + half * np.abs(h) + ref.tiny(half) + (2.0 ** -118 if size < 2.0 ** 24 else 2.0 ** -146)
        assert worst(f64(got)[fits], h[fits], bound[fits]) <= 1
        assert worst(f64(glast), last, el + 2.0 ** -118) <= 1


def test_one_line_of_many_grows(dev, R):
    """What a line's channel does is of no consequence to the others beside it."""
    g = torch.Generator().manual_seed(5)
    for lines, t, c in ((3, 2000, 70), (2, 900, 6)):
        x, a = torch.randn(lines, t, c, generator=g), torch.sigmoid(torch.randn(lines, t, c, generator=g) + 2)
        s = torch.randn(lines, c, generator=g)
        tame = R.scan(x.to(dev), a.to(dev), s.to(dev))
        a[1, 200:300, 3], a[1, 300:400, 3] = 0.5, 2.0
        a[0, 700, 5] = float("nan")
        x[1, 600, 0] = float("inf")
        s[1, 2] = 1e20
        ok = np.ones((lines, c), bool)
        ok[0, 5] = ok[1, 0] = False
        clean_a, clean_x = a.clone(), x.clone()
        clean_a[0, 700, 5], clean_x[1, 600, 0] = 0.0, 0.0
        h, eh, last, el = ref.scan(f64(clean_x), f64(clean_a), f64(s))
        got, glast, states = R.scan(x.to(dev), a.to(dev), s.to(dev), keep=True)
        where = np.broadcast_to(ok[:, None], h.shape)
        assert worst(f64(got)[where], h[where], (eh + U * np.abs(h))[where]) <= 1
        assert worst(f64(glast)[ok], last[ok], (el + U * np.abs(last))[ok]) <= 1
        assert torch.isnan(got[0, 700:, 5]).all() and torch.isposinf(got[1, 600:, 0]).all()
        assert torch.equal(got[lines - 1, :200, 0], tame[0][lines - 1, :200, 0])
        gy, gl = torch.randn(lines, t, c, generator=g), torch.randn(lines, c, generator=g)
        want, bound = ref.scan_backward(f64(gy), f64(clean_x), f64(clean_a), f64(s), f64(gl))
        grads = R.scan_backward(gy.to(dev), x.to(dev), a.to(dev), states, gl.to(dev))
        for v, w, b in zip(grads, want, bound):
            where = np.broadcast_to(ok if w.ndim == 2 else ok[:, None], w.shape)
            assert worst(f64(v)[where], w[where], (b + U * np.abs(w) + 2.0 ** -149)[where]) <= 1
