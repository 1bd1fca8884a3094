"""Row operators on the GPU against their definitions in float64
(rows_reference.py).

Tolerances.  u = 2^-24 is half a float32 step, h half a step of an output's
type.  A sum of m float32 products in any order is off by at most
m u (1 + small) times the sum of the magnitudes; tensor cores may cut where an
addition rounds, so products count 2 u a term.  An output's rounding adds h
times its value.  The activations' functions are good to 2^-19 of |z| (exp to
2 + 1.2 |z| units of 2^-23 for the |z| <= 8 that occur here)."""
import numpy as np
import pytest
import torch

import rows_reference as ref
from rows_reference import U, f64, half_step, worst

pytestmark = pytest.mark.gpu

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def R():
    from plattice_pytorch_b200 import rows
    return rows


def _randn(shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


# ---------------------------------------------------------------- 8-bit rows

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,c", [(1, 1), (3, 8), (5, 31), (2, 32), (7, 33), (129, 50), (65, 256), (9, 1000)])
def test_pack8_bits(dev, R, rows, c, dtype):
    x = _randn((rows, c), 1, torch.float32) * torch.exp(2 * _randn((rows, 1), 2))
    x[0, 0] = 0.0
    x = x.to(DTYPES[dtype])
    r = R.pack8(x.to(dev))
    q, s = ref.pack8(f64(x))
    assert np.array_equal(r.scale.cpu().numpy(), s)
    got = r.q.cpu().numpy()
    assert np.array_equal(got, q)
    want = ref.unpack8(q, s, c)
    for out in (torch.float32, torch.bfloat16):   # exact in both
        assert np.array_equal(f64(R.unpack8(r, out)), want)
    y = f64(R.unpack8(r, torch.float16))
    assert np.array_equal(y, want.clip(-65504, 65504).astype(np.float16).astype(np.float64))


def test_pack8_ties_limits_and_scale_edges(dev, R):
    e = ref.E4M3[:127]
    mid = np.concatenate([e, (e[1:] + e[:-1]) / 2, -(e[1:] + e[:-1]) / 2])
    x = np.zeros((mid.size, 32))
    x[:, 0], x[:, 1] = 448.0, mid               # scale 1: every code and every tie
    edge = np.array([448.0, 448.0 * (1 + 2.0 ** -7), 224.0, 224.5, 2.0 ** -126, 2.0 ** -140, 3e38, 2.0 ** 127, 0.0])
    y = np.zeros((edge.size, 32))
    y[:, 5] = edge
    x = torch.from_numpy(np.concatenate([x, y])).float()
    r = R.pack8(x.to(dev))
    q, s = ref.pack8(f64(x))
    assert np.array_equal(r.scale.cpu().numpy(), s)
    assert np.array_equal(r.q.cpu().numpy(), q)
    assert np.array_equal(f64(R.unpack8(r)), ref.unpack8(q, s, 32))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_pack8_not_finite(dev, R, bad):
    x = _randn((4, 64), 3)
    x[1, 7] = bad
    x[2, 32:] = bad
    y = R.unpack8(R.pack8(x.to(dev))).cpu()
    clean = torch.where(torch.isfinite(x), x, torch.zeros(()))
    want = R.unpack8(R.pack8(clean.to(dev))).cpu()
    assert torch.equal(torch.isnan(y), ~torch.isfinite(x))
    assert torch.equal(y[torch.isfinite(x)], want[torch.isfinite(x)])


# ---------------------------------------------------------------- the norm

NORM_SHAPES = [(1, 1), (3, 8), (377, 50), (5, 64), (33, 100), (130, 256), (17, 512), (9, 1000), (3, 1024), (5, 1032),
               (3, 2049), (2, 4096), (2, 5000), (1, 16384)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,c", NORM_SHAPES)
def test_rms_norm(dev, R, rows, c, residual, dtype):
    t = DTYPES[dtype]
    x, r = _randn((rows, c), 4, t), _randn((rows, c), 5, t) if residual else None
    gain = 1 + 0.2 * _randn((c,), 6)
    rd = None if r is None else r.to(dev)
    y, h, rstd = R.rms_norm(x.to(dev), gain.to(dev), rd)
    ye, he, re_ = ref.rms_norm(f64(x), f64(gain), None if r is None else f64(r))
    k = 64 * U   # chains of at most 32 terms and 10 levels, the division, rsqrt (2 units), two products
    assert worst(f64(rstd), re_, k * re_) <= 1
    assert worst(f64(y), ye, (half_step(t) + k) * np.abs(ye) + 1e-30 + (t is torch.float16) * 2.0 ** -25) <= 1
    if residual:
        assert worst(f64(h), he, half_step(t) * np.abs(he) + (t is torch.float16) * 2.0 ** -25 + 1e-30) <= 1
    # in 8 bits: half a step of the code on top
    y8, h8, rstd8 = R.rms_norm(x.to(dev), gain.to(dev), rd, pack=True)
    assert torch.equal(rstd8, rstd) and torch.equal(h8, h)
    unit = 2.0 ** (y8.scale.cpu().numpy().astype(np.float64) - 127)
    unit = np.repeat(unit, 32, 1)[:, :c]
    assert worst(f64(R.unpack8(y8)), ye, (2.0 ** -4 + 2 * k) * np.abs(ye) + 2.0 ** -10 * unit) <= 1
    assert not y8.q[:, c:].any()
    amax = np.abs(np.pad(ye, ((0, 0), (0, -c % 32)))).reshape(rows, -1, 32).max(-1)
    s = y8.scale.cpu().numpy().astype(np.float64) - 127
    assert (amax <= 448 * 2.0 ** s * (1 + 2 * k)).all() and (amax * (1 + 2 * k) >= 224 * 2.0 ** s).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("grad_h", [False, True])
@pytest.mark.parametrize("rows,c", NORM_SHAPES)
def test_rms_norm_backward(dev, R, rows, c, grad_h, dtype):
    t = DTYPES[dtype]
    h, gy = _randn((rows, c), 7, t), _randn((rows, c), 8, t)
    gh = _randn((rows, c), 9, t) if grad_h else None
    gain = 1 + 0.2 * _randn((c,), 10)
    rstd = (1 / torch.sqrt((h.double() ** 2).mean(-1) + 1e-6)).float()
    gx, gg = R.rms_norm_backward(gy.to(dev), h.to(dev), rstd.to(dev), gain.to(dev), None if gh is None else gh.to(dev))
    a = [f64(v) for v in (gy, h, rstd, gain)]
    xe, ge = ref.rms_norm_backward(*a, None if gh is None else f64(gh))
    n = a[1] * a[2][:, None]
    gn = np.abs(a[0] * a[3])
    size = a[2][:, None] * (gn + np.abs(n) * (gn * np.abs(n)).mean(-1, keepdims=True))
    assert worst(f64(gx), xe, half_step(t) * np.abs(xe) + 64 * U * size + (0 if gh is None else 2 * U * np.abs(f64(gh)))
                 + (t is torch.float16) * 2.0 ** -25 + 1e-30) <= 1
    assert worst(f64(gg), ge, (rows + 8) * U * np.abs(a[0] * n).sum(0) + 1e-30) <= 1


def test_rms_norm_gradient_against_differences(dev, R):
    rows, c = 5, 37
    x, res = _randn((rows, c), 11), _randn((rows, c), 12)
    gain, gy, gh = 1 + 0.2 * _randn((c,), 13), _randn((rows, c), 14), _randn((rows, c), 15)
    _, h, rstd = R.rms_norm(x.to(dev), gain.to(dev), res.to(dev))
    gx, gg = R.rms_norm_backward(gy.to(dev), h, rstd, gain.to(dev), gh.to(dev))

    def loss(x_, g_):
        y, h_, _ = ref.rms_norm(x_, g_, f64(res))
        return (y * f64(gy)).sum() + (h_ * f64(gh)).sum()
    d = 1e-5
    for name, grad, size in (("x", f64(gx), (rows, c)), ("gain", f64(gg), (c,))):
        for seed in range(3):
            v = np.random.default_rng(seed).standard_normal(size)
            p = [f64(x), f64(gain)]
            i = 0 if name == "x" else 1
            hi, lo = list(p), list(p)
            hi[i], lo[i] = p[i] + d * v, p[i] - d * v
            slope = (loss(*hi) - loss(*lo)) / (2 * d)
            # differences: d^2 times a third derivative of the order of the terms; gradient: float32
            assert abs(slope - (grad * v).sum()) <= 1e-5 * np.abs(grad * v).sum()


@pytest.mark.parametrize("param", DTYPES)
def test_rms_norm_gain_types(dev, R, param):
    x, gy = _randn((19, 40), 16).to(dev), _randn((19, 40), 17).to(dev)
    gain = (1 + 0.2 * _randn((40,), 18)).to(DTYPES[param])
    y, h, rstd = R.rms_norm(x, gain.to(dev))
    ye, _, _ = ref.rms_norm(f64(x), f64(gain))
    assert worst(f64(y), ye, 65 * U * np.abs(ye)) <= 1
    _, gg = R.rms_norm_backward(gy, h, rstd, gain.to(dev))
    assert gg.dtype == DTYPES[param]
    n = f64(h) * f64(rstd)[:, None]
    _, ge = ref.rms_norm_backward(f64(gy), f64(h), f64(rstd), f64(gain))
    assert worst(f64(gg), ge, half_step(gg.dtype) * np.abs(ge) + 27 * U * np.abs(f64(gy) * n).sum(0)) <= 1


# ---------------------------------------------------------------- the linear map

LINEAR_SHAPES = [(1, 1, 1), (1, 64, 24), (3, 7, 2), (377, 50, 24), (130, 64, 8), (129, 130, 200), (257, 96, 33),
                 (64, 512, 72), (300, 33, 257), (16, 1024, 520), (40, 264, 1), (512, 1, 16), (1000, 256, 320)]


def _linear_input(rows, k, n, dtype, x8, R, dev):
    x = _randn((rows, k), 20)
    w = _randn((n, k), 21, dtype, 1 / np.sqrt(k))
    if x8:
        xin = R.pack8(x.to(dev))
        return xin, f64(R.unpack8(xin)), w
    x = x.to(dtype)
    return x.to(dev), f64(x), w


KINDS = [("fp32", False), ("bf16", False), ("fp16", False), ("fp32", True), ("bf16", True)]


def _forward_tolerance(xe, we, b, z, y, k, out):
    size = np.abs(xe) @ np.abs(we).T + (0 if b is None else np.abs(b))
    return 1.13 * 2 * U * (k + 8) * size + 2.0 ** -19 * np.abs(z) + half_step(out) * np.abs(y) \
        + (out is torch.float16) * 2.0 ** -25 + 1e-30


@pytest.mark.parametrize("dtype,x8", KINDS)
@pytest.mark.parametrize("rows,k,n", LINEAR_SHAPES)
@pytest.mark.parametrize("act,residual,keep,out32", [("none", False, None, False), ("gelu", True, "8bit", False),
                                                     ("silu", False, "full", True), ("relu", True, None, True)])
def test_linear(dev, R, rows, k, n, dtype, x8, act, residual, keep, out32):
    t = DTYPES[dtype]
    out = torch.float32 if out32 else t
    x, xe, w = _linear_input(rows, k, n, t, x8, R, dev)
    b = None if act == "none" else 0.3 * _randn((n,), 22)
    res = _randn((rows, n), 23, out) if residual else None
    y, z = R.linear(x, w.to(dev), None if b is None else b.to(dev), act=act,
                    residual=None if res is None else res.to(dev), keep=keep, out_dtype=out)
    we, be = f64(w), None if b is None else f64(b)
    ye, ze = ref.linear(xe, we, be, act, None if res is None else f64(res))
    tol = _forward_tolerance(xe, we, be, ze, ye, k, out)
    assert y.dtype == out and worst(f64(y), ye, tol + (0 if res is None else 2 * U * np.abs(f64(res)))) <= 1
    if keep == "full":
        assert z.dtype == out and worst(f64(z), ze, _forward_tolerance(xe, we, be, ze * 0, ze, k, out)) <= 1
    elif keep == "8bit":
        unit = np.repeat(2.0 ** (z.scale.cpu().numpy().astype(np.float64) - 127), 32, 1)[:, :n]
        raw = 2 * U * (k + 8) * (np.abs(xe) @ np.abs(we).T + 1)
        assert worst(f64(R.unpack8(z)), ze, 2.0 ** -4 * np.abs(ze) + 2.0 ** -10 * unit + 2 * raw) <= 1
        assert not z.q[:, n:].any()
    else:
        assert z is None


@pytest.mark.parametrize("dtype,x8", KINDS)
@pytest.mark.parametrize("rows,k,n,split", [(1, 64, 24, 16), (377, 50, 8, 5), (1000, 64, 24, 16), (257, 40, 2, 1),
                                            (130, 96, 150, 70), (33, 16, 300, 299)])
def test_linear_split(dev, R, rows, k, n, split, dtype, x8):
    t = DTYPES[dtype]
    x, xe, w = _linear_input(rows, k, n, t, x8, R, dev)
    b = _randn((n,), 22, t)
    (f, v), z = R.linear(x, w.to(dev), b.to(dev), split=split, out_dtype=torch.float32)
    assert z is None and f.shape == (rows, split) and v.shape == (rows, n - split)
    assert f.is_contiguous() and v.is_contiguous()
    ye, ze = ref.linear(xe, f64(w), f64(b))
    tol = _forward_tolerance(xe, f64(w), f64(b), ze * 0, ye, k, torch.float32)
    assert worst(np.concatenate([f64(f), f64(v)], 1), ye, tol) <= 1
    # backward of the pair
    gf, gv = _randn((rows, split), 24), _randn((rows, n - split), 25)
    got = R.linear_backward((gf.to(dev), gv.to(dev)), x, w.to(dev), bias_dtype=torch.float32)
    _check_gradients(got, np.concatenate([f64(gf), f64(gv)], 1), xe, f64(w), None, "none", t, torch.float32)


def _check_gradients(got, gy, xe, we, ze, act, t, out):
    gx, gw, gb = got
    xr, wr, br, gz = ref.linear_backward(gy, xe, we, ze, act)
    rows, n = gz.shape
    # gz: its rounding to the operands' type, and the slope's functions
    rel = (0 if t is torch.float32 or (act == "none" and out is t) else half_step(t)) \
        + (2.0 ** -18 if act in ("gelu", "silu") else 0)
    slack = 2.0 ** -18 * np.abs(gy) * (act in ("gelu", "silu"))
    tiny = (t is torch.float16) * 2.0 ** -25 + 1e-30
    az = np.abs(gz) * (rel + 2 * U) + slack + tiny
    assert worst(f64(gx), xr, az @ np.abs(we) + 2 * U * (n + 8) * (np.abs(gz) @ np.abs(we))
                 + half_step(t) * np.abs(xr) + tiny) <= 1
    assert worst(f64(gw), wr, az.T @ np.abs(xe) + 2 * U * (rows + 8) * (np.abs(gz).T @ np.abs(xe))
                 + half_step(t) * np.abs(wr) + tiny) <= 1
    az = np.abs(gz) * (2.0 ** -18 if act in ("gelu", "silu") else U) + slack
    assert worst(f64(gb), br, az.sum(0) + (rows + 8) * U * np.abs(gz).sum(0) + half_step(gb.dtype) * np.abs(br) + tiny) <= 1


@pytest.mark.parametrize("dtype,x8", KINDS)
@pytest.mark.parametrize("rows,k,n", LINEAR_SHAPES)
@pytest.mark.parametrize("act,keep,out32", [("none", None, False), ("gelu", "8bit", False), ("silu", "full", True),
                                            ("relu", "8bit", True)])
def test_linear_backward(dev, R, rows, k, n, dtype, x8, act, keep, out32):
    t = DTYPES[dtype]
    out = torch.float32 if out32 else t
    x, xe, w = _linear_input(rows, k, n, t, x8, R, dev)
    gy = _randn((rows, n), 26, out)
    z, ze = None, None
    if act != "none":
        zt = _randn((rows, n), 27, out).to(dev)
        z = R.pack8(zt) if keep == "8bit" else zt
        ze = f64(R.unpack8(z)) if keep == "8bit" else f64(zt)
    got = R.linear_backward(gy.to(dev), x, w.to(dev), z, act=act, bias_dtype=torch.float32)
    assert got[0].dtype == t and got[1].dtype == t and got[2].dtype == torch.float32
    _check_gradients(got, f64(gy), xe, f64(w), ze, act, t, out)


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_linear_gradient_against_differences(dev, R, act):
    rows, k, n = 9, 21, 13
    x, w, b = _randn((rows, k), 28), _randn((n, k), 29, scale=k ** -0.5), 0.3 * _randn((n,), 30)
    gy = _randn((rows, n), 31)
    _, z = R.linear(x.to(dev), w.to(dev), b.to(dev), act=act, keep=None if act == "none" else "full")
    got = R.linear_backward(gy.to(dev), x.to(dev), w.to(dev), z, act=act)
    p = [f64(x), f64(w), f64(b)]
    d = 1e-6
    for i, grad in enumerate(f64(g) for g in got):
        for seed in range(3):
            v = np.random.default_rng(seed).standard_normal(p[i].shape)
            hi, lo = list(p), list(p)
            hi[i], lo[i] = p[i] + d * v, p[i] - d * v
            slope = ((ref.linear(*hi, act)[0] - ref.linear(*lo, act)[0]) * f64(gy)).sum() / (2 * d)
            # float32 gradients (about 50 terms); a relu's kink within d of a z does not occur for these seeds
            assert abs(slope - (grad * v).sum()) <= 2e-5 * np.abs(grad * v).sum()


def test_linear_backward_need(dev, R):
    x, w, gy = _randn((50, 24), 32).to(dev), _randn((16, 24), 33).to(dev), _randn((50, 16), 34).to(dev)
    full = R.linear_backward(gy, x, w)
    for i in range(3):
        need = tuple(j == i for j in range(3))
        got = R.linear_backward(gy, x, w, need=need)
        assert [g is not None for g in got] == list(need)
        assert torch.equal(got[i], full[i])


# ---------------------------------------------------------------- every operator

def _calls(R, dev, rows=70, k=48, n=40, dtype=torch.bfloat16):
    x, res = _randn((rows, k), 40, dtype).to(dev), _randn((rows, k), 41, dtype).to(dev)
    gain = (1 + 0.2 * _randn((k,), 42)).to(dev)
    w, b = _randn((n, k), 43, dtype, k ** -0.5).to(dev), _randn((n,), 44).to(dev)
    gy, gk = _randn((rows, n), 45, dtype).to(dev), _randn((rows, k), 46, dtype).to(dev)

    def run():
        y8, h, rstd = R.rms_norm(x, gain, res, pack=True)
        y, z = R.linear(y8, w, b, act="gelu", keep="8bit")
        gx, gw, gb = R.linear_backward(gy, y8, w, z, act="gelu")
        gh, gg = R.rms_norm_backward(gx, h, rstd, gain, gk)
        return [R.unpack8(y8), h, rstd, y, R.unpack8(z), gx, gw, gb, gh, gg]
    return run


@pytest.mark.parametrize("rows", [70, 1])
def test_repeat_stream_and_graph_give_the_same_bits(dev, R, rows):
    run = _calls(R, dev, rows)
    want = run()
    for g, e in zip(run(), want):
        assert torch.equal(g, e)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run()
    torch.cuda.current_stream().wait_stream(s)
    for g, e in zip(got, want):
        assert torch.equal(g, e)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other):
        got2 = run()
    for _ in range(2):
        for g in got + got2:
            g.zero_()
        graph.replay()
        other.replay()
        for g, h, e in zip(got, got2, want):
            assert torch.equal(g, e) and torch.equal(h, e)


def test_storage_that_is_not_aligned(dev, R):
    """Contiguous views that start one element into their storage."""
    def shifted(t):
        s = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        v = s[1:].view(t.shape)
        v.copy_(t)
        return v
    for dtype in DTYPES.values():
        rows, k, n = 37, 64, 48
        x, w = _randn((rows, k), 50, dtype).to(dev), _randn((n, k), 51, dtype, k ** -0.5).to(dev)
        gain, res = _randn((k,), 52, dtype).to(dev), _randn((rows, k), 53, dtype).to(dev)
        gy, rn = _randn((rows, n), 54, dtype).to(dev), _randn((rows, n), 55, dtype).to(dev)
        assert torch.equal(R.pack8(x).q, R.pack8(shifted(x)).q)
        # the lanes of an unaligned row hold other channels, so its sums are added in another order.  Each
        # result is within its bound of the definition (the tests above: (h + 64 u) |y|, 64 u rstd, and
        # h |g| + 64 u size for a gradient), so two of them differ by at most twice that
        close = lambda a, b, t: worst(f64(a), f64(b), t) <= 1  # noqa: E731
        hs = half_step(dtype)
        y, h, rstd = R.rms_norm(x, gain, res)
        ys, h2, rs = R.rms_norm(shifted(x), shifted(gain), shifted(res))
        tiny = 2.0 ** -24 if dtype is torch.float16 else 1e-30
        assert torch.equal(h, h2)
        assert close(y, ys, 2.01 * (hs + 64 * U) * np.abs(f64(y)) + tiny) and close(rs, rstd, 128 * U * f64(rstd))
        gx, gg = R.rms_norm_backward(x, h, rstd, gain)
        gx2, gg2 = R.rms_norm_backward(shifted(x), shifted(h), shifted(rstd), shifted(gain))
        nn, gn = np.abs(f64(h) * f64(rstd)[:, None]), np.abs(f64(x) * f64(gain))
        size = f64(rstd)[:, None] * (gn + nn * (gn * nn).mean(-1, keepdims=True))
        assert close(gx, gx2, 2.01 * hs * np.abs(f64(gx)) + 128 * U * size + tiny)
        assert close(gg, gg2, 2.01 * hs * np.abs(f64(gg)) + 2 * (rows + 8) * U * np.abs(f64(x) * nn).sum(0) + tiny)
        ye, _ = R.linear(x, w, residual=rn)
        yg, _ = R.linear(shifted(x), shifted(w), residual=shifted(rn))
        assert torch.equal(ye, yg)
        for a, b in zip(R.linear_backward(gy, x, w), R.linear_backward(shifted(gy), shifted(x), shifted(w))):
            assert torch.equal(a, b)


@pytest.mark.parametrize("shape", [(0, 16), (3, 0, 16)])
def test_no_rows(dev, R, shape):
    x, w, gain = torch.empty(shape, device=dev), torch.randn(5, 16, device=dev), torch.randn(16, device=dev)
    r = R.pack8(x)
    assert R.unpack8(r).shape == shape
    y, h, rstd = R.rms_norm(x, gain)
    assert y.shape == shape and rstd.shape == shape[:-1]
    gx, gg = R.rms_norm_backward(y, h, rstd, gain)
    assert gx.shape == shape and not gg.any()
    z, _ = R.linear(x, w)
    assert z.shape == shape[:-1] + (5,)
    gx, gw, gb = R.linear_backward(z, r, w)
    assert gx.shape == shape and not gw.any() and not gb.any()


def test_leading_shape(dev, R):
    x = _randn((3, 5, 7, 24), 60).to(dev)
    w, gain = _randn((10, 24), 61).to(dev), _randn((24,), 62).to(dev)
    flat = x.view(-1, 24)
    assert torch.equal(R.unpack8(R.pack8(x)).view(-1, 24), R.unpack8(R.pack8(flat)))
    y, h, rstd = R.rms_norm(x, gain)
    assert h is x and y.shape == x.shape and rstd.shape == x.shape[:-1]
    assert torch.equal(R.linear(R.pack8(x), w)[0].view(-1, 10), R.linear(R.pack8(flat), w)[0])


def test_rows_of_not_finite_values_stay_in_their_rows(dev, R):
    for dtype in DTYPES.values():
        x, w = _randn((140, 64), 63, dtype), _randn((40, 64), 64, dtype, 0.125).to(dev)
        clean, _ = R.linear(x.to(dev), w)
        x[5, 3], x[130, 60] = float("nan"), float("inf")
        y, _ = R.linear(x.to(dev), w)
        bad = torch.zeros(140, dtype=torch.bool)
        bad[5] = bad[130] = True
        assert torch.equal(y.cpu()[~bad], clean.cpu()[~bad])
        assert not torch.isfinite(y[5]).any() and not torch.isfinite(y[130]).any()


def test_python_and_extension_calls_agree(dev, R, monkeypatch):
    """The calls through the torch extension and through ctypes give the same
    bits, shapes and types."""
    def collect():
        out = list(_calls(R, dev)()) + list(_calls(R, dev, 5, 40, 72, torch.float32)())
        x, w, b = _randn((9, 33), 70).to(dev), _randn((12, 33), 71).to(dev), _randn((12,), 72).to(dev)
        (f, v), z = R.linear(x, w, b, split=5)
        out += [f, v, *R.linear_backward((f, v), x, w)]
        out += [R.linear(x.bfloat16(), w.bfloat16(), act="relu", keep="full", out_dtype=torch.float32)[i] for i in (0, 1)]
        y, h, rstd = R.rms_norm(x, x[0].contiguous())
        out += [y, h, rstd, *R.rms_norm_backward(y, h, rstd, x[0].contiguous())]
        return out
    fast = collect()
    assert R._cpp() is not None
    monkeypatch.setattr(R, "_EXT", None)
    slow = collect()
    for a, b in zip(fast, slow):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_refusals_on_the_device(dev, R):
    x, w, g = torch.zeros(4, 8, device=dev), torch.zeros(3, 8, device=dev), torch.zeros(8, device=dev)
    for call, text in [
            (lambda: R.pack8(x.double()), "float32, bfloat16 or float16"),
            (lambda: R.pack8(x.t()), "contiguous"),
            (lambda: R.pack8(x.cpu()), "CUDA"),
            (lambda: R.rms_norm(x, g.cpu()), "CUDA"),
            (lambda: R.rms_norm(x, g, x.half()), "residual"),
            (lambda: R.rms_norm_backward(x, x, g, g), "rstd"),
            (lambda: R.linear(x, w.half()), "same type"),
            (lambda: R.linear(x, w, residual=x), "residual"),
            (lambda: R.linear(x, w, split=1, act="relu"), "split"),
            (lambda: R.linear(R.pack8(x), w.half()), "8-bit"),
            (lambda: R.linear(x, w, act="tanh"), "act"),
            (lambda: R.linear_backward(x, x, w), "grad_y"),
            (lambda: R.linear_backward(torch.zeros(4, 3, device=dev), x, w, act="gelu"), "z is needed"),
            (lambda: R.linear_backward(torch.zeros(4, 3, device=dev), x, w, R.pack8(x), act="gelu"), "z must be"),
            (lambda: R.linear_backward(torch.zeros(4, 3, device=dev), None, w), "x is needed")]:
        with pytest.raises(RuntimeError, match=text):
            call()
    got = R.linear_backward(torch.ones(4, 3, device=dev), None, w, need=(True, False, True))
    assert got[0].shape == (4, 8) and got[1] is None and got[2].tolist() == [4.0, 4.0, 4.0]


# Several tiles along each side, more tiles than SMs, bands of columns (n over
# 18 tiles of 256), parts of the sum, depths that end inside a slice.
BIG_SHAPES = [(300, 200, 5200), (20000, 72, 264), (5000, 1100, 96), (130, 2100, 1000)]


@pytest.mark.parametrize("dtype,x8", KINDS)
@pytest.mark.parametrize("rows,k,n", BIG_SHAPES)
def test_linear_many_tiles(dev, R, rows, k, n, dtype, x8):
    t = DTYPES[dtype]
    x, xe, w = _linear_input(rows, k, n, t, x8, R, dev)
    b, res = 0.3 * _randn((n,), 22), _randn((rows, n), 23, t)
    y, z = R.linear(x, w.to(dev), b.to(dev), act="silu", residual=res.to(dev), keep="8bit")
    ye, ze = ref.linear(xe, f64(w), f64(b), "silu", f64(res))
    tol = _forward_tolerance(xe, f64(w), f64(b), ze, ye, k, t)
    assert worst(f64(y), ye, tol + 2 * U * np.abs(f64(res))) <= 1
    plain, _ = R.linear(x, w.to(dev), out_dtype=torch.float32)
    pe, _ = ref.linear(xe, f64(w))
    assert worst(f64(plain), pe, _forward_tolerance(xe, f64(w), None, pe * 0, pe, k, torch.float32)) <= 1
    gy = _randn((rows, n), 26, t)
    got = R.linear_backward(gy.to(dev), x, w.to(dev), z, act="silu", bias_dtype=torch.float32)
    _check_gradients(got, f64(gy), xe, f64(w), f64(R.unpack8(z)), "silu", t, t)


@pytest.mark.parametrize("n,k", [(8, 200), (24, 130), (32, 64), (17, 1000)])
@pytest.mark.parametrize("dtype,x8", KINDS)
def test_linear_narrow_many_rows(dev, R, n, k, dtype, x8):
    """More blocks of rows than warps, several slices of channels."""
    t, rows = DTYPES[dtype], 30011
    x, xe, w = _linear_input(rows, k, n, t, x8, R, dev)
    y, z = R.linear(x, w.to(dev), act="gelu", keep="8bit")
    ye, ze = ref.linear(xe, f64(w), None, "gelu")
    assert worst(f64(y), ye, _forward_tolerance(xe, f64(w), None, ze, ye, k, t)) <= 1
    gy = _randn((rows, n), 26, t)
    got = R.linear_backward(gy.to(dev), x, w.to(dev), z, act="gelu", bias_dtype=torch.float32)
    _check_gradients(got, f64(gy), xe, f64(w), f64(R.unpack8(z)), "gelu", t, t)


def test_offsets_beyond_32_bits(dev, R):
    """A tensor of more than 2^31 values: the last rows come out as they do alone."""
    if torch.cuda.mem_get_info(dev)[0] < 24 << 30:
        pytest.skip("needs 24 GB of free device memory")
    rows, c = 1 << 20, 2112
    assert rows * c > 1 << 31
    tail = _randn((40, c), 80, torch.bfloat16).to(dev)
    x = torch.zeros(rows, c, dtype=torch.bfloat16, device=dev)
    x[-40:] = tail
    r = R.pack8(x)
    alone = R.pack8(tail)
    assert torch.equal(r.q[-40:], alone.q) and torch.equal(r.scale[-40:], alone.scale) and not r.q[:-40].any()
    assert torch.equal(R.unpack8(r, torch.bfloat16)[-40:], R.unpack8(alone, torch.bfloat16))
    gain = _randn((c,), 81).to(dev)
    y, _, rstd = R.rms_norm(x, gain)
    ya, _, ra = R.rms_norm(tail, gain)
    assert torch.equal(y[-40:], ya) and torch.equal(rstd[-40:], ra)
    del y, rstd
    w, gy = _randn((8, c), 82, torch.bfloat16, c ** -0.5).to(dev), torch.zeros(rows, 8, dtype=torch.bfloat16, device=dev)
    gy[-40:] = _randn((40, 8), 83, torch.bfloat16).to(dev)
    out, _ = R.linear(r, w, out_dtype=torch.float32)
    xe = f64(R.unpack8(alone))
    oe = xe @ f64(w).T
    assert worst(f64(out[-40:]), oe, _forward_tolerance(xe, f64(w), None, oe * 0, oe, c, torch.float32)) <= 1
    for src, se in ((r, xe), (x, f64(tail))):
        got = R.linear_backward(gy, src, w, bias_dtype=torch.float32)
        assert not got[0][:-40].any()
        _check_gradients((got[0][-40:], got[1], got[2]), f64(gy[-40:]), se, f64(w), None, "none", torch.bfloat16,
                         torch.bfloat16)
    w = _randn((40, c), 84, torch.bfloat16, c ** -0.5).to(dev)
    out, _ = R.linear(x, w)
    oe = f64(tail) @ f64(w).T
    assert worst(f64(out[-40:]), oe, _forward_tolerance(f64(tail), f64(w), None, oe * 0, oe, c, torch.bfloat16)) <= 1


@pytest.mark.parametrize("rows,k,n", [(300, 5000, 24), (140, 9000, 8), (3, 5000, 24), (1, 264, 520), (2, 100, 40), (9, 72, 40),
                                      (600, 640, 700)])
@pytest.mark.parametrize("dtype,x8", KINDS)
def test_linear_deep_sums_and_few_rows(dev, R, rows, k, n, dtype, x8):
    """Few output channels over more input channels than shared memory holds
    weights of, few rows, sums deeper than a chunk on both sides."""
    t = DTYPES[dtype]
    x, xe, w = _linear_input(rows, k, n, t, x8, R, dev)
    b = 0.3 * _randn((n,), 22)
    for out, act, keep in ((torch.float32, "none", None), (t, "relu", "8bit"), (torch.float32, "silu", "full")):
        y, z = R.linear(x, w.to(dev), b.to(dev), act=act, out_dtype=out, keep=keep)
        ye, ze = ref.linear(xe, f64(w), f64(b), act)
        assert worst(f64(y), ye, _forward_tolerance(xe, f64(w), f64(b), ze, ye, k, out)) <= 1
        gy = _randn((rows, n), 26, out)
        got = R.linear_backward(gy.to(dev), x, w.to(dev), z, act=act, bias_dtype=torch.float32)
        zk = None if z is None else f64(R.unpack8(z)) if keep == "8bit" else f64(z)
        _check_gradients(got, f64(gy), xe, f64(w), zk, act, t, out)


@pytest.mark.parametrize("k,n", [(1024, 40), (4096, 72), (2048, 24)])
def test_float32_sums_stay_float32(dev, R, k, n):
    """A deep sum of float32 products is as near as float32 additions in
    blocks are: u sqrt(m) of the sum of squares' root for random signs, m the
    longest chain of additions (here at most k / 16), where a chain that cuts
    instead of rounding would be off by u m."""
    rows = 512
    x, w = _randn((rows, k), 90), _randn((n, k), 91, scale=k ** -0.5)
    y, _ = R.linear(x.to(dev), w.to(dev))
    ye = f64(x) @ f64(w).T
    rel = np.linalg.norm(f64(y) - ye) / np.linalg.norm(ye)
    assert rel <= 2 * U * np.sqrt(k / 16) + 4 * U
    gy = _randn((8192, n), 92)
    xl = _randn((8192, 64), 93)
    got = R.linear_backward(gy.to(dev), xl.to(dev), _randn((n, 64), 94).to(dev))
    we = f64(gy).T @ f64(xl)
    assert np.linalg.norm(f64(got[1]) - we) / np.linalg.norm(we) <= 2 * U * np.sqrt(8192 / 16) + 4 * U


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("dtype,out32", [("fp32", True), ("bf16", False), ("bf16", True)])
def test_linear_backward_many_kept_values(dev, R, dtype, out32, act):
    """Millions of kept 8-bit values, their blocks' scales from 2^-24 to 2^8:
    the slopes of some come from a table, of the others from the function."""
    t = DTYPES[dtype]
    out = torch.float32 if out32 else t
    rows, k, n = 20000, 40, 256
    x, xe, w = _linear_input(rows, k, n, t, True, R, dev)
    z = _randn((rows, n), 98) * 2.0 ** torch.randint(-22, 10, (rows, n // 32), generator=torch.Generator().manual_seed(99)
                                                     ).repeat_interleave(32, 1)
    z8 = R.pack8(z.clamp(-100, 100).to(dev))
    gy = _randn((rows, n), 100, out)
    got = R.linear_backward(gy.to(dev), x, w.to(dev), z8, act=act, bias_dtype=torch.float32)
    _check_gradients(got, f64(gy), xe, f64(w), f64(R.unpack8(z8)), act, t, out)


@pytest.mark.parametrize("dtype,x8", [("fp32", False), ("bf16", True)])
def test_linear_backward_of_millions_of_channels(dev, R, dtype, x8):
    """More input channels than a grid has room for slices of 64 of."""
    t, rows, k, n = DTYPES[dtype], 3, 65535 * 64 + 40, 2
    x, xe, w = _linear_input(rows, k, n, t, x8, R, dev)
    gy = _randn((rows, n), 97, t)
    got = R.linear_backward(gy.to(dev), x, w.to(dev), bias_dtype=torch.float32)
    _check_gradients(got, f64(gy), xe, f64(w), None, "none", t, t)


@pytest.mark.parametrize("c", [256, 250, 33, 1030])
def test_norm_sum_in_place(dev, R, c):
    """The C call with h stored over x, or over the residual."""
    from plattice_pytorch_b200 import _lib
    rows = 3001
    x, r, gain = (_randn(s, i).to(dev) for i, s in ((101, (rows, c)), (102, (rows, c)), (103, (c,))))
    y, h, rstd = R.rms_norm(x, gain, r)
    for over in range(2):
        a, b, y2, rstd2 = x.clone(), r.clone(), torch.empty_like(y), torch.empty_like(rstd)
        rc = _lib.lib().plattice_rms_norm(y2.data_ptr(), None, (a, b)[over].data_ptr(), rstd2.data_ptr(), a.data_ptr(),
                                          b.data_ptr(), gain.data_ptr(), 0, 0, 1e-6, rows, c,
                                          torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert torch.equal((a, b)[over], h) and torch.equal(y2, y) and torch.equal(rstd2, rstd)


def test_changed_fields_of_rows8_are_refused(dev, R):
    w = torch.zeros(5, 64, device=dev)
    for shape in ((7, 64), (3, 64), (4, 32), (4, 65)):
        r = R.pack8(torch.zeros(4, 64, device=dev))
        r.shape = shape
        for call in (lambda: R.unpack8(r), lambda: R.linear(r, w),
                     lambda: R.linear_backward(torch.zeros(4, 5, device=dev), r, w)):
            with pytest.raises(RuntimeError):
                call()


# Rows enough for the forms that many rows take, at sizes where each can go wrong.
LARGER_SHAPES = [(2500, 50, 24), (2401, 7, 2), (2400, 264, 1), (4000, 64, 8), (2500, 1000, 32), (2385, 1, 16),
                 (9500, 200, 17), (2100, 130, 200), (2500, 96, 33), (2401, 512, 72), (3700, 33, 257), (8000, 29, 41),
                 (2500, 9000, 8), (150, 72, 5000), (17, 40, 4800), (2370, 640, 32)]


@pytest.mark.parametrize("dtype,x8", KINDS)
@pytest.mark.parametrize("rows,k,n", LARGER_SHAPES)
@pytest.mark.parametrize("act,residual,keep,out32", [("none", False, None, True), ("gelu", True, "8bit", False),
                                                     ("silu", False, "full", False), ("relu", True, None, True)])
def test_linear_larger(dev, R, rows, k, n, dtype, x8, act, residual, keep, out32):
    test_linear(dev, R, rows, k, n, dtype, x8, act, residual, keep, out32)


@pytest.mark.parametrize("dtype,x8", KINDS)
@pytest.mark.parametrize("rows,k,n,split", [(2500, 64, 24, 16), (2399, 50, 8, 5), (2500, 700, 13, 1), (3000, 96, 150, 70)])
def test_linear_split_larger(dev, R, rows, k, n, split, dtype, x8):
    test_linear_split(dev, R, rows, k, n, split, dtype, x8)


def test_repeat_stream_and_graph_larger(dev, R):
    test_repeat_stream_and_graph_give_the_same_bits(dev, R, 7001)


@pytest.mark.parametrize("k,n", [(64, 24), (200, 24), (64, 40), (72, 520)])
def test_not_finite_and_unaligned_larger(dev, R, k, n):
    """Rows of values that are not finite stay in their rows, and storage that
    starts one element later gives the same products within their bounds."""
    rows = 5000
    for dtype in DTYPES.values():
        x, w = _randn((rows, k), 63, dtype), _randn((n, k), 64, dtype, k ** -0.5)
        clean, _ = R.linear(x.to(dev), w.to(dev))
        moved = torch.empty(rows * k + 1, dtype=dtype, device=dev)[1:].view(rows, k).copy_(x)
        y, _ = R.linear(moved, w.to(dev))
        ye = f64(x) @ f64(w).T
        for got in (clean, y):
            assert worst(f64(got), ye, _forward_tolerance(f64(x), f64(w), None, 0 * ye, ye, k, dtype)) <= 1
        x[5, 3], x[4130, 60] = float("nan"), float("inf")
        y, _ = R.linear(x.to(dev), w.to(dev))
        good = torch.ones(rows, dtype=torch.bool)
        good[5] = good[4130] = False
        assert torch.equal(y.cpu()[good], clean.cpu()[good])
        assert not torch.isfinite(y[5]).any() and not torch.isfinite(y[4130]).any()


def test_inference_mode_and_inputs_with_gradients(dev, R):
    """The calls are not autograd Functions: they give the same under every
    grad mode, and nothing they return has a history."""
    x = _randn((70, 64), 110).to(dev)
    w, g = _randn((40, 64), 111).to(dev), _randn((64,), 112).to(dev)

    def run(x, w, g):
        y8, h, rstd = R.rms_norm(x, g, x, pack=True)
        y, z = R.linear(y8, w, act="gelu", keep="8bit")
        gx, gw, gb = R.linear_backward(y, y8, w, z, act="gelu")
        return [R.unpack8(y8), h, rstd, y, R.unpack8(z), gx, gw, gb, *R.rms_norm_backward(gx, h, rstd, g)]
    want = run(x, w, g)
    with torch.inference_mode():
        got = run(x.clone(), w.clone(), g.clone())
        assert all(t.is_inference() for t in got)
    got2 = run(*(t.clone().requires_grad_() for t in (x, w, g)))
    assert not any(t.requires_grad for t in got2)
    for a, b, c in zip(want, got, got2):
        assert torch.equal(a, b) and torch.equal(a, c)
