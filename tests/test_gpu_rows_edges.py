"""Row operators at the edges of their ranges: gradients far from 1, values
that are not finite or nearly infinite, float32's last bits, mixed types,
largest sizes.  Definitions in float64 as in rows_reference.py; u = 2^-24 is
half a float32 step."""
import math
import subprocess
import sys

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


# ------------------------------------------------- float16 with any gradient

# One row, few output channels in one pass, tiled products; the last with rows
# that lie on no 16-byte boundaries.
GRAD_SHAPES = [(1, 64, 24), (377, 50, 8), (3000, 200, 17), (500, 72, 40), (3000, 600, 24), (700, 33, 91)]


def _check_grads(got, gy, xe, we, ze, act, t, out, gz_error):
    """Gradients against their definitions: gz off by gz_error of itself (and
    the slope's functions, 2^-18 of gy), sums 2 u a term, one rounding to t."""
    xr, wr, br, gz = ref.linear_backward(gy, xe, we, ze, act)
    rows, n = gz.shape
    az = np.abs(gz) * (gz_error + 2 * U) + 2.0 ** -18 * np.abs(gy) * (act != "none")
    tiny = (t is torch.float16) * 2.0 ** -25 + 1e-37
    for g, e, off, m, size in ((got[0], xr, az @ np.abs(we), n, np.abs(gz) @ np.abs(we)),
                               (got[1], wr, az.T @ np.abs(xe), rows, np.abs(gz).T @ np.abs(xe))):
        g = f64(g)
        assert np.isfinite(g).all()
        assert worst(g, e, off + 2 * U * (m + 8) * size + half_step(t) * np.abs(e) + tiny) <= 1
    assert worst(f64(got[2]), br, az.sum(0) + (rows + 8) * U * np.abs(gz).sum(0) + U * np.abs(br) + 1e-37) <= 1


@pytest.mark.parametrize("act", ["none", "gelu", "relu"])
@pytest.mark.parametrize("scale", [1e-9, 1e-6, 1e6])
@pytest.mark.parametrize("rows,k,n", GRAD_SHAPES)
def test_float16_with_float32_gradients_of_any_size(dev, R, rows, k, n, scale, act):
    """Gradients that float16 does not hold, with weights and inputs that bring
    the results back into its range.  gz keeps 16 bits or more (2^-17), and
    what its parts' products leave out is 2^-17 of them."""
    t = torch.float16
    back = min(max(1 / scale, 1e-4), 1e4) / 8   # float16 holds x and w
    x, w = _randn((rows, k), 1, t, back / math.sqrt(rows)), _randn((n, k), 2, t, back / math.sqrt(n))
    gy = _randn((rows, n), 3, scale=scale)
    z = None if act == "none" else _randn((rows, n), 4).to(dev)
    got = R.linear_backward(gy.to(dev), x.to(dev), w.to(dev), z, act=act, bias_dtype=torch.float32)
    _check_grads(got, f64(gy), f64(x), f64(w), None if z is None else f64(z), act, t, torch.float32, 2.0 ** -16)


def test_float16_weight_gradient_of_a_million_tiny_gradients(dev, R):
    rows = 1 << 20
    for n, k in ((5, 16), (40, 16)):
        x, w = torch.ones(rows, k, dtype=torch.float16, device=dev), torch.ones(n, k, dtype=torch.float16, device=dev)
        gx, gw, gb = R.linear_backward(torch.full((rows, n), 1e-8, device=dev), x, w, bias_dtype=torch.float32)
        # gz in 16 bits, a step of float32 cut for each 16 of at most 16384 rows, one rounding to float16;
        # the bias's sums are chains of fewer than 2^12 float32 additions
        assert worst(f64(gw), np.full((n, k), rows * 1e-8), (2.0 ** -11 + 2.0 ** -16 + 1024 * 2.0 ** -23) * rows * 1e-8) <= 1
        assert worst(f64(gb), np.full(n, rows * 1e-8), 2.0 ** -12 * rows * 1e-8) <= 1
        assert worst(f64(gx), np.full((rows, k), n * 1e-8), 2.0 ** -25 + 2.0 ** -11 * n * 1e-8) <= 1


@pytest.mark.parametrize("rows,k,n", GRAD_SHAPES[:3])
@pytest.mark.parametrize("keep", ["8bit", "full"])
def test_float16_gradients_behind_an_activation(dev, R, rows, k, n, keep):
    """float16 gradients at the type's end, in one pass: times gelu's slope they
    are past it, and gz has a second part for that."""
    t = torch.float16
    gy = torch.where(_randn((rows, n), 5) > 0, 6.5e4, 3e-3).to(t)
    z = _randn((rows, n), 6, t).abs().to(dev) + 1   # slopes of 1.08 to 1.13
    z8 = R.pack8(z) if keep == "8bit" else z
    x, w = _randn((rows, k), 7, t, 1e-3), _randn((n, k), 8, t, 1e-3)
    got = R.linear_backward(gy.to(dev), x.to(dev), w.to(dev), z8, act="gelu", bias_dtype=torch.float32)
    ze = f64(R.unpack8(z8)) if keep == "8bit" else f64(z)
    _check_grads(got, f64(gy), f64(x), f64(w), ze, "gelu", t, t, 2.0 ** -16)


@pytest.mark.parametrize("rows,k,n", GRAD_SHAPES)
@pytest.mark.parametrize("act", ["none", "relu", "silu"])
def test_smallest_float16_gradients(dev, R, rows, k, n, act):
    """Gradients of float16's smallest number: a relu leaves them as they are,
    a slope rounds each to a step or none at most."""
    t = torch.float16
    gy = torch.full((rows, n), 2.0 ** -24).to(t)
    z = _randn((rows, n), 57, t).abs() + 1   # slopes of 0.9 to 1.1
    x, w = torch.full((rows, k), 1024.0).to(t), torch.full((n, k), 1024.0).to(t)
    gx, gw, gb = R.linear_backward(gy.to(dev), x.to(dev), w.to(dev), None if act == "none" else z.to(dev), act=act)
    off = 0.1 + 2.0 ** -11 if act == "silu" else 2.0 ** -11   # |slope - 1| <= 0.1
    assert worst(f64(gx), np.full((rows, k), n * 2.0 ** -14), off * n * 2.0 ** -14 + 2.0 ** -25) <= 1
    assert worst(f64(gw), np.full((n, k), rows * 2.0 ** -14), off * rows * 2.0 ** -14 + 2.0 ** -25) <= 1


def test_float16_split_gradients(dev, R):
    t, rows, k = torch.float16, 900, 64
    for n, cut in ((24, 16), (90, 50)):
        x, w, gy = _randn((rows, k), 9, t, 1e-4), _randn((n, k), 10, t, 1e-4), _randn((rows, n), 11, scale=1e6)
        pair = (gy[:, :cut].contiguous().to(dev), gy[:, cut:].contiguous().to(dev))
        got = R.linear_backward(pair, x.to(dev), w.to(dev), bias_dtype=torch.float32)
        _check_grads(got, f64(gy), f64(x), f64(w), None, "none", t, torch.float32, 2.0 ** -16)


# ---------------------------------- float32 gradients beside 16-bit operands

@pytest.mark.parametrize("x8", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("rows,k,n", GRAD_SHAPES)
def test_float32_gradients_keep_16_bits(dev, R, rows, k, n, dtype, x8):
    """Sums whose large parts cancel: what rounding gz to 8 or 11 bits would
    lose is all that is left of them."""
    t = DTYPES[dtype]
    if x8 and t is torch.float16:
        pytest.skip("8-bit rows take no float16 weights")
    sign = lambda s, i: torch.where(_randn(s, i) > 0, 1.0, -1.0)  # noqa: E731
    x, w = sign((rows, k), 12), sign((n, k), 13).to(t)
    gy = 1 + 2.0 ** -10 * torch.rand(rows, n, generator=torch.Generator().manual_seed(14))
    xin = R.pack8(x.to(dev)) if x8 else x.to(t).to(dev)
    got = R.linear_backward(gy.to(dev), xin, w.to(dev), bias_dtype=torch.float32)
    _check_grads(got, f64(gy), f64(x), f64(w), None, "none", t, torch.float32, 2.0 ** -16)


# ---------------------------------------------------------------- float32

FORMS = [(3, 24), (5000, 24), (700, 40), (5000, 72)]   # rows, n: few rows, few channels, tiles


@pytest.mark.parametrize("rows,n", FORMS)
def test_float32_products_are_float32(dev, R, rows, n):
    """One product of two values just below a bfloat16 step, where the parts
    are largest: at most 2^-8 and 2^-17 beside values of 1 and more, so the two
    products of them that are left out come to 2^-24 = u.  The product of the
    first parts is exact, adding the others to it costs at most 2 u, and the
    others' own sums, 2^-7 of it, less than u."""
    v = np.float32(1 + 2.0 ** -7 - 2.0 ** -23)
    for a, b in ((v, v), (v, -v), (np.float32(1 + 2.0 ** -8 + 2.0 ** -23), v)):
        x = torch.full((rows, 1), float(a), device=dev)
        w = torch.full((n, 1), float(b), device=dev)
        y, _ = R.linear(x, w)
        e = float(a) * float(b)
        assert np.abs(f64(y) / e - 1).max() <= 4 * U
        gy = torch.zeros(rows, n, device=dev)
        gy[0, n - 1] = float(a)
        gx, gw, _ = R.linear_backward(gy, x, w)
        assert abs(f64(gx)[0, 0] / e - 1) <= 4 * U and abs(f64(gw)[n - 1, 0] / float(a) ** 2 - 1) <= 4 * U


@pytest.mark.parametrize("rows,n", FORMS)
def test_gelu_in_float32(dev, R, rows, n):
    """Relative to the value, into the tail: 15 u of the fit, the reciprocal and
    the exponential, and u z^2 of the exponent's rounding."""
    z = torch.linspace(-12.5, 12.5, rows * n).view(rows, n)
    z[0, :4] = torch.tensor([0.0, -1e-6, 1e-6, -0.5])
    w = torch.eye(n)
    y, kept = R.linear(z.to(dev), w.to(dev), act="gelu", keep="full")
    assert torch.equal(kept.cpu(), z)
    ze = f64(z)
    phi = np.vectorize(lambda t: 0.5 * math.erfc(-t / math.sqrt(2)))(ze)
    tol = 2.0 ** -20 * (1 + ze * ze / 16) + 2 * U
    assert worst(f64(y), ze * phi, tol * np.abs(ze * phi) + 1e-37) <= 1
    for kept8 in (False, True):
        zk = R.pack8(z.to(dev)) if kept8 else z.to(dev)
        ze = f64(R.unpack8(zk)) if kept8 else f64(z)
        phi = np.vectorize(lambda t: 0.5 * math.erfc(-t / math.sqrt(2)))(ze)
        dens = ze * np.exp(-ze * ze / 2) / math.sqrt(2 * math.pi)
        gx, _, _ = R.linear_backward(torch.ones(rows, n, device=dev), z.to(dev), w.to(dev), zk, act="gelu",
                                     need=(True, False, False))
        tol = 2.0 ** -20 * (1 + ze * ze / 16) + 2 * U
        assert worst(f64(gx), phi + dens, tol * (phi + np.abs(dens)) + 1e-37) <= 1


# ---------------------------------------------------------------- not finite

def _same(got, want, tol):
    """The same infinities and NaN; finite values within tol."""
    got = f64(got)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(np.isinf(got), inf) and np.array_equal(got[inf], want[inf])
    fine = np.isfinite(want)
    assert (np.abs(got - want)[fine] <= tol[fine]).all()


def _weighted(x, w):
    with np.errstate(invalid="ignore"):
        return (x[:, None, :] * w[None, :, :]).sum(-1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n", FORMS)
@pytest.mark.parametrize("k", [50, 64, 700])
def test_infinite_inputs_give_infinite_sums(dev, R, rows, n, k, dtype):
    t = DTYPES[dtype]
    x, w = _randn((rows, k), 16, t), _randn((n, k), 17, t)
    x[0, 3], x[rows - 1, k - 1] = math.inf, -math.inf
    x[rows // 2, 7], x[rows // 2, 8] = math.inf, math.nan
    w[1, 5], w[n - 1, 3] = -math.inf, math.inf
    x[1, 5] = 0.0   # times the infinite weight: NaN
    y, _ = R.linear(x.to(dev), w.to(dev))
    some = [0, 1, 2, rows // 2, rows - 1]
    e = _weighted(f64(x[some]), f64(w))
    tol = (2 * U * (k + 8) + half_step(t)) * _weighted(np.abs(np.where(np.isfinite(f64(x[some])), f64(x[some]), 0)),
                                                       np.abs(np.where(np.isfinite(f64(w)), f64(w), 0))) + 1e-6
    _same(y[some], e, tol)


@pytest.mark.parametrize("rows,n", FORMS)
def test_infinite_weights_of_8_bit_rows(dev, R, rows, n):
    k = 96
    for t in (torch.float32, torch.bfloat16):
        x, w = R.pack8(_randn((rows, k), 18).abs().add(0.5).to(dev)), _randn((n, k), 19, t)
        w[0, 5], w[n - 1, 95] = math.inf, -math.inf
        y, _ = R.linear(x, w.to(dev), out_dtype=torch.float32)
        xe = f64(R.unpack8(x))[:3]
        e = _weighted(xe, f64(w))
        _same(y[:3], e, 2 * U * (k + 8) * _weighted(np.abs(xe), np.abs(np.where(np.isfinite(f64(w)), f64(w), 0))) + 1e-6)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,n", [(37, 64, 24), (1, 40, 3), (375, 50, 8), (503, 33, 91)])
def test_infinite_input_in_the_last_row(dev, R, rows, k, n, dtype):
    """Where the last block of rows is not whole, the last row counts once."""
    t = DTYPES[dtype]
    x, w, gy = _randn((rows, k), 20, t), _randn((n, k), 21, t), _randn((rows, n), 22, t)
    x[rows - 1, 2] = math.inf
    _, gw, _ = R.linear_backward(gy.to(dev), x.to(dev), w.to(dev))
    e = f64(gy).T @ f64(x)
    _same(gw, e, (2 * U * (rows + 8) + half_step(t)) * (np.abs(f64(gy)).T @ np.abs(np.where(np.isfinite(f64(x)), f64(x), 0))) + 1e-6)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("out32", [False, True])
@pytest.mark.parametrize("rows,k,n", [(37, 64, 24), (375, 50, 8), (500, 72, 40), (503, 33, 91)])
def test_infinite_gradients_and_inputs(dev, R, rows, k, n, dtype, out32):
    """An infinite gradient and an infinite input, in the sums they belong to and
    in no other."""
    t = DTYPES[dtype]
    out = torch.float32 if out32 else t
    x, w, gy = _randn((rows, k), 20, t), _randn((n, k), 21, t), _randn((rows, n), 22, out)
    x[5, 2] = math.inf
    gy[3, 1] = -math.inf
    got = R.linear_backward(gy.to(dev), x.to(dev), w.to(dev), bias_dtype=torch.float32)
    ge, xe, we = f64(gy), f64(x), f64(w)
    fin = lambda a: np.abs(np.where(np.isfinite(a), a, 0))  # noqa: E731
    with np.errstate(invalid="ignore"):
        gx = np.stack([(ge * we[:, j][None]).sum(1) for j in range(k)], 1)
        gw = np.stack([(ge * xe[:, j][:, None]).sum(0) for j in range(k)], 1)
    _same(got[0], gx, (2 * U * (n + 8) + 2.0 ** -16 + half_step(t)) * (fin(ge) @ fin(we)) + 1e-6)
    _same(got[1], gw, (2 * U * (rows + 8) + 2.0 ** -16 + half_step(t)) * (fin(ge).T @ fin(xe)) + 1e-6)
    _same(got[2], ge.sum(0), 2 * U * (rows + 8) * fin(ge).sum(0))


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", DTYPES)
def test_padding_of_rows_that_are_not_finite(dev, R, dtype, bad):
    """Zeros behind the last channel, whatever the row holds."""
    t = DTYPES[dtype]
    for c in (1, 3, 8, 33, 50, 72, 1030):
        x = _randn((40, c), 23, t)
        x[3], x[7, 0] = bad, bad
        y8, _, _ = R.rms_norm(x.to(dev), torch.ones(c, device=dev), pack=True)
        assert not y8.q[:, c:].any()
        assert not R.pack8(x.to(dev)).q[:, c:].any()
    for rows, n in FORMS + [(5000, 9), (5000, 41)]:
        x = _randn((rows, 64), 24, t)
        x[1], x[2, 5] = bad, bad
        for xin in (x.to(dev),) + ((R.pack8(x.to(dev)),) if t is not torch.float16 else ()):
            _, z = R.linear(xin, _randn((n, 64), 25, t).to(dev), act="relu", keep="8bit")
            assert not z.q[:, n:].any()


# ------------------------------------------------- the largest finite values

@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("c", [1, 3, 32, 50, 64])
def test_pack8_of_the_largest_values(dev, R, c, dtype):
    """A block whose largest value is above 240 2^120 stays finite and within
    2^-4 of itself."""
    t = DTYPES[dtype]
    top = torch.finfo(t).max
    for v in (top, -top, 3.32e38, 3.25e38, 3.2e38):
        x = torch.zeros(5, c)
        x[1, c // 2], x[3, 0] = v, v / 2
        x = x.to(t)
        y = f64(R.unpack8(R.pack8(x.to(dev))))
        assert np.isfinite(y).all() and worst(y, f64(x), 2.0 ** -4 * np.abs(f64(x)) + 1e-37) <= 1


@pytest.mark.parametrize("c", [1, 2, 31, 34, 64, 520])
def test_norm_in_8_bits_of_the_largest_values(dev, R, c):
    x = torch.ones(7, c, device=dev)
    gain = torch.full((c,), 3.35e38, device=dev)
    y8, _, _ = R.rms_norm(x, gain, pack=True)
    y = f64(R.unpack8(y8))
    assert np.isfinite(y).all() and worst(y, np.full((7, c), 3.35e38), 2.0 ** -4 * 3.36e38) <= 1


@pytest.mark.parametrize("rows,n", FORMS)
def test_kept_z_of_the_largest_values(dev, R, rows, n):
    for t in (torch.float32, torch.bfloat16):
        b = torch.full((n,), 3.38e38, dtype=t, device=dev)
        _, z = R.linear(torch.zeros(rows, 8, dtype=t, device=dev), torch.zeros(n, 8, dtype=t, device=dev), b, act="relu", keep="8bit")
        y = f64(R.unpack8(z))
        assert np.isfinite(y).all() and worst(y, np.broadcast_to(f64(b), y.shape), 2.0 ** -4 * 3.4e38) <= 1


# ------------------------------------------------------- arguments and sizes

@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_channels_whose_byte_offsets_pass_32_bits(dev, R, dtype):
    """One row whose last channels lie more than 2^31 bytes behind its first."""
    t = DTYPES[dtype]
    k = (1 << 29) + 64 if t is torch.float32 else 1 << 30
    if torch.cuda.mem_get_info(dev)[0] < 8 << 30:
        pytest.skip("needs 8 GB of free device memory")
    x, w = torch.zeros(1, k, dtype=t, device=dev), torch.zeros(1, k, dtype=t, device=dev)
    at = [0, 77, (1 << 29) - 1, (1 << 29) + 3, k - 64, k - 1]
    x[0, at] = _randn((6,), 50, t).to(dev)
    w[0, at] = _randn((6,), 51, t).to(dev)
    y, _ = R.linear(x, w, out_dtype=torch.float32)
    e = f64(x[0, at]) * f64(w[0, at])
    assert abs(f64(y)[0, 0] - e.sum()) <= 2.0 ** -20 * abs(e).sum()   # six terms in float32


def test_sum_that_takes_seconds(dev, R):
    """An input gradient over 2^30 output channels: one tile of 2^24 slices,
    longer than a wait that does not know its sum would have patience for."""
    n, k = 1 << 30, 8
    if torch.cuda.mem_get_info(dev)[0] < 32 << 30:
        pytest.skip("needs 32 GB of free device memory")
    w, gy = torch.zeros(n, k, dtype=torch.bfloat16, device=dev), torch.zeros(1, n, dtype=torch.bfloat16, device=dev)
    at = [0, 12345, n // 2 + 7, n - 65, n - 1]
    w[at] = _randn((5, k), 52, torch.bfloat16).to(dev)
    gy[0, at] = _randn((5,), 53, torch.bfloat16).to(dev)
    x = torch.zeros(1, k, dtype=torch.bfloat16, device=dev)
    gx, _, _ = R.linear_backward(gy, x, w, need=(True, False, False))
    e = f64(gy[0, at]) @ f64(w[at])
    assert worst(f64(gx)[0], e, (2.0 ** -8 + 2.0 ** -20) * (np.abs(f64(gy[0, at])) @ np.abs(f64(w[at])))) <= 1
    torch.cuda.synchronize()
    R.linear_backward(gy[:, :64].contiguous(), x, w[:64], need=(True, False, False))   # would report it


def test_weight_gradient_of_a_million_like_rows(dev, R):
    """Sums of like terms in float16: one rounding, and a step of float32 cut for
    each 16 of the at most 16384 rows that the matrix instructions add up."""
    rows, k, n, t = 1 << 20, 4096, 1024, torch.float16
    if torch.cuda.mem_get_info(dev)[0] < 32 << 30:
        pytest.skip("needs 32 GB of free device memory")
    g = torch.Generator().manual_seed(54)
    part = lambda m, bits: (1 + torch.randint(0, 1 << bits, (m,), generator=g) * 2.0 ** -bits).to(t).to(dev)  # noqa: E731
    a, b, h, c = part(rows, 4), part(k, 4), part(rows, 4), part(n, 4) / 256   # 5 bits each; sums below 65504
    _, gw, _ = R.linear_backward(h[:, None] * c, a[:, None] * b, torch.zeros(n, k, dtype=t, device=dev), need=(False, True, False))
    e = (a.double() * h.double()).sum() * c.double()[:, None] * b.double()   # products of 10 bits: exact in float16
    assert float((gw.double() / e - 1).abs().max()) <= 2.0 ** -11 + 16384 / 16 * 2.0 ** -23 + 70 * U


@pytest.mark.parametrize("dtype,deep", [("fp16", 1 << 17), ("bf16", 1 << 20)])
def test_deep_sums_of_like_terms(dev, R, dtype, deep):
    """The same over input and output channels: one rounding, and at most a step of
    float32 cut for each 16 of a chunk of 512, which then are added in float32."""
    t = DTYPES[dtype]
    g = torch.Generator().manual_seed(55)
    part = lambda m: (1 + torch.randint(0, 8, (m,), generator=g) / 8).to(t).to(dev)  # noqa: E731  4 bits
    bound = half_step(t) + 32 * 2.0 ** -23 + deep / 512 * U
    b, d = part(deep) / 16, part(deep) / 16
    total = (b.double() * d.double()).sum()
    for rows, n in ((400, 200), (5000, 40)):
        a, c = part(rows), part(n)
        y, _ = R.linear(a[:, None] * b, c[:, None] * d)
        assert float((y.double() / (a.double()[:, None] * c.double() * total) - 1).abs().max()) <= bound
    a, c = part(200), part(64)
    gx, _, _ = R.linear_backward(a[:, None] * b, torch.zeros(200, 64, dtype=t, device=dev), d[:, None] * c,
                                 need=(True, False, False))
    assert float((gx.double() / (a.double()[:, None] * c.double() * total) - 1).abs().max()) <= bound


@pytest.mark.parametrize("dtype,x8", [("fp32", False), ("bf16", False), ("fp16", False), ("fp32", True), ("bf16", True)])
@pytest.mark.parametrize("rows,n,cut", [(3, 24, 16), (5000, 24, 16), (5000, 7, 3), (700, 40, 33), (5000, 72, 1)])
def test_split_result_beside_a_kept_z(dev, R, rows, n, cut, dtype, x8):
    """Without activation the kept z is the result before the split, rounded once
    from the same sum."""
    t, k = DTYPES[dtype], 40
    x, w, b = _randn((rows, k), 58, t).to(dev), _randn((n, k), 59, t).to(dev), _randn((n,), 60).to(dev)
    xin = R.pack8(x) if x8 else x
    for keep in ("full", "8bit"):
        (f, v), z = R.linear(xin, w, b, split=cut, keep=keep)
        y = torch.cat([f, v], 1)
        if keep == "full":
            assert torch.equal(z, y)
        else:
            unit = np.repeat(2.0 ** (z.scale.cpu().numpy().astype(np.float64) - 127), 32, 1)[:, :n]
            off = (2.0 ** -4 + 2 * half_step(t)) * np.abs(f64(y)) + 2.0 ** -10 * unit
            assert worst(f64(R.unpack8(z)), f64(y), off) <= 1


def test_half_a_pair_of_gradients_is_refused(dev, R):
    x, w, g = torch.zeros(4, 8, device=dev), torch.zeros(3, 8, device=dev), torch.zeros(4, 3, device=dev)
    for pair in ((g, None), [g, None], (None, g)):
        with pytest.raises(RuntimeError, match="grad_y"):
            R.linear_backward(pair, x, w)


_CAPTURED = """
import ctypes, sys, torch
from plattice_pytorch_b200 import _lib, rows
word = ctypes.CDLL(_lib.LIB_PATH)._ZN2pl10fault_wordEv
word.restype = ctypes.c_void_p
x, w = torch.randn(512, 64, device="cuda"), torch.randn(72, 64, device="cuda")
rows.pack8(x)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y, _ = rows.linear(x, w)
    there = word()
graph.replay()
torch.cuda.synchronize()
assert float((y - x.double() @ w.double().t()).abs().max()) < 1e-3
assert there, "no word"
"""


def test_first_product_in_a_capture_can_report_a_fault(dev):
    """A captured product whose waits give up has a place to say so, also when
    no product ran before the capture."""
    got = subprocess.run([sys.executable, "-c", _CAPTURED], capture_output=True, text=True, timeout=300)
    assert got.returncode == 0, got.stderr[-2000:]


# ---------------------------------------------------------------- under autograd

@pytest.fixture
def P():
    import plattice_pytorch_b200 as P
    return P


def test_layer_is_float32_unless_asked(dev, P):
    """What a layer computes is not rounded to 8 bits without a word of the caller."""
    torch.manual_seed(5)
    m = P.PermutoLatticeLayer(64, 5, 3, act="gelu", device=dev)
    x = _randn((13, 29, 64), 32).to(dev)
    with torch.no_grad():
        n, _, _ = P.rows.rms_norm(x, m.gain)
        (f, v), _ = P.rows.linear(n, m.w_in, m.b_in, split=5, out_dtype=torch.float32)
        o = P.PermutoLatticeFeatureFunction.apply(f, v)
        want = P.RowLinearFunction.apply(o, m.w_out, m.b_out, x, "gelu", False)
        scale = float((want - x).abs().max())
        assert float((m(x) - want).abs().max()) <= 1e-4 * scale   # atomics of the filter's splat
    w = _randn((40, 64), 33).to(dev).requires_grad_(True)
    gy = _randn((13, 29, 40), 34).to(dev)
    P.RowLinearFunction.apply(x, w, None, None).backward(gy)
    assert torch.equal(w.grad, P.rows.linear_backward(gy, x, w.detach())[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_in_8_bits_when_asked(dev, P, dtype):
    """checkpoint8=True is the chain of the Functions with it."""
    t = DTYPES[dtype]
    torch.manual_seed(6)
    m = P.PermutoLatticeLayer(64, 5, 3, act="silu", checkpoint8=True, dtype=t, device=dev)
    x = _randn((16, 24, 64), 35, t).to(dev).requires_grad_(True)
    y = m(x)
    f, v = P.RowNormLinearFunction.apply(x, None, m.gain, m.w_in, m.b_in, 1e-6, "none", 5, torch.float32, True)
    o = P.PermutoLatticeFeatureFunction.apply(f, v)
    want = P.RowLinearFunction.apply(o.to(t), m.w_out, m.b_out, x, "silu", True)
    # the splat's atomics add in another order (1e-4 here), then a step of the type (at most 2^-7 of a value)
    assert float((y - want).detach().float().abs().max()) <= 1e-4 + 2.0 ** -7 * float(want.detach().float().abs().max())
    for g, p in zip(torch.autograd.grad(y.float().square().mean(), [x, *m.parameters()]), [x, *m.parameters()]):
        assert g.shape == p.shape and g.dtype == p.dtype and bool(torch.isfinite(g).all()) and bool(g.any())


@pytest.mark.parametrize("xt,wt", [("fp32", "bf16"), ("bf16", "fp32")])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_linear_of_mixed_types(dev, P, xt, wt, residual):
    leaf = lambda s, i, t: _randn(s, i, DTYPES[t]).to(dev).requires_grad_(True)  # noqa: E731
    x, gain, w, b = leaf((50, 64), 26, xt), leaf((64,), 27, xt), leaf((8, 64), 28, wt), leaf((8,), 29, wt)
    r = leaf((50, 64), 30, xt) if residual else None
    out = P.RowNormLinearFunction.apply(x, r, gain, w, b)
    out = out if residual else (out,)
    gs = [_randn(tuple(o.shape), 31 + i, o.dtype).to(dev) for i, o in enumerate(out)]
    torch.autograd.backward(out, gs)
    with torch.no_grad():
        n, h, rstd = P.rows.rms_norm(x, gain, r, pack=True)
        y, _ = P.rows.linear(n, w, b)
        gn, gw, gb = P.rows.linear_backward(gs[0], n, w)
        gx, gg = P.rows.rms_norm_backward(gn.to(x.dtype), h, rstd, gain, gs[1] if residual else None)
    assert torch.equal(out[0], y)
    for got, want in ((x.grad, gx), (gain.grad, gg), (w.grad, gw), (b.grad, gb)):
        assert got.dtype == want.dtype and torch.equal(got, want)
    assert r is None or torch.equal(r.grad, gx)
    with pytest.raises(RuntimeError, match="same type"):
        P.RowNormLinearFunction.apply(x, r, gain, w, b, 1e-6, "none", 0, None, False)
