"""The row operators from their definitions in float64 on the CPU (numpy), for the tests."""
import math

import numpy as np
import torch

U = 2.0 ** -24   # half a step of float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def f64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def _e4m3_values():
    v = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        mag = (1 + m / 8) * 2.0 ** (e - 7) if e else m * 2.0 ** -9
        v[c] = np.nan if (c & 127) == 127 else (-mag if c >= 128 else mag)
    return v


E4M3 = _e4m3_values()


def _encode(t):
    """Nearest e4m3 codes of values within +-448, ties to the even code."""
    grid = E4M3[:127]
    a = np.abs(t)
    hi = np.clip(np.searchsorted(grid, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - grid[lo], grid[hi] - a
    code = np.where(dl < dh, lo, np.where(dl > dh, hi, np.where(lo % 2 == 0, lo, hi)))
    return (code + np.where(np.signbit(t), 128, 0)).astype(np.uint8)


def pack8(x):
    """(codes [rows, width], scale bytes [rows, width / 32]) of float64 x [rows, c]."""
    rows, c = x.shape
    width = (c + 31) // 32 * 32
    b = np.zeros((rows, width))
    b[:, :c] = x
    b = b.reshape(rows, width // 32, 32)
    fine = np.isfinite(b)
    amax = np.abs(np.where(fine, b, 0.0)).max(-1)
    m, e = np.frexp(amax)
    s = np.where(amax > 0, e - 9 + (m > 0.875), -110).clip(-110, 120)
    q = _encode(np.where(fine, b, 0.0) / 2.0 ** s[..., None].astype(np.float64))
    q = np.where(fine, q, 0x7f).astype(np.uint8)
    return q.reshape(rows, width), (s + 127).astype(np.uint8)


def unpack8(q, scale, c):
    rows = q.shape[0]
    v = E4M3[q].reshape(rows, -1, 32) * 2.0 ** (scale.astype(np.float64) - 127)[..., None]
    return v.reshape(rows, -1)[:, :c]


_erf = np.vectorize(math.erf)


def act(z, name):
    if name == "relu":
        return np.maximum(z, 0)
    if name == "gelu":
        return 0.5 * z * (1 + _erf(z / math.sqrt(2)))
    if name == "silu":
        return z / (1 + np.exp(-z))
    return z


def act_slope(z, name):
    if name == "relu":
        return (z > 0).astype(np.float64)
    if name == "gelu":
        return 0.5 * (1 + _erf(z / math.sqrt(2))) + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        s = 1 / (1 + np.exp(-z))
        return s * (1 + z * (1 - s))
    return np.ones_like(z)


def rms_norm(x, gain, residual=None, eps=1e-6):
    h = x if residual is None else x + residual
    rstd = 1 / np.sqrt((h * h).mean(-1) + eps)
    return h * rstd[..., None] * gain, h, rstd


def rms_norm_backward(gy, h, rstd, gain, gh=None):
    n = h * rstd[..., None]
    gn = gy * gain
    gx = rstd[..., None] * (gn - n * (gn * n).mean(-1, keepdims=True))
    return (gx if gh is None else gx + gh), (gy * n).reshape(-1, h.shape[-1]).sum(0)


def linear(x, w, b=None, name="none", residual=None):
    z = x @ w.T
    z = z if b is None else z + b
    y = act(z, name)
    return (y if residual is None else y + residual), z


def linear_backward(gy, x, w, z=None, name="none"):
    gz = gy if name == "none" else gy * act_slope(z, name)
    return gz @ w, gz.T @ x, gz.sum(0), gz


def worst(actual, expected, tolerance):
    """max |actual - expected| / tolerance; at most 1 is within."""
    actual, expected = np.asarray(actual, np.float64), np.asarray(expected, np.float64)
    if not actual.size:
        return 0.0
    assert actual.shape == expected.shape
    return float((np.abs(actual - expected) / tolerance).max())
