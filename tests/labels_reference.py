"""Embedding, line recurrence, log probabilities and clipping from their definitions in
float64 on the CPU (numpy), with the bounds of a float32 evaluation's errors beside them."""
import numpy as np

from rows_reference import U


def tiny(half):
    """Half of the smallest step of results whose relative half step is `half`."""
    return {2.0 ** -11: 2.0 ** -25, 2.0 ** -8: 2.0 ** -134}.get(half, 2.0 ** -149)


def embed(ids, table, scale):
    inside = (ids >= 0) & (ids < len(table))
    y = table[np.where(inside, ids, 0)] * scale
    y[~inside] = 0.0
    return y


def embed_backward(gy, ids, n, scale):
    """(sums, bound): terms are added in float32 in some order, each addition within U of
    the sum of magnitudes; the scale's rounding and product take 2 U more."""
    gy, ids = gy.reshape(-1, gy.shape[-1]), ids.reshape(-1)
    g, m, k = np.zeros((n, gy.shape[-1])), np.zeros((n, gy.shape[-1])), np.zeros((n, 1))
    inside = (ids >= 0) & (ids < n)
    np.add.at(g, ids[inside], gy[inside])
    np.add.at(m, ids[inside], np.abs(gy[inside]))
    np.add.at(k, ids[inside], 1)
    return g * scale, (k * U * m + 2 * U * np.abs(g)) * abs(scale)


def recurrence(a, u, first, m_first=None):
    """h over axis -2 and the bound of its float32 error: M adds up magnitudes along the
    line, and each step (a product and a sum, u's own two roundings, and for lines that are
    cut the product of the gates) is within 4 U of M."""
    h, e = np.empty_like(u), np.empty_like(u)
    hh, mm, ee = first, np.abs(first), np.zeros_like(first)
    for t in range(u.shape[-2]):
        hh = a[..., t, :] * hh + u[..., t, :]
        mm = np.abs(a[..., t, :]) * mm + np.abs(u[..., t, :])
        ee = np.abs(a[..., t, :]) * ee + 4 * U * mm
        h[..., t, :], e[..., t, :] = hh, ee
    return h, e


def scan(x, a, state=None, blend=False, reverse=False):
    """h, last and their bounds."""
    if reverse:
        x, a = x[..., ::-1, :], a[..., ::-1, :]
    first = np.zeros(x.shape[:-2] + x.shape[-1:]) if state is None else state
    u = (1 - a) * x if blend else x
    h, e = recurrence(a, u, first)
    last, e_last = (h[..., -1, :], e[..., -1, :]) if x.shape[-2] else (first, np.zeros_like(first))
    back = (lambda v: v[..., ::-1, :]) if reverse else (lambda v: v)
    return back(h), back(e), last, e_last


def scan_backward(gh, x, a, state=None, glast=None, blend=False, reverse=False):
    """(grad_x, grad_gate, grad_state) and their bounds."""
    if reverse:
        x, a, gh = x[..., ::-1, :], a[..., ::-1, :], gh[..., ::-1, :]
    first = np.zeros(x.shape[:-2] + x.shape[-1:]) if state is None else state
    late = np.zeros_like(first) if glast is None else glast
    if x.shape[-2] == 0:
        return (x, x, late), (x, x, np.zeros_like(first))
    u = (1 - a) * x if blend else x
    h, eh = recurrence(a, u, first)
    before = np.concatenate([first[..., None, :], h[..., :-1, :]], -2)
    e_before = np.concatenate([np.zeros_like(first)[..., None, :], eh[..., :-1, :]], -2)
    later = np.concatenate([a[..., 1:, :], np.ones_like(a[..., :1, :])], -2)
    G, eG = recurrence(later[..., ::-1, :], gh[..., ::-1, :], late)
    G, eG = G[..., ::-1, :], eG[..., ::-1, :]
    d = before - x if blend else before
    e_d = e_before + U * (np.abs(before) + np.abs(x)) if blend else e_before
    gx = (1 - a) * G if blend else G
    e_gx = (np.abs(1 - a) * eG + 3 * U * np.abs(gx)) if blend else eG
    ga = G * d
    e_ga = np.abs(d) * eG + np.abs(G) * e_d + eG * e_d + 2 * U * np.abs(ga)
    gs = a[..., 0, :] * G[..., 0, :]
    e_gs = np.abs(a[..., 0, :]) * eG[..., 0, :] + 2 * U * np.abs(gs)
    back = (lambda v: v[..., ::-1, :]) if reverse else (lambda v: v)
    return (back(gx), back(ga), gs), (back(e_gx), back(e_ga), e_gs)


class LogProbs:
    """Rows of scores x [rows, n] (finite or -inf): logp of every class, entropy, lse, the
    order of the classes, and the bounds `e_*` of a float32 evaluation:

    * x - m is within U |d|; its exponential within 2 U |d| + 8 U of itself (the argument's
      product with log2(e), two units for the function); sums of n terms by at least 32
      lanes (or one lane for up to 128 classes) within (n / 32 + 40) U (n U)
    * s = log(sum) takes the sum's relative error and 4 U of its own
    """

    def __init__(self, x):
        self.x = x
        rows, n = x.shape
        m = x.max(1, keepdims=True)
        self.empty = empty = np.isneginf(m[:, 0])
        safe = np.where(empty[:, None], 0.0, m)
        d = np.where(empty[:, None], -np.inf, x - safe)
        e = np.exp(d)
        total = np.where(empty[:, None], 1.0, e.sum(1, keepdims=True))
        self.m, s = m, np.log(total)
        self.logp = d - s
        self.p = p = np.where(empty[:, None], 0.0, e / total)
        with np.errstate(invalid="ignore"):
            pd = np.where(p > 0, p * d, 0.0)
            self.entropy = np.where(empty, 0.0, (s[:, 0] - pd.sum(1)))
            pd2 = np.where(p > 0, p * d * d, 0.0).sum(1)
        self.lse = np.where(empty, -np.inf, (m + s)[:, 0])
        self.top = np.argsort(-x, axis=1, kind="stable")
        depth = (n if n <= 128 else n / 32 + 40) + 8
        w = -pd.sum(1)
        self.e_s = U * (depth + 2 * w) + 4 * U * s[:, 0]
        self.e_logp = U * np.where(np.isfinite(d), np.abs(d), 0) + self.e_s[:, None] + 2 * U * np.where(
            np.isfinite(self.logp), np.abs(self.logp), 0)
        self.e_entropy = self.e_s + U * (depth + 4) * w + 2 * U * pd2 + 2 * U * (s[:, 0] + w)
        self.e_lse = self.e_s + U * np.where(empty, 0.0, np.abs(self.lse))

    def backward(self, labels, gl=None, ge=None, gz=None):
        """(gradient of x, bound)."""
        rows, n = self.x.shape
        zero = np.zeros(rows)
        gl, ge, gz = (zero if g is None else g for g in (gl, ge, gz))
        inside = zero.astype(bool) if labels is None else (labels >= 0) & (labels < n)
        one = np.zeros((rows, n))
        at = np.where(inside)[0]
        if len(at):
            one[at, labels[at]] = 1.0
        gl = np.where(inside, gl, 0.0)[:, None]
        ge, gz = ge[:, None], gz[:, None]
        lp = np.where(self.p > 0, self.logp, 0.0)
        with np.errstate(invalid="ignore"):
            lh = np.where(self.p > 0, lp + self.entropy[:, None], 0.0)
        g = gl * (one - self.p) - ge * self.p * lh + gz * self.p
        rp = self.e_logp + 2 * U * np.abs(lp) + 10 * U   # of p, relative
        e = (np.abs(gl) * (self.p * rp + 6 * U * np.abs(one - self.p))
             + np.abs(ge) * self.p * (rp * np.abs(lh) + self.e_logp + self.e_entropy[:, None] + 3 * U * np.abs(lh))
             + np.abs(gz) * self.p * rp + 4 * U * (np.abs(gl) * np.abs(one - self.p) + np.abs(ge * self.p * lh) + np.abs(gz) * self.p))
        closed = self.empty[:, None]
        return np.where(closed, 0.0, g), np.where(closed, 0.0, e)
