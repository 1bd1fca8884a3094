"""The log probabilities of labels_reference.py and their bounds in float64 on the device, for
more rows than numpy goes through in a test's time."""
import torch

from rows_reference import U


class LogProbs:
    def __init__(self, x):
        self.x = x = x.double()
        n = x.shape[1]
        m = x.max(1, keepdim=True)[0]
        self.empty = empty = torch.isneginf(m)
        d = torch.where(empty, -torch.inf, x - torch.where(empty, 0.0, m))
        e = d.exp()
        total = torch.where(empty, 1.0, e.sum(1, keepdim=True))
        self.m, s = m, total.log()
        self.logp = d - s
        self.p = p = torch.where(empty, 0.0, e / total)
        pd = torch.where(p > 0, p * d, 0.0)
        w = -pd.sum(1, keepdim=True)
        self.entropy = torch.where(empty, 0.0, s + w)
        self.lse = m + s
        pd2 = torch.where(p > 0, p * d * d, 0.0).sum(1, keepdim=True)
        depth = (n if n <= 128 else n / 32 + 40) + 8
        self.e_s = U * (depth + 2 * w) + 4 * U * s
        size = lambda v: torch.where(torch.isfinite(v), v.abs(), 0.0)  # noqa: E731
        self.e_logp = U * size(d) + self.e_s + 2 * U * size(self.logp)
        self.e_entropy = self.e_s + U * (depth + 4) * w + 2 * U * pd2 + 2 * U * (s + w)
        self.e_lse = self.e_s + U * size(self.lse)

    def order(self, top):
        """The `top` best classes: of equal scores the lowest first."""
        return torch.sort(self.x + 0.0, dim=1, descending=True, stable=True)[1][:, :top]

    def backward(self, labels, gl, ge, gz):
        n = self.x.shape[1]
        labels = labels.long()[:, None]
        inside = (labels >= 0) & (labels < n)
        one = torch.zeros_like(self.x).scatter_(1, labels.clamp(0, n - 1), inside.double())
        gl, ge, gz = torch.where(inside, gl.double()[:, None], 0.0), ge.double()[:, None], gz.double()[:, None]
        p = self.p
        lp = torch.where(p > 0, self.logp, 0.0)
        lh = torch.where(p > 0, lp + self.entropy, 0.0)
        rest = (one - p).abs()
        g = gl * (one - p) - ge * p * lh + gz * p
        rp = torch.where(torch.isfinite(self.e_logp), self.e_logp, 0.0) + 2 * U * lp.abs() + 10 * U
        e = (gl.abs() * (p * rp + 6 * U * rest) + ge.abs() * p * (rp * lh.abs() + self.e_logp + self.e_entropy + 3 * U * lh.abs())
             + gz.abs() * p * rp + 4 * U * (gl.abs() * rest + (ge * p * lh).abs() + gz.abs() * p))
        return torch.where(self.empty, 0.0, g), torch.where(self.empty, 0.0, e)
