"""Rows from labels, log probabilities of labels and their gradients against float64
definitions (labels_reference.py), over types, sizes, masks and alignments."""
import numpy as np
import pytest
import torch

import labels_reference as ref
from rows_reference import U, f64, half_step, worst

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


def _randn(shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def _labels(shape, n, seed, outside=0.1, wide=True):
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, n, shape)
    ids = np.where(rng.random(shape) < outside, rng.choice([-1, n, 255 + n, -(1 << 31)], shape), ids)
    return torch.from_numpy(ids.astype(np.int64 if wide else np.int32))


def _rounded(dtype, value):
    half = half_step(dtype)
    return half * np.abs(value) + ref.tiny(half)


# ---------------------------------------------------------------- rows from labels

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,n,c", [((1,), 1, 1), ((7,), 5, 3), ((13, 29), 21, 50), ((100,), 1000, 64), ((3, 5, 2), 4, 1030),
                                       ((4097,), 33, 8), ((2,), 3, 4096), ((0,), 3, 8), ((), 6, 12)])
def test_embed(dev, R, dtype, shape, n, c):
    table = _randn((n, c), 1, dtype)
    for wide in (True, False):
        ids = _labels(shape, n, 2, wide=wide)
        got = R.embed(ids.to(dev), table.to(dev), scale=1.7)
        assert got.shape == shape + (c,) and got.dtype == dtype
        want = ref.embed(ids.numpy().reshape(-1), f64(table), 1.7).reshape(shape + (c,))
        assert worst(f64(got), want, _rounded(dtype, want) + 2 * U * np.abs(want) + 1e-300) <= 1


def test_embed_repeats_the_table_exactly(dev, R):
    table = _randn((9, 40), 1, torch.bfloat16).to(dev)
    ids = torch.arange(9, device=dev).flip(0)
    assert torch.equal(R.embed(ids, table), table.flip(0))


def test_embed_of_nonfinite_rows(dev, R):
    table = torch.tensor([[1.0, float("inf"), float("nan")], [2.0, -0.0, 3.0]], device=dev)
    got = R.embed(torch.tensor([1, -1, 0, 2], device=dev), table, 2.0)
    assert torch.equal(got[0], torch.tensor([4.0, -0.0, 6.0], device=dev)) and not got[1].any() and not got[3].any()
    assert got[2, 0] == 2 and torch.isposinf(got[2, 1]) and torch.isnan(got[2, 2])


@pytest.mark.parametrize("count,n", [(40, 30), (20000, 30), (20000, 3000)])
def test_gradients_that_are_not_finite(dev, R, count, n):
    """Reach their own label's row and no other; those of rows without a label reach none."""
    g = _randn((count, 16), 12)
    ids = _labels((count,), n, 13, 0.2)
    ids[0], ids[1], ids[2] = 4, 5, -1
    g[0, 3], g[1, 7], g[2] = float("inf"), float("nan"), float("nan")
    got = R.embed_backward(g.to(dev), ids.to(dev), n).cpu()
    assert torch.isposinf(got[4, 3]) and torch.isnan(got[5, 7])
    got[4, 3] = got[5, 7] = 0
    assert torch.isfinite(got).all()


EMBED_SIZES = [((1,), 1, 1), ((7,), 5, 3), ((13, 29), 21, 50), ((100,), 1000, 64), ((3, 5, 2), 4, 1030), ((4097,), 33, 8),
               ((9000,), 3, 8), ((20000,), 257, 24), ((5000,), 70000, 16), ((2,), 3, 4096), ((0,), 3, 8), ((40000,), 1, 17),
               ((70000,), 21, 64), ((300,), 256, 2048), ((8192,), 97, 2), ((8193,), 300, 4), ((2049,), 1100, 3), ((32768,), 70000, 2), ((32769,), 2000, 2),
               ((20011,), 5, 24), ((300000,), 96, 6),
               ((500,), 12, 5000), ((300000,), 200000, 1), ((1200000,), 1000, 1), ((4200000,), 200, 1), ((4194305,), 1000000, 1),
               ((4200001,), 60000, 1), ((200000,), 1, 3), ((150000,), 2, 4), ((200000,), 1, 5)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,n,c", EMBED_SIZES)
def test_embed_backward(dev, R, dtype, shape, n, c):
    gy = _randn(shape + (c,), 3, dtype)
    for wide, outside in ((True, 0.1), (False, 0.0)):
        ids = _labels(shape, n, 4, outside, wide)
        want, bound = ref.embed_backward(f64(gy), ids.numpy(), n, 0.6)
        for out in TYPES:
            got = R.embed_backward(gy.to(dev), ids.to(dev), n, scale=0.6, dtype=out)
            assert got.shape == (n, c) and got.dtype == out
            assert worst(f64(got), want, _rounded(out, want) + bound + 1e-300) <= 1


@pytest.mark.parametrize("skew", ["one", "zipf", "runs", "none"])
def test_embed_backward_of_skewed_labels(dev, R, skew):
    rng = np.random.default_rng(5)
    k, n, c = 30000, 5000, 36
    ids = {"one": np.full(k, 77), "zipf": np.minimum(rng.zipf(1.3, k) - 1, n - 1), "runs": np.arange(k) // 700,
           "none": np.full(k, -1)}[skew].astype(np.int64)
    gy = _randn((k, c), 6, torch.bfloat16)
    want, bound = ref.embed_backward(f64(gy), ids, n, 1.0)
    got = R.embed_backward(gy.to(dev), torch.from_numpy(ids).to(dev), n, dtype=torch.float32)
    assert worst(f64(got), want, _rounded(torch.float32, want) + bound + 1e-300) <= 1
    again = R.embed_backward(gy.to(dev), torch.from_numpy(ids).to(dev), n, dtype=torch.float32)
    assert torch.equal(got, again)


def test_embed_of_unaligned_rows(dev, R):
    for dtype in TYPES:
        base = _randn((1 + 50 * 16,), 7, dtype).to(dev)
        table = base[1:].view(50, 16)
        ids = _labels((333,), 50, 8).to(dev)
        y = R.embed(ids, table, 3.0)
        assert torch.equal(y, R.embed(ids, table.clone(), 3.0))
        gbase = _randn((1 + 333 * 16,), 9, dtype).to(dev)
        g = gbase[1:].view(333, 16)
        assert torch.equal(R.embed_backward(g, ids, 50), R.embed_backward(g.clone(), ids, 50))
        gbase = _randn((1 + 30000 * 16,), 9, dtype).to(dev)   # a small table with many labels
        g, ids = gbase[1:].view(30000, 16), _labels((30000,), 50, 8).to(dev)
        want, bound = ref.embed_backward(f64(g), ids.cpu().numpy(), 50, 1.0)
        got = R.embed_backward(g, ids, 50, dtype=torch.float32)
        assert worst(f64(got), want, _rounded(torch.float32, want) + bound) <= 1
        assert torch.equal(got, R.embed_backward(g.clone(), ids, 50, dtype=torch.float32))


def test_embed_function(dev, R):
    import plattice_pytorch_b200 as P
    table = _randn((21, 64), 1).to(dev).requires_grad_(True)
    ids = _labels((5, 40), 21, 2).to(dev)
    y = P.RowEmbedFunction.apply(ids, table, 2.0)
    g = _randn((5, 40, 64), 3).to(dev)
    y.backward(g)
    assert torch.equal(table.grad, R.embed_backward(g, ids, 21, 2.0))
    table.grad = None
    P.RowEmbedFunction.apply(ids, table, 2.0).sum().backward()   # a gradient without strides of its own
    inside = ids[(ids >= 0) & (ids < 21)]
    assert torch.equal(table.grad, 2.0 * torch.bincount(inside, minlength=21).float()[:, None].expand(21, 64))


# ---------------------------------------------------------------- log probabilities

def _scores(rows, n, dtype, seed, masked=True):
    x = _randn((rows, n), seed, torch.float32, 3.0) + _randn((rows, 1), seed + 1, torch.float32, 4.0)
    if masked:
        rng = np.random.default_rng(seed)
        x[torch.from_numpy(rng.random((rows, n)) < 0.1)] = float("-inf")
        x[torch.from_numpy(rng.random(rows) < 0.05)] = float("-inf")
        if rows > 3:
            x[3] = float("-inf")
            x[2] = torch.finfo(dtype).min
            x[1] = 0.0
    return x.to(dtype)


LOGP_SIZES = [(1, 1), (5, 2), (40, 3), (33, 21), (257, 32), (9, 33), (20, 100), (3, 255), (70, 256), (12, 1000), (6, 1024),
              (4, 2050), (5, 5003), (2, 33000), (1, 70001), (150, 4096), (0, 7), (2, 131072), (300, 64), (130, 65), (300, 127), (129, 128), (200, 129), (1, 300001), (40, 40000)]


def _check_logp(dev, R, x, top, labels):
    n = x.shape[-1]
    want = ref.LogProbs(f64(x))
    r = R.log_probs(x.to(dev), None if labels is None else labels.to(dev), top=top)
    assert worst(f64(r.entropy), want.entropy, want.e_entropy + 2.0 ** -149) <= 1
    fine = ~want.empty
    assert worst(f64(r.lse)[fine], want.lse[fine], want.e_lse[fine] + 2.0 ** -149) <= 1
    assert np.isneginf(f64(r.lse)[~fine]).all()
    assert np.array_equal(f64(r.stats)[:, 0], want.m[:, 0])
    if labels is not None:
        at = labels.numpy()
        inside = (at >= 0) & (at < n)
        lp = want.logp[np.arange(len(at)), np.where(inside, at, 0)]
        el = want.e_logp[np.arange(len(at)), np.where(inside, at, 0)]
        got = f64(r.logp)
        assert not got[~inside].any()
        closed = inside & np.isneginf(lp)
        assert np.isneginf(got[closed]).all()
        ok = inside & ~closed
        assert worst(got[ok], lp[ok], el[ok] + 2.0 ** -149) <= 1
    if top:
        ids = want.top[:, :top]
        assert r.top_ids.dtype == torch.int64 and np.array_equal(r.top_ids.cpu().numpy(), ids)
        lp, el = np.take_along_axis(want.logp, ids, 1), np.take_along_axis(want.e_logp, ids, 1)
        got = f64(r.top_logp)
        closed = np.isneginf(lp)
        assert np.isneginf(got[closed]).all()
        assert worst(got[~closed], lp[~closed], el[~closed] + 2.0 ** -149) <= 1
    return r, want


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", LOGP_SIZES)
def test_log_probs(dev, R, dtype, rows, n):
    for masked in (False, True):
        x = _scores(rows, n, dtype, 10, masked)
        for wide, top in ((True, 0), (False, min(n, 5))):
            _check_logp(dev, R, x, top, _labels((rows,), n, 11, 0.1, wide))


@pytest.mark.parametrize("top", [1, 2, 7, 8, 31, 32])
@pytest.mark.parametrize("rows,n", [(3, 32), (50, 40), (5, 300), (2, 9001), (1, 65536)])
def test_alternatives(dev, R, rows, n, top):
    for dtype in TYPES:   # 16 bits: many equal scores
        _check_logp(dev, R, _scores(rows, n, dtype, 20), top, None)
    few = torch.randint(0, 3, (rows, n), generator=torch.Generator().manual_seed(1)).float()
    _check_logp(dev, R, few, top, None)
    falling = torch.arange(n, 0, -1).float().expand(rows, n).contiguous()
    _check_logp(dev, R, falling, top, None)
    _check_logp(dev, R, falling.flip(1).contiguous(), top, None)
    zeros = torch.where(few > 1, 0.0, -0.0)   # equal, whatever their signs
    r = R.log_probs(zeros.to(dev), top=top)
    assert torch.equal(r.top_ids.cpu(), torch.arange(top).expand(rows, top))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", LOGP_SIZES)
def test_log_probs_backward(dev, R, dtype, rows, n):
    for masked in (False, True):
        x, labels = _scores(rows, n, dtype, 30, masked), _labels((rows,), n, 31)
        r = R.log_probs(x.to(dev), labels.to(dev))
        want = ref.LogProbs(f64(x))
        g = [_randn((rows,), 32 + i) for i in range(3)]
        for use in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1), (0, 0, 0)):
            gs = [v if u else None for v, u in zip(g, use)]
            got = R.log_probs_backward(x.to(dev), r, labels.to(dev), *(None if v is None else v.to(dev) for v in gs))
            assert got.dtype == dtype and got.shape == x.shape
            grad, bound = want.backward(labels.numpy(), *(None if v is None else f64(v) for v in gs))
            assert worst(f64(got), grad, bound + _rounded(dtype, grad)) <= 1


def test_gradient_is_the_difference(dev, R):
    """Of logp, entropy and lse with respect to each score: central differences in float64
    of the definition, to their own error (h^2 / 6 of third derivatives below 1)."""
    x = _scores(6, 17, torch.float32, 40, masked=False)
    labels, h = torch.tensor([0, 3, 16, -1, 5, 2]), 1e-4
    g = [f64(_randn((6,), 41 + i)) for i in range(3)]

    def loss(v):
        w = ref.LogProbs(v)
        lp = np.where(labels.numpy() < 0, 0.0, w.logp[np.arange(6), labels.numpy()])
        return g[0] * lp + g[1] * w.entropy + g[2] * w.lse
    r = R.log_probs(x.to(dev), labels.to(dev))
    got = f64(R.log_probs_backward(x.to(dev), r, labels.to(dev), *(torch.from_numpy(v).float().to(dev) for v in g)))
    for j in range(17):
        up, down = f64(x), f64(x)
        up[:, j] += h
        down[:, j] -= h
        assert np.abs((loss(up) - loss(down)) / (2 * h) - got[:, j]).max() < 5e-6


def test_scores_that_are_not_finite(dev, R):
    x = _randn((4, 50), 50).to(dev)
    x[0, 7], x[1, 9] = float("nan"), float("inf")
    x[3] = float("-inf")
    labels = torch.tensor([1, 1, 1, 1], device=dev)
    r = R.log_probs(x, labels, top=3)
    for t in (r.logp, r.entropy, r.top_logp):
        assert torch.isnan(t[:2]).all() and not torch.isnan(t[2:]).any()
    assert r.logp[3] == float("-inf") and r.entropy[3] == 0 and r.top_ids[3].tolist() == [0, 1, 2]
    order = torch.sort(torch.nan_to_num(x[:2], nan=-1e9, posinf=1e9), dim=1, descending=True, stable=True)[1][:, :3]
    assert torch.equal(r.top_ids[:2], order)
    one = torch.ones(4, device=dev)
    g = R.log_probs_backward(x, r, labels, one, one, one)
    assert torch.isnan(g[:2]).all() and torch.isfinite(g[2:]).all() and not g[3].any()
    plain = R.log_probs(x[2:3].contiguous(), labels[2:3], top=3)
    for a, b in zip(plain, r):
        assert torch.equal(a[0], b[2])


@pytest.mark.parametrize("n", [3, 70, 300, 1200, 6000, 40001, 140000])
def test_confident_answers_keep_their_precision(dev, R, n):
    """Rows by a thread, a warp, a CTA and a cluster; to the bounds of the exponentials
    (|d| up to 41 counts, 2 U |d| + 8 U) and of sums of n terms, relative to what is left."""
    x = torch.tensor([[20.0, 0.0, -1.0], [1e4, 0.0, 0.0], [40.0, 1.0, 2.0]])
    x = torch.cat([x, torch.full((3, n - 3), -70.0)], 1)
    for dtype in (torch.float32, torch.bfloat16):
        v = x.to(dtype).to(dev)
        labels = torch.zeros(3, dtype=torch.int64, device=dev)
        r = R.log_probs(v, labels, top=2)
        below = f64(v)[:, 1:] - f64(v)[:, :1]   # all of them: float64's sum with the 1 would lose exp(-40), too
        rest = np.exp(below).sum(1)
        entropy = np.log1p(rest) - (np.exp(below) * below).sum(1) / (1 + rest)
        e = (2 * 41 + 8 + 10 + n / 32 + 40) * U
        assert worst(f64(r.logp), -np.log1p(rest), e * rest + 2.0 ** -149) <= 1
        assert worst(f64(r.top_logp)[:, 0], -np.log1p(rest), e * rest + 2.0 ** -149) <= 1
        g = f64(R.log_probs_backward(v, r, labels, torch.ones(3, device=dev)))
        want = rest / (1 + rest)
        assert worst(g[:, 0], want, (e + half_step(dtype)) * want + 2.0 ** -134) <= 1
        assert worst(f64(r.entropy), entropy, 2 * e * entropy + 2.0 ** -126) <= 1


def test_log_probs_of_unaligned_rows(dev, R):
    for dtype in TYPES:
        for rows, n in ((40, 64), (7, 2048), (1, 40000)):
            x = _scores(rows, n, dtype, 60)
            base = torch.empty(1 + rows * n, dtype=dtype, device=dev)
            moved = base[1:].view(rows, n)
            moved.copy_(x)
            labels = _labels((rows,), n, 61).to(dev)
            r, _ = _check_logp(dev, R, x, 4, labels.cpu())
            q = R.log_probs(moved, labels, top=4)
            assert torch.equal(q.top_ids, r.top_ids) and torch.equal(q.stats[..., 0], r.stats[..., 0])
            want = ref.LogProbs(f64(x))
            assert worst(f64(q.entropy), want.entropy, want.e_entropy + 2.0 ** -149) <= 1
            g = _randn((rows,), 62).to(dev)
            got = R.log_probs_backward(moved, q, labels, g)
            grad, bound = want.backward(labels.cpu().numpy(), f64(g))
            assert worst(f64(got), grad, bound + _rounded(dtype, grad)) <= 1


@pytest.mark.parametrize("n", [7, 100, 900, 5000, 70000])
@pytest.mark.parametrize("offset", [3e5, 5e6, -2e9, 1e30, -3e38, 60000.0, -65000.0])
def test_scores_of_any_size(dev, R, offset, n):
    """Scores around a large one: the exponentials are of the differences (what the type
    leaves of them), whatever the size; so are the gradients."""
    for dtype in TYPES:
        if abs(offset) > torch.finfo(dtype).max:
            continue
        x = _randn((4, n), 80, torch.float32, 4.0).double()
        x = (x + offset).clamp(torch.finfo(dtype).min, torch.finfo(dtype).max).to(dtype)
        x[1, ::2] = float("-inf")
        x[2, 3] = offset / 2
        labels = torch.tensor([1, 1, 3, 5])
        r, want = _check_logp(dev, R, x, 2, labels)
        g = [_randn((4,), 81 + i) for i in range(2)]
        got = R.log_probs_backward(x.to(dev), r, labels.to(dev), *(v.to(dev) for v in g))
        grad, bound = want.backward(labels.numpy(), *(f64(v) for v in g))
        assert worst(f64(got), grad, bound + _rounded(dtype, grad)) <= 1


def test_log_prob_function(dev, R):
    import plattice_pytorch_b200 as P
    x = _scores(60, 21, torch.float32, 70).to(dev).view(6, 10, 21).requires_grad_(True)
    labels = _labels((6, 10), 21, 71).to(dev)
    logp, entropy, lse = P.RowLogProbFunction.apply(x, labels)
    gs = [_randn((6, 10), 72 + i).to(dev) for i in range(3)]
    torch.autograd.backward((logp, entropy, lse), gs)
    r = R.log_probs(x.detach(), labels)
    assert torch.equal(logp, r.logp) and torch.equal(entropy, r.entropy) and torch.equal(lse, r.lse)
    want = R.log_probs_backward(x.detach(), r, labels, *gs)
    assert torch.equal(x.grad, want)
    x.grad = None
    P.RowLogProbFunction.apply(x, labels)[1].sum().backward()
    assert torch.equal(x.grad, R.log_probs_backward(x.detach(), r, None, None, torch.ones_like(entropy)))
