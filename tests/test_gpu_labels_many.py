"""Label operators and log probabilities at sizes where a warp, a CTA or a cluster has more
than one unit of work, a small table more than one slab of channels, a sort more than two
digits: against float64."""
import numpy as np
import pytest
import torch

import labels_reference as ref
from labels_device import LogProbs
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


def _within(got, want, bound):
    """All of got: -inf where want is, NaN where want is (rows with +inf), else within the bound."""
    ok = torch.where(torch.isneginf(want), got.double() == want, (got.double() - want).abs() <= bound)
    return bool(torch.where(torch.isnan(want), torch.isnan(got), ok).all())


# rows of a warp one after the other; more than a batch of 32 rows (8 with alternatives) of a
# CTA, of clusters of 2, 4 and 8, and of rows that no cluster holds
MANY = [(60000, 300), (60000, 129), (30011, 520), (40000, 1500), (40000, 1504), (12000, 4100), (6000, 9000), (3000, 20000), (3000, 40001),
        (1500, 70001), (700, 140000), (400, 300001)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", MANY)
def test_log_probs_of_many_rows(dev, R, dtype, rows, n):
    g = torch.Generator(device=dev).manual_seed(n)
    randn = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    x = randn(rows, n) * 3 + 4 * randn(rows, 1)
    x[torch.rand(rows, n, generator=g, device=dev) < 0.05] = -torch.inf
    x[torch.rand(rows, generator=g, device=dev) < 0.01] = -torch.inf
    x[7] = 1.5
    x = x.to(dtype)
    labels = torch.randint(-1, n + 1, (rows,), generator=g, device=dev)
    gl, ge, gz = randn(rows), randn(rows), randn(rows)
    results = {top: R.log_probs(x, labels, top=top) for top in (0, 3, 20)}
    grad = R.log_probs_backward(x, results[0], labels, gl, ge, gz)
    half = half_step(dtype)
    step = 60_000_000 // n
    for first in range(0, rows, step):
        at = slice(first, min(rows, first + step))
        want = LogProbs(x[at])
        order = want.order(20)
        label = labels[at]
        inside = (label >= 0) & (label < n)
        pick = label.clamp(0, n - 1)[:, None]
        logp = torch.where(inside, want.logp.gather(1, pick)[:, 0], 0.0)
        e_logp = torch.where(inside, want.e_logp.gather(1, pick)[:, 0], 0.0)
        for top, r in results.items():
            assert _within(r.logp[at], logp, e_logp + 2.0 ** -149)
            assert _within(r.entropy[at], want.entropy[:, 0], want.e_entropy[:, 0] + 2.0 ** -149)
            assert _within(r.lse[at], want.lse[:, 0], want.e_lse[:, 0] + 2.0 ** -149)
            assert torch.equal(r.stats[at][:, 0].double(), want.m[:, 0])
            if top:
                ids = order[:, :top]
                assert torch.equal(r.top_ids[at], ids)
                assert _within(r.top_logp[at], want.logp.gather(1, ids), want.e_logp.gather(1, ids) + 2.0 ** -149)
        w, e = want.backward(label, gl[at], ge[at], gz[at])
        assert _within(grad[at], w, e + half * w.abs() + ref.tiny(half))
        del want, w, e


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("top", [6, 20, 32])
def test_alternatives_of_rows_that_no_cluster_holds(dev, R, dtype, top):
    n = 300001 if dtype == torch.float32 else 600001
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(5, n, generator=g, device=dev)
    x[1, 5000:] = -torch.inf
    x[2] = torch.randint(0, 3, (n,), generator=g, device=dev).float()
    x[3] = torch.arange(n, device=dev).float()
    x[4, 10:] = -torch.inf   # fewer than asked for are open
    x = x.to(dtype)
    want = LogProbs(x)
    r = R.log_probs(x, top=top)
    ids = want.order(top)
    assert torch.equal(r.top_ids, ids)
    assert _within(r.top_logp, want.logp.gather(1, ids), want.e_logp.gather(1, ids) + 2.0 ** -149)


def test_log_probs_of_two_equal_scores(dev, R):
    r = R.log_probs(torch.zeros(70000, 2, device=dev), torch.ones(70000, dtype=torch.int32, device=dev), top=2)
    assert float((r.logp.double() + np.log(2.0)).abs().max()) < 4 * U
    assert float((r.entropy.double() - np.log(2.0)).abs().max()) < 4 * U


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", [(500, 2), (300, 40), (200, 700), (40, 5000), (3, 100000)])
def test_gradients_of_probabilities_near_zero(dev, R, dtype, rows, n):
    """Scores as far apart as 200.  A probability below 2^-126 counts as 0: what it is
    multiplied by, at most |gl| + |ge| (|log p| + entropy) + |gz|, is added to the bound as often;
    twice, as p relative to the largest score is cut off, which is up to its own size above it."""
    g = torch.Generator(device=dev).manual_seed(n)
    x = (torch.randn(rows, n, generator=g, device=dev) * 30).to(dtype)
    labels = torch.randint(-1, n + 1, (rows,), generator=g, device=dev)
    gl, ge, gz = (torch.randn(rows, generator=g, device=dev) for _ in range(3))
    want = LogProbs(x)
    r = R.log_probs(x, labels)
    w, e = want.backward(labels, gl, ge, gz)
    many = gl.abs()[:, None] + ge.abs()[:, None] * (want.logp.abs() + want.entropy) + gz.abs()[:, None]
    half = half_step(dtype)
    assert _within(R.log_probs_backward(x, r, labels, gl, ge, gz), w, e + half * w.abs() + ref.tiny(half) + 2.0 ** -125 * many)
    assert _within(r.entropy, want.entropy[:, 0], want.e_entropy[:, 0] + 2.0 ** -149)


# ---------------------------------------------------------------- small tables

# (labels, n, c): one and several slabs of channels, one and several columns of CTAs, one CTA
# and many, tables whose 16-bit rows go 8 and 4 bytes a lane, channels that end inside a slab
TABLES = [(600, 1, 8), (20000, 21, 256), (20000, 21, 264), (10000, 3, 4096), (40000, 24, 136), (40000, 60, 128), (33000, 60, 200), (50000, 96, 64),
          (50000, 96, 1024), (50000, 95, 1032), (15000, 25, 72), (2000, 2, 24), (1100, 2, 16384), (100003, 7, 8)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count,n,c", TABLES)
def test_sums_of_small_tables(dev, R, dtype, count, n, c):
    g = torch.Generator(device=dev).manual_seed(c)
    flat = torch.randn(count * c + 1, generator=g, device=dev).to(dtype)
    ids = torch.randint(-1, n + 1, (count,), generator=g, device=dev)
    inside = (ids >= 0) & (ids < n)
    for first in (0, 1):   # rows on 16-byte boundaries, and on none
        gy = flat[first:first + count * c].view(count, c)
        rows = gy[inside].double()
        want = torch.zeros(n, c, dtype=torch.float64, device=dev).index_add_(0, ids[inside], rows)
        size = torch.zeros(n, c, dtype=torch.float64, device=dev).index_add_(0, ids[inside], rows.abs())
        k = torch.bincount(ids[inside], minlength=n).double()[:, None]
        for out in (dtype, torch.float32):
            half = half_step(out)
            got = R.embed_backward(gy, ids, n, scale=0.6, dtype=out)
            bound = (k * U * size + 2 * U * want.abs()) * 0.6 + half * 0.6 * want.abs() + ref.tiny(half)
            assert _within(got, want * 0.6, bound + 2.0 ** -149), (first, out)
            assert torch.equal(got, R.embed_backward(gy, ids, n, scale=0.6, dtype=out))


# ---------------------------------------------------------------- sorts of many digits

@pytest.mark.parametrize("count,n,c", [(3000, (1 << 20) + 5, 3), (30000, (1 << 22) + 1, 2), (40000, (1 << 23) + 7, 1), (300000, (1 << 21) + 3, 8),
                                       (5000, (1 << 30) + 9, 1), (60000, (1 << 31) - 1, 1)])
def test_gradients_of_very_large_tables(dev, R, count, n, c):
    rng = np.random.default_rng(n)
    some = rng.integers(0, n, max(1, count // 3))   # each some times
    some[:4] = 0, n - 1, n // 2, n - 2
    ids = some[rng.integers(0, len(some), count)]
    ids[rng.random(count) < 0.05] = -1
    ids[:4] = some[:4]
    g = torch.Generator().manual_seed(2)
    gy = torch.randn(count, c, generator=g).bfloat16()
    got = R.embed_backward(gy.to(dev), torch.from_numpy(ids).to(dev), n)
    found, place = np.unique(ids, return_inverse=True)
    want, bound = ref.embed_backward(f64(gy), place - (1 if found[0] < 0 else 0), len(found), 1.0)
    found = found[found >= 0]
    want, bound = want[:len(found)], bound[:len(found)]
    half = half_step(torch.bfloat16)
    assert worst(f64(got[torch.from_numpy(found).to(dev)]), want, bound + half * np.abs(want) + ref.tiny(half)) <= 1
    got[torch.from_numpy(found).to(dev)] = 0
    assert not got.any()
