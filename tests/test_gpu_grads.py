"""The norm of many gradients together and the gradients scaled down, against float64."""
import math

import numpy as np
import pytest
import torch

from labels_reference import tiny
from rows_reference import U, f64, half_step, worst

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def G():
    from plattice_pytorch_b200 import grads
    return grads


def _tensors(sizes, seed, dev, types=TYPES, scale=0.1):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(*(s if isinstance(s, tuple) else (s,)), generator=g) * scale).to(types[i % len(types)]).to(dev)
            for i, s in enumerate(sizes)]


def _norm(tensors):
    return math.sqrt(math.fsum(float(np.square(f64(t)).sum()) for t in tensors))


LISTS = [[1], [0, 3], [7, 8, 9], [(64,), (8, 64), (8,), (64, 8), (64,)], [8192, 8193, 8191, 1, 16384], [100003, 5, 70000],
         list(range(1, 600)), [(3, 0, 2), (2, 3, 5)], [0, 0], [2500000]]

# eight squares added in float32 (all positive: 8 U of themselves), the norm half of it and its
# own rounding; the factor's sum, quotient and the product a rounding each
E_NORM = 6 * U
E_OUT = E_NORM + 4 * U


@pytest.mark.parametrize("sizes", LISTS)
def test_norm(dev, G, sizes):
    t = _tensors(sizes, 1, dev)
    want = _norm(t)
    got = G.grad_norm(t)
    assert got.shape == () and got.dtype == torch.float32 and got.device == dev
    assert abs(float(got) - want) <= E_NORM * want
    assert torch.equal(got, G.grad_norm(iter(t)))


@pytest.mark.parametrize("types", [TYPES, TYPES[:1], TYPES[1:2], TYPES[2:]])
@pytest.mark.parametrize("sizes", LISTS)
@pytest.mark.parametrize("ratio", [0.25, 4.0])
def test_clip(dev, G, sizes, types, ratio):
    t = _tensors(sizes, 2, dev, types)
    base = [f64(v) for v in t]
    norm = _norm(t)
    most = ratio * norm + (1.0 if norm == 0 else 0.0)
    factor = min(1.0, float(np.float32(most)) / (norm + 1e-6))

    def check(got, out):
        assert abs(float(got) - norm) <= E_NORM * norm
        for o, b in zip(out, base):
            half = half_step(o.dtype)
            assert worst(f64(o), b * factor, (half + E_OUT) * np.abs(b * factor) + tiny(half) + 1e-300) <= 1
    out = [torch.empty_like(v) for v in t]
    check(G.clip_grads(t, most, out=out), out)
    wide = [torch.empty_like(v, dtype=torch.float32) for v in t]
    check(G.clip_grads(t, most, out=wide), wide)
    assert all(np.array_equal(f64(v), b) for v, b in zip(t, base))
    if ratio > 1:
        assert all(torch.equal(o, v) for o, v in zip(out, t))
    check(G.clip_grads(t, most), t)   # in place


def test_a_given_norm(dev, G):
    t = _tensors([1000, 33], 3, dev)
    base = [f64(v) for v in t]
    norm = torch.tensor(8.0, device=dev)
    assert G.clip_grads(t, 2.0, norm=norm, eps=0.0) is norm
    for v, b in zip(t, base):
        half = half_step(v.dtype)
        assert worst(f64(v), b / 4, half * np.abs(b / 4) + tiny(half)) <= 1


@pytest.mark.parametrize("scale", [1e30, 3e37, 1e-25, 1e-38, 1e-42])
def test_squares_that_float32_does_not_hold(dev, G, scale):
    t = _tensors([5000, 17], 4, dev, [torch.float32, torch.bfloat16], 1.0)
    t = [(v.double() * scale).to(v.dtype) for v in t]
    want = _norm(t)
    if want > 3.5e38:   # past float32: its nearest number is infinity; what is scaled by it is finite all the same
        assert float(G.grad_norm(t)) == float("inf")
        out = [torch.empty_like(v) for v in t]
        G.clip_grads(t, 1e38, out=out)
        assert abs(_norm(out) - 1e38) <= 1e38 * half_step(torch.bfloat16)
        return
    assert abs(float(G.grad_norm(t)) - want) <= E_NORM * want + 2.0 ** -149
    mixed = t + _tensors([100], 5, dev)
    assert abs(float(G.grad_norm(mixed)) - _norm(mixed)) <= E_NORM * _norm(mixed)


def test_norms_that_are_not_finite(dev, G):
    for bad in (float("inf"), float("nan")):
        t = _tensors([50, 60], 6, dev, [torch.float32])
        t[1][7] = bad
        norm = G.clip_grads(t, 1.0)
        assert not torch.isfinite(norm) and torch.isnan(norm) == math.isnan(bad)
        assert torch.isnan(t[1][7])
        if math.isinf(bad):   # scaled by 0
            assert not t[0].any() and not t[1][:7].any()
        else:
            assert torch.isnan(t[0]).all()
    t = _tensors([50], 7, dev, [torch.float32])
    base = t[0].clone()
    G.clip_grads(t, float("inf"))
    assert torch.equal(t[0], base)
    zero = [torch.zeros(9, device=dev)]
    assert float(G.clip_grads(zero, 0.0, eps=0.0)) == 0 and not zero[0].any()
    G.clip_grads(t, 0.0)
    assert not t[0].any()


def test_shared_memory_is_refused(dev, G):
    a, b = _tensors([100, 100], 8, dev, [torch.float32])
    whole = torch.zeros(300, device=dev)
    for tensors, out in (([a, a], None), ([a, b], [b, whole[:100]]), ([whole[:100], whole[50:150]], None),
                         ([whole[:200], whole[:50]], [whole[:200], a[:50]])):
        with pytest.raises(RuntimeError, match="memory"):
            G.clip_grads(tensors, 1.0, out=out)
    with pytest.raises(RuntimeError, match="memory"):   # the outs share
        G.clip_grads([a, b], 1.0, out=[whole[:100], whole[99:199]])
    with pytest.raises(RuntimeError, match="memory"):   # its own tensor, moved by one
        G.clip_grads([whole[:100]], 1.0, out=[whole[1:101]])
    h = torch.zeros(100, dtype=torch.bfloat16, device=dev)
    with pytest.raises(RuntimeError, match="memory"):   # float32 over its own 16 bits
        G.clip_grads([whole[:50].view(torch.bfloat16)], 1.0, out=[whole[:100]])
    one = torch.ones((), device=dev)
    with pytest.raises(RuntimeError, match="memory"):   # the norm given
        G.clip_grads([a, one], 1.0, norm=one)
    G.clip_grads([one], 1.0, out=[torch.empty_like(one)], norm=one)   # only read
    # read twice, written apart: allowed
    out = [torch.empty_like(a), torch.empty_like(a)]
    norm = G.clip_grads([a, a], 1.0, out=out)
    assert torch.equal(out[0], out[1]) and abs(float(norm) - _norm([a, a])) <= E_NORM * _norm([a, a])
    assert float(G.grad_norm([h, h])) == 0


def test_written_tensors_count_as_changed(dev, G):
    t = _tensors([10], 9, dev, [torch.float32])
    before = t[0]._version
    G.clip_grads(t, 1e-3)
    assert t[0]._version > before
    w = torch.ones(4, device=dev, requires_grad=True)
    with pytest.raises(RuntimeError, match="requires grad"):
        G.clip_grads([w], 1.0)
    with torch.no_grad():
        G.clip_grads([w], 1.0)
    assert abs(float(w.detach().norm()) - 1) < 1e-5


def test_unaligned_gradients(dev, G):
    for dtype in TYPES:
        base = _tensors([20001], 10, dev, [dtype])[0]
        t = [base[1:9000], base[9001:]]
        want = _norm(t)
        out = [torch.empty(v.numel() + 1, dtype=torch.float32, device=dev)[1:] for v in t]
        got = G.clip_grads(t, 0.5 * want, out=out)
        assert abs(float(got) - want) <= E_NORM * want
        for o, v in zip(out, t):
            b = f64(v) * (0.5 * want / (want + 1e-6))
            assert worst(f64(o), b, (U + E_OUT) * np.abs(b) + 1e-300) <= 1
