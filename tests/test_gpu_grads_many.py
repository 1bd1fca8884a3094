"""Clipping of more gradients than one round of the device takes, and the norm's bits."""
import math

import numpy as np
import pytest
import torch

from labels_reference import tiny
from rows_reference import U, half_step

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
E_NORM = 6 * U   # as in test_gpu_grads.py
E_OUT = E_NORM + 4 * U


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def G():
    from plattice_pytorch_b200 import grads
    return grads


@pytest.mark.parametrize("sizes", [[300000], [1, 200000, 77777], [5000] * 80])
def test_the_norm_does_not_depend_on_what_is_written(dev, G, sizes):
    """grad_norm and clip_grads of the same gradients give the same bits, wherever the
    results lie and of whatever type they are: also of a few values that are not 0, whose
    squares' order shows in the norm."""
    for dtype in TYPES:
        g = torch.Generator(device=dev).manual_seed(1)
        for seed in range(8):
            first, few = seed % 2, seed > 1   # on 16-byte boundaries, or on none
            t = [torch.randn(first + n, generator=g, device=dev).to(dtype)[first:] for n in sizes]
            if few:
                for v in t:
                    v[8:] = 0
            want = G.grad_norm(t)
            for type_ in (dtype, torch.float32):
                for shift in (0, 1):
                    out = [torch.empty(shift + n, dtype=type_, device=dev)[shift:] for n in sizes]
                    assert torch.equal(G.clip_grads(t, 1.0, out=out), want), (dtype, first, type_, shift)
            assert torch.equal(G.clip_grads(t, 1.0), want)


@pytest.mark.parametrize("types", [TYPES, TYPES[:1], TYPES[1:2]])
@pytest.mark.parametrize("ratio", [0.25, 4.0])
def test_more_pieces_than_ctas(dev, G, types, ratio):
    """70 tensors of uneven sizes, some on no 16-byte boundary, 24 million values: CTAs go
    through several pieces, and from one tensor to the next."""
    rng = np.random.default_rng(3)
    sizes = [int(s) for s in np.exp(rng.uniform(np.log(10), np.log(3e6), 69))]
    sizes.append(max(1, 24_000_000 - sum(sizes)))
    g = torch.Generator(device=dev).manual_seed(4)
    shifts = [int(rng.integers(0, 2)) for _ in sizes]
    t = [(0.1 * torch.randn(s + k, generator=g, device=dev)).to(types[i % len(types)])[k:] for i, (s, k) in enumerate(zip(sizes, shifts))]
    norm = math.sqrt(math.fsum(float(v.double().square().sum()) for v in t))
    factor = min(1.0, float(np.float32(ratio * norm)) / (norm + 1e-6))
    base = [v.clone() for v in t]

    def check(got, out):
        assert abs(float(got) - norm) <= E_NORM * norm
        for o, b in zip(out, base):
            half = half_step(o.dtype)
            want = b.double() * factor
            assert bool(((o.double() - want).abs() <= (half + E_OUT) * want.abs() + tiny(half)).all())
    assert abs(float(G.grad_norm(t)) - norm) <= E_NORM * norm
    out = [torch.empty_like(v, dtype=torch.float32) for v in t]
    check(G.clip_grads(t, ratio * norm, out=out), out)
    assert all(torch.equal(v, b) for v, b in zip(t, base))
    check(G.clip_grads(t, ratio * norm), t)
