"""Row operators at the edges of their ranges: gradients far from 1, values
that are not finite or nearly infinite, float32's last bits, mixed types,
largest sizes.  Definitions in float64 as in rows_reference.py; u = 2^-24 is
half a float32 step."""
import numpy as np
import pytest
import torch

from rows_reference import U, f64

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
