"""Row operators without a GPU: the C entry points' checks before any CUDA call,
and the Python layer's checks of its arguments."""
import ctypes
import os

import numpy as np
import pytest
import torch

import rows_reference as ref


@pytest.fixture(scope="module")
def lib():
    from plattice_pytorch_b200 import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libplattice_b200.so not built (python -m plattice_pytorch_b200.build)")
    return _lib.lib()


FAKE = ctypes.c_void_p(256)   # never dereferenced: every call below returns before using it


def test_pack_and_norm_arguments(lib):
    from plattice_pytorch_b200 import _lib
    bad, ok = _lib.ERR_INVALID, _lib.OK
    assert lib.plattice_rows_pack8(FAKE, FAKE, FAKE, 3, 4, 8, None) == bad       # no such type
    assert lib.plattice_rows_pack8(FAKE, FAKE, FAKE, 0, -1, 8, None) == bad
    assert lib.plattice_rows_pack8(FAKE, FAKE, FAKE, 0, 4, 0, None) == bad
    assert lib.plattice_rows_pack8(FAKE, None, FAKE, 0, 4, 8, None) == bad
    assert lib.plattice_rows_pack8(FAKE, FAKE, FAKE, 0, 1 << 40, 64, None) == bad
    assert lib.plattice_rows_pack8(None, None, None, 0, 0, 8, None) == ok        # no rows
    assert lib.plattice_rows_unpack8(FAKE, 4, FAKE, FAKE, 4, 8, None) == bad
    assert lib.plattice_rows_unpack8(FAKE, 1, None, FAKE, 4, 8, None) == bad
    args = [FAKE, None, None, FAKE, FAKE, None, FAKE, 0, 0, 1e-6, 4, 8, None]
    for i, v in ((0, None), (3, None), (4, None), (6, None), (7, 5), (8, -1), (10, -2), (11, 0), (11, 16385)):
        a = list(args)
        a[i] = v
        assert lib.plattice_rms_norm(*a) == bad
    b = ctypes.c_size_t(0)
    assert lib.plattice_rms_norm_backward_workspace_size(1000, 64, ctypes.byref(b)) == ok and b.value >= 64 * 4
    assert lib.plattice_rms_norm_backward_workspace_size(1000, 0, ctypes.byref(b)) == bad
    args = [FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None, FAKE, b.value, 0, 0, 1000, 64, None]
    for i, v in ((0, None), (1, None), (2, None), (3, None), (4, None), (5, None), (7, None), (12, 0)):
        a = list(args)
        a[i] = v
        assert lib.plattice_rms_norm_backward(*a) == bad
    a = list(args)
    a[8] = 255
    assert lib.plattice_rms_norm_backward(*a) == _lib.ERR_WORKSPACE


def _args(**kw):
    from plattice_pytorch_b200 import _lib
    a = _lib.LinearArgs()
    for n in ("x", "w", "y0", "y1", "grad0", "grad1", "grad_x", "grad_w", "grad_bias", "workspace"):
        setattr(a, n, 256)
    a.rows, a.k, a.n, a.workspace_bytes = 100, 64, 24, 1 << 30
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_linear_arguments(lib):
    from plattice_pytorch_b200 import _lib
    b = ctypes.c_size_t(0)
    for fn in ("plattice_linear", "plattice_linear_backward"):
        f, size = getattr(lib, fn), getattr(lib, fn + "_workspace_size")
        assert size(ctypes.byref(_args()), ctypes.byref(b)) == _lib.OK
        for kw in ({"rows": -1}, {"k": 0}, {"n": 0}, {"split": 24}, {"split": -1}, {"dtype": 3}, {"out_dtype": 7},
                   {"bias_dtype": -1}, {"act": 4}, {"dtype": 1, "out_dtype": 2}, {"dtype": 2, "out_dtype": 2, "x_scale": 256},
                   {"split": 5, "act": 1}, {"rows": 1 << 40}):
            assert size(ctypes.byref(_args(**kw)), ctypes.byref(b)) == _lib.ERR_INVALID, kw
            assert f(ctypes.byref(_args(**kw)), None) == _lib.ERR_INVALID, kw
        assert f(ctypes.byref(_args(workspace=None, rows=100000, n=72)), None) == _lib.ERR_WORKSPACE   # float32: parts of x and w
        assert f(ctypes.byref(_args(workspace_bytes=0, rows=100000, n=72)), None) == _lib.ERR_WORKSPACE
        assert f(ctypes.byref(_args(dtype=1, out_dtype=1, x=264, x_scale=256)), None) == _lib.ERR_INVALID   # codes not aligned
    for kw in ({"x": None}, {"w": None}, {"y0": None}, {"split": 5, "y1": None}, {"z": None, "z_scale": 256},
               {"z": 272, "z_scale": 256}, {"split": 5, "residual": 256}):
        assert lib.plattice_linear(ctypes.byref(_args(**kw)), None) == _lib.ERR_INVALID, kw
    for kw in ({"x": None}, {"w": None}, {"grad0": None}, {"split": 5, "grad1": None}, {"act": 2}):
        assert lib.plattice_linear_backward(ctypes.byref(_args(**kw)), None) == _lib.ERR_INVALID, kw
    assert lib.plattice_linear(ctypes.byref(_args(rows=0)), None) == _lib.OK


def test_linear_alignments(lib):
    """Codes and workspaces on the boundaries that the kernels' wide accesses need."""
    from plattice_pytorch_b200 import _lib
    for n in (24, 72):
        assert lib.plattice_linear_backward(ctypes.byref(_args(n=n, act=2, z=264, z_scale=256)), None) == _lib.ERR_INVALID
        assert lib.plattice_linear_backward(ctypes.byref(_args(n=n, workspace=272)), None) == _lib.ERR_WORKSPACE
    assert lib.plattice_linear(ctypes.byref(_args(rows=100000, n=72, workspace=264)), None) == _lib.ERR_WORKSPACE


@pytest.fixture
def rows(monkeypatch):
    """The module with CPU tensors let through its first check and the library out of reach."""
    from plattice_pytorch_b200 import rows as R

    def contiguous(t, name):
        if not isinstance(t, torch.Tensor):
            raise RuntimeError(f"{name} must be CUDA")
        if not t.is_contiguous():
            raise RuntimeError(f"{name} must be contiguous")

    def reached(*a):
        raise AssertionError("the library was reached")
    monkeypatch.setattr(R, "_check_input", contiguous)
    monkeypatch.setattr(R, "_call", reached)
    monkeypatch.setattr(R, "_lib_h", reached)
    return R


def test_cpu_tensors_are_refused():
    from plattice_pytorch_b200 import rows as R
    x, w = torch.zeros(4, 8), torch.zeros(3, 8)
    for call in (lambda: R.pack8(x), lambda: R.rms_norm(x, x[0]), lambda: R.linear(x, w),
                 lambda: R.linear_backward(x, x, w), lambda: R.Rows8(x, x, (4, 8)),
                 lambda: R.rms_norm_backward(x, x, x[:, 0], x[0])):
        with pytest.raises(RuntimeError, match="must be CUDA"):
            call()


def test_python_refusals(rows):
    R = rows
    x, w, g = torch.zeros(4, 8), torch.zeros(3, 8), torch.zeros(8)
    r8 = R.Rows8(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8), (4, 8))
    half = torch.float16
    for call, text in [
            (lambda: R.pack8(x.double()), "float32, bfloat16 or float16"),
            (lambda: R.pack8(x.t()), "contiguous"),
            (lambda: R.pack8(torch.zeros(4, 0)), "channels"),
            (lambda: R.unpack8(x), "Rows8"),
            (lambda: R.unpack8(r8, torch.float64), "dtype"),
            (lambda: R.Rows8(r8.q, r8.scale, (4, 40)), "q must be"),
            (lambda: R.Rows8(r8.q, r8.scale[:3], (4, 8)), "scale must be"),
            (lambda: R.Rows8(r8.q.to(torch.int8), r8.scale, (4, 8)), "uint8"),
            (lambda: R.rms_norm(x, g[:7]), "gain"),
            (lambda: R.rms_norm(x, g.double()), "gain"),
            (lambda: R.rms_norm(x, g, x.to(half)), "residual"),
            (lambda: R.rms_norm(x, g, x[:3]), "residual"),
            (lambda: R.rms_norm(torch.zeros(1, 16385), torch.zeros(16385)), "16384"),
            (lambda: R.rms_norm_backward(x, x, x[:, 0].contiguous()[:2], g), "rstd"),
            (lambda: R.rms_norm_backward(x.to(half), x, torch.zeros(4), g), "grad_y"),
            (lambda: R.rms_norm_backward(x, x, torch.zeros(4), g, x[:1]), "grad_h"),
            (lambda: R.linear(x, w.to(half)), "same type"),
            (lambda: R.linear(x, torch.zeros(3, 7)), "channels"),
            (lambda: R.linear(r8, w.to(half)), "8-bit"),
            (lambda: R.linear(r8, torch.zeros(3, 9)), "channels"),
            (lambda: R.linear(x, w, act="tanh"), "act"),
            (lambda: R.linear(x, w, torch.zeros(4)), "bias"),
            (lambda: R.linear(x, w, residual=torch.zeros(4, 4)), "residual"),
            (lambda: R.linear(x, w, split=3), "split"),
            (lambda: R.linear(x, w, split=1, act="relu"), "split"),
            (lambda: R.linear(x, w, split=1, residual=torch.zeros(4, 3)), "split"),
            (lambda: R.linear(x, w, out_dtype=half), "out_dtype"),
            (lambda: R.linear(x, w, keep="half"), "keep"),
            (lambda: R.linear_backward(torch.zeros(4, 2), x, w), "grad_y"),
            (lambda: R.linear_backward(torch.zeros(4, 3), x, w, act="gelu"), "z is needed"),
            (lambda: R.linear_backward(torch.zeros(4, 3), x, w, torch.zeros(4, 2), act="gelu"), "z must be"),
            (lambda: R.linear_backward(torch.zeros(4, 3), x, w, r8, act="gelu"), "z must be"),
            (lambda: R.linear_backward((torch.zeros(4, 2), torch.zeros(4, 2)), x, w), "grad_y"),
            (lambda: R.linear_backward((torch.zeros(4, 3), torch.zeros(4, 0)), x, w), "grad_y"),
            (lambda: R.linear_backward(torch.zeros(4, 3), x, w, bias_dtype=torch.float64), "bias_dtype"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            call()
    with pytest.raises(AssertionError, match="reached"):
        R.pack8(x)


def test_rows_of_kept_images(rows):
    from plattice_pytorch_b200 import plattice
    for shape, want in (((5, 7, 3), (105,)), ((1 << 14, 1 << 13, 8), (1 << 30,)),
                        ((1 << 14, (1 << 13) + 1, 8), (1 << 14, (1 << 16) + 8))):
        t = torch.empty(shape, device="meta")
        kept = t.view(plattice._long_rows(shape))
        assert tuple(kept.shape) == want
        rows._check_rows(kept, "x")   # what pack8 takes


def test_reference_codes_match_torch():
    """The tests' own e4m3 encoder against torch's conversion, every tie included."""
    v = ref.E4M3[:127]
    t = np.concatenate([v, (v[1:] + v[:-1]) / 2, np.random.default_rng(0).uniform(0, 448, 5000)])
    t = np.concatenate([t, -t])
    want = torch.from_numpy(t).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(ref._encode(torch.from_numpy(t).float().double().numpy()), want)
