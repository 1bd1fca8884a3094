"""Numbers that float32 does not hold are refused where a kernel takes a float32: they would
arrive as infinity, whose product with 0 is NaN and whose sum scales everything to 0."""
import ctypes

import pytest
import torch

from test_labels_host import FAKE, _grads, grads, lib   # noqa: F401
from test_rows_host import rows   # noqa: F401

FAR = (1e39, -1e39, 10 ** 400, float("inf"), float("-inf"), float("nan"))


def test_python(rows, grads):   # noqa: F811
    R, G = rows, grads
    x, ids = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    for v in FAR:
        for call in (lambda: R.embed(ids, x, v), lambda: R.embed_backward(x, ids, 5, v)):
            with pytest.raises(RuntimeError, match="scale"):
                call()
        with pytest.raises(RuntimeError, match="eps"):
            G.clip_grads([x], 1.0, eps=v)
        if v != float("inf"):   # of a largest norm: a copy
            with pytest.raises(RuntimeError, match="max_norm"):
                G.clip_grads([x], v)
    for call in (lambda: R.embed(ids, x, 3.4e38), lambda: R.embed_backward(x, ids, 5, -3.4e38), lambda: G.clip_grads([x], 3.4e38),
                 lambda: G.clip_grads([x], float("inf"), eps=3.4e38)):
        with pytest.raises(AssertionError, match="reached"):
            call()


def test_c(lib):   # noqa: F811
    from plattice_pytorch_b200 import _lib
    for v in (1e39, float("inf"), float("nan")):
        v = ctypes.c_float(v).value
        assert lib.plattice_embed(FAKE, FAKE, 1, FAKE, 0, v, 10, 5, 8, None) == _lib.ERR_INVALID
        assert lib.plattice_embed_backward(FAKE, 0, FAKE, 0, FAKE, 1, v, FAKE, 1 << 30, 10000, 300, 64, None) == _lib.ERR_INVALID
        assert lib.plattice_clip_grads(_grads((4096, 8192, 10, 0, 0)), 1, 1.0, v, None, FAKE, FAKE, 1 << 30, None) == _lib.ERR_INVALID
