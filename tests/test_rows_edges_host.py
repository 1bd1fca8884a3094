"""Row operators without a GPU, at the edges of what their calls take."""
import os
import types

import pytest
import torch

from test_rows_host import rows   # noqa: F401  CPU tensors let through, the library out of reach


def test_half_a_pair_of_gradients_is_refused(rows):   # noqa: F811
    x, w, g = torch.zeros(4, 8), torch.zeros(3, 8), torch.zeros(4, 3)
    for pair in ((g, None), [g, None], (None, g), (g,), (g, g, g)):
        with pytest.raises(RuntimeError, match="grad_y must be a tensor or a pair"):
            rows.linear_backward(pair, x, w)


def test_an_extension_without_the_calls_is_passed_over(monkeypatch):
    import plattice_pytorch_b200 as P
    from plattice_pytorch_b200 import _lib, rows as R
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libplattice_b200.so not built (python -m plattice_pytorch_b200.build)")
    monkeypatch.setattr(P, "_plattice_torch", types.ModuleType("_plattice_torch"), raising=False)
    monkeypatch.setattr(R, "_EXT", R._UNSET)
    assert R._cpp() is None
    with pytest.raises(RuntimeError, match="must be CUDA"):
        R.pack8(torch.zeros(4, 8))
