"""Pointers off their element's boundary are refused by the C entry points of the label
operators, recurrence, log probabilities and clipping, before any CUDA call."""
import ctypes

import pytest

from test_labels_host import FAKE, _grads, _logp_args, _scan_args, lib   # noqa: F401

at = ctypes.c_void_p


@pytest.mark.parametrize("dtype,off", [(0, 258), (0, 257), (1, 257), (2, 257)])
def test_embed(lib, dtype, off):   # noqa: F811
    from plattice_pytorch_b200 import _lib
    good = [FAKE, FAKE, 1, FAKE, dtype, 1.0, 10, 5, 8, None]
    for i, v in ((0, off), (3, off), (1, 260)):
        a = list(good)
        a[i] = at(v)
        assert lib.plattice_embed(*a) == _lib.ERR_INVALID, (i, v)
    good = [FAKE, dtype, FAKE, dtype, FAKE, 0, 1.0, FAKE, 1 << 30, 10000, 300, 64, None]
    for i, v in ((0, off), (2, off), (4, 258)):
        a = list(good)
        a[i] = at(v)
        assert lib.plattice_embed_backward(*a) == _lib.ERR_INVALID, (i, v)
    a = list(good)
    a[0], a[9] = at(off), 0   # no labels: the table is written all the same
    assert lib.plattice_embed_backward(*a) == _lib.ERR_INVALID


@pytest.mark.parametrize("dtype,off", [(0, 258), (1, 257), (2, 257)])
@pytest.mark.parametrize("steps", [1, 100, 100000])
def test_scan(lib, dtype, off, steps):   # noqa: F811
    from plattice_pytorch_b200 import _lib
    for name, rows, states in (("plattice_scan", ("x", "gate", "h"), ("state", "last", "states")),
                               ("plattice_scan_backward", ("x", "gate", "grad_h", "grad_x", "grad_gate"),
                                ("states", "grad_last", "grad_state"))):
        for field in rows:
            assert getattr(lib, name)(_scan_args(dtype=dtype, steps=steps, **{field: off}), None) == _lib.ERR_INVALID, field
        for field in states:
            assert getattr(lib, name)(_scan_args(dtype=dtype, steps=steps, **{field: 258}), None) == _lib.ERR_INVALID, field


@pytest.mark.parametrize("dtype,off", [(0, 258), (1, 257), (2, 257)])
def test_log_probs(lib, dtype, off):   # noqa: F811
    from plattice_pytorch_b200 import _lib
    for kw in ({"logits": off}, {"stats": 260}, {"logp": 258}, {"entropy": 258}, {"lse": 258}, {"top_logp": 258}, {"top_ids": 260},
               {"labels": 260}, {"labels": 258, "labels_wide": 0}):
        assert lib.plattice_log_probs(_logp_args(dtype=dtype, **kw), None) == _lib.ERR_INVALID, kw
    for kw in ({"logits": off}, {"grad_logits": off}, {"stats": 260}, {"grad_logp": 258}, {"grad_entropy": 258}, {"grad_lse": 258},
               {"entropy": 258}, {"labels": 260}):
        assert lib.plattice_log_probs_backward(_logp_args(dtype=dtype, **kw), None) == _lib.ERR_INVALID, kw


def test_clip(lib):   # noqa: F811
    from plattice_pytorch_b200 import _lib
    run = lambda norm_in, norm_out, out=8192: lib.plattice_clip_grads(  # noqa: E731
        _grads((4096, out, 10, 0, 0)), 1, 1.0, 0.0, norm_in, norm_out, FAKE, 1 << 30, None)
    assert run(at(258), None) == run(None, at(258)) == run(at(257), at(256)) == _lib.ERR_INVALID
    assert run(None, at(258), None) == _lib.ERR_INVALID
