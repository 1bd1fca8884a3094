"""Embedding, line recurrence, log probabilities and clipping without a GPU: the C entry
points' checks before any CUDA call, and the Python layer's checks of its arguments."""
import ctypes
import os

import numpy as np
import pytest
import torch

import labels_reference as ref
from test_rows_host import rows   # noqa: F401  CPU tensors let through, the library out of reach


@pytest.fixture(scope="module")
def lib():
    from plattice_pytorch_b200 import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libplattice_b200.so not built (python -m plattice_pytorch_b200.build)")
    return _lib.lib()


FAKE = ctypes.c_void_p(256)   # never dereferenced: every call below returns before using it


def test_embed_arguments(lib):
    from plattice_pytorch_b200 import _lib
    bad, ok = _lib.ERR_INVALID, _lib.OK
    good = [FAKE, FAKE, 1, FAKE, 0, 1.0, 10, 5, 8, None]
    for i, v in ((0, None), (1, None), (3, None), (4, 3), (6, -1), (7, 0), (7, 1 << 31), (8, 0), (8, (1 << 21) + 1), (6, 1 << 40),
                 (1, ctypes.c_void_p(260))):
        a = list(good)
        a[i] = v
        assert lib.plattice_embed(*a) == bad, (i, v)
    assert lib.plattice_embed(None, None, 0, None, 0, 1.0, 0, 5, 8, None) == ok
    b = ctypes.c_size_t(0)
    for count, n, c in ((-1, 5, 8), (1 << 31, 5, 8), (10, 0, 8), (10, 5, 0)):
        assert lib.plattice_embed_backward_workspace_size(count, n, c, ctypes.byref(b)) == bad
    assert lib.plattice_embed_backward_workspace_size(10000, 300, 64, ctypes.byref(b)) == ok and b.value >= 10000 * 8
    good = [FAKE, 0, FAKE, 1, FAKE, 1, 1.0, FAKE, b.value, 10000, 300, 64, None]
    for i, v in ((0, None), (1, 3), (2, None), (3, 4), (4, None), (9, 1 << 31), (10, 0), (11, 0)):
        a = list(good)
        a[i] = v
        assert lib.plattice_embed_backward(*a) == bad, (i, v)
    for i, v in ((7, None), (7, ctypes.c_void_p(264)), (8, b.value - 1)):
        a = list(good)
        a[i] = v
        assert lib.plattice_embed_backward(*a) == _lib.ERR_WORKSPACE


def _scan_args(**kw):
    from plattice_pytorch_b200 import _lib
    a = _lib.ScanArgs()
    for n in ("x", "gate", "h", "last", "states", "grad_h", "grad_x", "grad_gate", "grad_state", "workspace"):
        setattr(a, n, 256)
    a.lines, a.steps, a.c, a.workspace_bytes = 4, 100, 8, 1 << 30
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def test_scan_arguments(lib):
    from plattice_pytorch_b200 import _lib
    b = ctypes.c_size_t(0)
    for name in ("plattice_scan", "plattice_scan_backward"):
        f, size = getattr(lib, name), getattr(lib, name + "_workspace_size")
        assert size(_scan_args(), ctypes.byref(b)) == _lib.OK
        for kw in ({"dtype": 3}, {"lines": -1}, {"steps": -1}, {"c": 0}, {"lines": 1 << 30, "steps": 1 << 10}, {"steps": 1 << 40}):
            assert size(_scan_args(**kw), ctypes.byref(b)) == _lib.ERR_INVALID, kw
            assert f(_scan_args(**kw), None) == _lib.ERR_INVALID, kw
        assert f(_scan_args(lines=0), None) == _lib.OK
    for kw in ({"x": None}, {"gate": None}, {"h": None}):
        assert lib.plattice_scan(_scan_args(**kw), None) == _lib.ERR_INVALID, kw
    for kw in ({"x": None}, {"gate": None}, {"states": None}, {"grad_h": None}, {"grad_x": None}, {"grad_gate": None}):
        assert lib.plattice_scan_backward(_scan_args(**kw), None) == _lib.ERR_INVALID, kw
    long = {"lines": 1, "steps": 1 << 20}
    for name in ("plattice_scan", "plattice_scan_backward"):
        assert getattr(lib, name + "_workspace_size")(_scan_args(**long), ctypes.byref(b)) == _lib.OK
        if b.value:   # cut into pieces
            for kw in ({"workspace": None}, {"workspace": 264}, {"workspace_bytes": b.value - 1}):
                assert getattr(lib, name)(_scan_args(**long, **kw), None) == _lib.ERR_WORKSPACE, kw


def _logp_args(**kw):
    from plattice_pytorch_b200 import _lib
    a = _lib.LogProbsArgs()
    for n in ("logits", "labels", "logp", "entropy", "stats", "lse", "top_logp", "top_ids", "grad_logp", "grad_entropy", "grad_lse",
              "grad_logits"):
        setattr(a, n, 256)
    a.rows, a.n, a.top, a.labels_wide = 10, 50, 4, 1
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def test_log_probs_arguments(lib):
    from plattice_pytorch_b200 import _lib
    bad = _lib.ERR_INVALID
    for f in (lib.plattice_log_probs, lib.plattice_log_probs_backward):
        for kw in ({"dtype": 3}, {"rows": -1}, {"n": 0}, {"top": 33}, {"top": -1}, {"n": 3}, {"rows": 1 << 40}, {"logits": None},
                   {"stats": None}, {"stats": 260}, {"labels": 260}, {"labels": None}):
            assert f(_logp_args(**kw), None) == bad, kw
        assert f(_logp_args(rows=0), None) == _lib.OK
    for kw in ({"top_logp": None}, {"top_ids": None}):
        assert lib.plattice_log_probs(_logp_args(**kw), None) == bad
    for kw in ({"entropy": None}, {"grad_logits": None}):
        assert lib.plattice_log_probs_backward(_logp_args(**kw), None) == bad


def _grads(*items):
    from plattice_pytorch_b200 import _lib
    table = (_lib.Grad * max(1, len(items)))()
    for q, (g, out, size, dtype, out_dtype) in zip(table, items):
        q.g, q.out, q.size, q.dtype, q.out_dtype = g, out, size, dtype, out_dtype
    return table


def test_clip_arguments(lib):
    from plattice_pytorch_b200 import _lib
    bad, b = _lib.ERR_INVALID, ctypes.c_size_t(0)
    size = lambda *items: lib.plattice_clip_grads_workspace_size(_grads(*items), len(items), ctypes.byref(b))  # noqa: E731
    run = lambda items, most=1.0, eps=0.0, norm_in=None, norm_out=FAKE, ws=FAKE, bytes_=1 << 30: lib.plattice_clip_grads(  # noqa: E731
        _grads(*items), len(items), most, eps, norm_in, norm_out, ws, bytes_, None)
    one = (4096, 4096, 10, 0, 0)
    assert size(one) == _lib.OK and b.value > 0
    assert lib.plattice_clip_grads_workspace_size(None, 1, ctypes.byref(b)) == bad
    for item in ((4096, 4096, 10, 3, 0), (4096, 4096, -1, 0, 0), (None, 4096, 10, 0, 0), (4098, 4098, 10, 0, 0),
                 (4096, 4096, (1 << 40) + 1, 0, 0)):
        assert size(item) == bad and run([item]) == bad, item
    for item in ((4096, 8192, 10, 0, 1), (4096, 8192, 10, 1, 2), (4096, 4096, 10, 1, 0), (4096, 8194, 10, 0, 0)):
        assert run([item]) == bad, item   # out's type and place
    assert run([one, (8192, None, 10, 0, 0)]) == bad             # an out for all or none
    assert run([(4096, None, 10, 0, 0)], norm_out=None) == bad   # nothing wanted
    for most, eps in ((-1.0, 0.0), (float("nan"), 0.0), (1.0, -1.0), (1.0, float("nan"))):
        assert run([one], most, eps) == bad
    for kw in ({"ws": None}, {"bytes_": 8}, {"ws": ctypes.c_void_p(264)}):
        assert run([one], **kw) == _lib.ERR_WORKSPACE, kw


def test_memory_that_clipped_gradients_may_not_share(lib):
    """Against every pair of spans; the refusal comes before any CUDA call, what is
    allowed ends at the missing workspace."""
    from plattice_pytorch_b200 import _lib
    rng = np.random.default_rng(1)
    seen = set()
    for _ in range(4000):
        items = []
        for _ in range(int(rng.integers(1, 5))):
            g, size, dtype = int(4 * rng.integers(1, 40)), int(rng.integers(0, 9)), int(rng.integers(0, 2))
            out_dtype = int(rng.choice([0, dtype]))
            out = g if out_dtype == dtype and rng.random() < 0.5 else int(4 * rng.integers(1, 60))
            if out == g and out_dtype != dtype:
                out += 4
            items.append((g, out, size, dtype, out_dtype))
        span = lambda at, size, dtype: (at, at + size * (2 if dtype else 4))  # noqa: E731
        meet = lambda a, b: max(a[0], b[0]) < min(a[1], b[1])  # noqa: E731
        ins = [span(g, s, t) for g, o, s, t, u in items]
        outs = [span(o, s, u) for g, o, s, t, u in items]
        if not any(s for _, _, s, _, _ in items):
            continue
        outs.append(span(FAKE.value, 1, 0))   # the norm
        items.append((0, FAKE.value, 0, 0, 0))
        ins.append((0, 0))
        shared = any(meet(outs[i], outs[j]) for i in range(len(items)) for j in range(i))
        shared |= any(meet(outs[i], ins[j]) and not (i == j and items[i][0] == items[i][1])
                      for i in range(len(items)) for j in range(len(items)))
        items.pop()
        rc = lib.plattice_clip_grads(_grads(*items), len(items), 1.0, 0.0, None, FAKE, None, 0, None)
        assert rc == (_lib.ERR_INVALID if shared else _lib.ERR_WORKSPACE), (items, shared)
        seen.add(shared)
    assert seen == {True, False}


def test_the_norm_given_may_not_be_written_over(lib):
    from plattice_pytorch_b200 import _lib
    run = lambda norm_in, norm_out, g=4096, out=4096: lib.plattice_clip_grads(  # noqa: E731
        _grads((g, out, 10, 0, 0), (4200, 4200, 0, 0, 0)), 2, 1.0, 0.0, norm_in, norm_out, None, 0, None)
    at = ctypes.c_void_p
    for norm in (4096, 4100, 4132):
        assert run(at(norm), None) == run(at(norm), at(norm)) == run(None, at(norm)) == _lib.ERR_INVALID, norm
        # read as a gradient, too: harmless, but not where it is written
        assert run(None, at(norm), 4096, 8192) == run(at(norm), at(norm), 4096, 8192) == _lib.ERR_INVALID, norm
    for norm in (4092, 4136):
        assert run(None, at(norm)) == _lib.ERR_WORKSPACE


@pytest.fixture
def grads(rows, monkeypatch):   # noqa: F811
    from plattice_pytorch_b200 import grads as G
    for name in ("_check_input", "_call", "_lib_h"):
        monkeypatch.setattr(G, name, getattr(rows, name))
    return G


def test_cpu_tensors_are_refused():
    from plattice_pytorch_b200 import grads as G, rows as R
    x, ids = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: R.embed(ids, x), lambda: R.embed_backward(x, ids, 5), lambda: R.scan(x, x), lambda: R.log_probs(x, ids),
                 lambda: R.scan_backward(x, x, x, x), lambda: G.grad_norm([x]), lambda: G.clip_grads([x], 1.0)):
        with pytest.raises(RuntimeError, match="must be CUDA"):
            call()


def test_python_refusals(rows, grads):   # noqa: F811
    R, G = rows, grads
    x, ids, half = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64), torch.float16
    line, s = torch.zeros(2, 20, 8), torch.zeros(2, 8)
    r = R.LogProbs(torch.zeros(4), torch.zeros(4), torch.zeros(4), torch.zeros(4, 2), None, None)
    for call, text in [
            (lambda: R.embed(ids.float(), x), "int64 or int32"),
            (lambda: R.embed(ids, x.double()), "table"),
            (lambda: R.embed(ids, x[0]), "table"),
            (lambda: R.embed(ids, x.t()), "contiguous"),
            (lambda: R.embed(ids, torch.zeros(0, 3)), "table"),
            (lambda: R.embed(ids, x, float("nan")), "scale"),
            (lambda: R.embed(ids, x, torch.ones(1)), "scale"),
            (lambda: R.embed_backward(x, ids[:3], 5), "ids must be"),
            (lambda: R.embed_backward(x, ids.to(torch.int16), 5), "int64 or int32"),
            (lambda: R.embed_backward(x.double(), ids, 5), "grad_y"),
            (lambda: R.embed_backward(x, ids, 0), "n must be"),
            (lambda: R.embed_backward(x, ids, 5.0), "n must be"),
            (lambda: R.embed_backward(x, ids, 5, float("inf")), "scale"),
            (lambda: R.embed_backward(x, ids, 5, dtype=torch.float64), "dtype"),
            (lambda: R.scan(x[0], x[0]), "steps"),
            (lambda: R.scan(line, line.to(half)), "gate"),
            (lambda: R.scan(line, line[:1]), "gate"),
            (lambda: R.scan(line.double(), line.double()), "x must be"),
            (lambda: R.scan(line, line, s[0]), "state"),
            (lambda: R.scan(line, line, s.to(half)), "state"),
            (lambda: R.scan(line.transpose(0, 1), line), "contiguous"),
            (lambda: R.scan_backward(line, line, line, torch.zeros(2, 1, 8)), "states"),
            (lambda: R.scan_backward(line.to(half), line, line, torch.zeros(2, 2, 8)), "grad_h"),
            (lambda: R.scan_backward(line, line, line, torch.zeros(2, 2, 8), s[:1]), "grad_last"),
            (lambda: R.log_probs(x.double()), "logits"),
            (lambda: R.log_probs(x, ids[:2]), "labels"),
            (lambda: R.log_probs(x, x[:, 0].contiguous()), "int64 or int32"),
            (lambda: R.log_probs(x, ids, top=9), "top"),
            (lambda: R.log_probs(torch.zeros(2, 50), top=33), "top"),
            (lambda: R.log_probs(x, ids, top=-1), "top"),
            (lambda: R.log_probs(x, ids, top=1.0), "top"),
            (lambda: R.log_probs_backward(x, (1, 2), ids), "LogProbs"),
            (lambda: R.log_probs_backward(x, r, None, torch.zeros(4)), "labels are needed"),
            (lambda: R.log_probs_backward(x, r, ids, torch.zeros(3)), "grad_logp"),
            (lambda: R.log_probs_backward(x, r, ids, torch.zeros(4).to(half)), "grad_logp"),
            (lambda: R.log_probs_backward(x, r._replace(stats=torch.zeros(4)), ids, torch.zeros(4)), "stats"),
            (lambda: R.log_probs_backward(x, r._replace(entropy=torch.zeros(3)), ids, None, torch.zeros(4)), "entropy"),
            (lambda: R.log_probs_backward(x, r, ids, None, None, torch.zeros(4, 1)), "grad_lse"),
            (lambda: G.grad_norm(x), "list"),
            (lambda: G.grad_norm([]), "at least one"),
            (lambda: G.grad_norm([x, None]), "must be CUDA"),
            (lambda: G.grad_norm([x, x.double()]), "float32, bfloat16 or float16"),
            (lambda: G.grad_norm([x.t()]), "contiguous"),
            (lambda: G.clip_grads([x], -1.0), "max_norm"),
            (lambda: G.clip_grads([x], float("nan")), "max_norm"),
            (lambda: G.clip_grads([x], torch.ones(())), "max_norm"),
            (lambda: G.clip_grads([x], 1.0, eps=-1.0), "eps"),
            (lambda: G.clip_grads([x], 1.0, out=[]), "out must be"),
            (lambda: G.clip_grads([x], 1.0, out=[x.clone(), x.clone()]), "as many"),
            (lambda: G.clip_grads([x], 1.0, out=[torch.zeros(4, 7)]), "out"),
            (lambda: G.clip_grads([x], 1.0, out=[x.to(half)]), "out"),
            (lambda: G.clip_grads([x], 1.0, norm=torch.ones(1)), "norm"),
            (lambda: G.clip_grads([x.clone().requires_grad_(True)], 1.0), "requires grad"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            call()
    for call in (lambda: R.embed(ids, x), lambda: R.scan(line, line, s), lambda: R.log_probs(x, ids, top=8),
                 lambda: R.log_probs_backward(x, r, ids, torch.zeros(4)), lambda: G.grad_norm([x]), lambda: G.clip_grads([x], 1)):
        with pytest.raises(AssertionError, match="reached"):
            call()


def test_reference_gradients_are_differences():
    """The tests' own definitions against central differences of themselves."""
    rng = np.random.default_rng(2)
    x = rng.normal(size=(5, 7)) * 2
    x[1, 3] = -np.inf
    labels = np.array([0, 2, -1, 6, 3])
    g = rng.normal(size=(3, 5))
    grad, _ = ref.LogProbs(x).backward(labels, *g)

    def loss(v):
        w = ref.LogProbs(v)
        lp = np.where(labels < 0, 0.0, w.logp[np.arange(5), labels])
        return (g[0] * lp + g[1] * w.entropy + g[2] * w.lse).sum()
    for i in range(5):
        for j in range(7):
            if np.isfinite(x[i, j]):
                up, down = x.copy(), x.copy()
                up[i, j] += 1e-5
                down[i, j] -= 1e-5
                assert abs((loss(up) - loss(down)) / 2e-5 - grad[i, j]) < 1e-7
    a, u, s, w, v = rng.uniform(0, 1, (2, 9, 3)), rng.normal(size=(2, 9, 3)), rng.normal(size=(2, 3)), rng.normal(size=(2, 9, 3)), rng.normal(size=(2, 3))
    for blend in (False, True):
        for reverse in (False, True):
            def total(x, a, s):
                h, _, last, _ = ref.scan(x, a, s, blend, reverse)
                return (h * w).sum() + (last * v).sum()
            grads, _ = ref.scan_backward(w, u, a, s, v, blend, reverse)
            base = [u, a, s]
            for k, got in enumerate(grads):
                for at in np.ndindex(got.shape):
                    up, down = [b.copy() for b in base], [b.copy() for b in base]
                    up[k][at] += 1e-4
                    down[k][at] -= 1e-4
                    assert abs((total(*up) - total(*down)) / 2e-4 - got[at]) < 1e-8
