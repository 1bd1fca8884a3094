"""The operators of a network that learns from label maps, as one is made of them: labels in,
the recurrence and the lattice layer in between, log probabilities of labels out, all
gradients clipped together.  Against the float64 definitions, in captured graphs, on other
streams, two calls at once, and of strided gradients."""
import math

import numpy as np
import pytest
import torch

from rows_reference import U, f64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def P():
    import plattice_pytorch_b200 as P
    return P


def _randn(shape, seed, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale


class _Net(torch.nn.Module):
    """Labels [H, W] -> rows -> recurrence along the lines with learned gates -> scores."""

    def __init__(self, P, n, c, classes, seed, lattice=False):
        super().__init__()
        self.P = P
        self.table = torch.nn.Parameter(_randn((n, c), seed))
        self.w_gate = torch.nn.Parameter(_randn((c, c), seed + 1, 1 / math.sqrt(c)))
        self.w_out = torch.nn.Parameter(_randn((classes, c), seed + 2, 1 / math.sqrt(c)))
        self.b_out = torch.nn.Parameter(_randn((classes,), seed + 3, 0.1))
        self.layer = P.PermutoLatticeLayer(c, pd=2, vd=3) if lattice else None

    def forward(self, ids, target):
        P = self.P
        x = P.RowEmbedFunction.apply(ids, self.table, 0.5)
        gate = torch.sigmoid(P.RowLinearFunction.apply(x, self.w_gate, None, None, "none", False))
        h, last = P.RowScanFunction.apply(x, gate, None, True, False)
        if self.layer is not None:
            h = self.layer(h)
        scores = P.RowLinearFunction.apply(h, self.w_out, self.b_out, None, "none", False)
        logp, entropy, lse = P.RowLogProbFunction.apply(scores, target)
        return logp, entropy, lse, last


def _loss(logp, entropy, lse, last):
    return -logp.mean() + 0.1 * entropy.mean() + 1e-3 * lse.square().mean() + 0.01 * last.square().mean()


def test_a_step_against_float64(dev, P):
    """Loss and all gradients of one step, and the clipped gradients, against the same
    network of float64 torch operations under autograd.  Tolerance: float32 products round
    to 2^-24 of their sums of magnitudes, the chain has five products and 30 steps of a
    recurrence whose gates damp; 2e-5 of each gradient's largest value is 300 such units."""
    torch.manual_seed(0)
    net = _Net(P, 9, 24, 7, 1).to(dev)
    rng = np.random.default_rng(2)
    ids = torch.from_numpy(rng.integers(-1, 10, (12, 30))).to(dev)
    target = torch.from_numpy(rng.integers(-1, 7, (12, 30)).astype(np.int32)).to(dev)
    loss = _loss(*net(ids, target))
    loss.backward()

    p64 = {k: v.detach().double().cpu().requires_grad_(True) for k, v in net.named_parameters()}
    i, t = ids.cpu(), target.cpu().long()
    inside = ((i >= 0) & (i < 9))[..., None]
    x = torch.where(inside, p64["table"][i.clamp(0, 8)] * 0.5, 0.0)
    gate = torch.sigmoid(x @ p64["w_gate"].t())
    hs, h = [], torch.zeros(12, 24, dtype=torch.float64)
    for k in range(30):
        h = gate[:, k] * h + (1 - gate[:, k]) * x[:, k]
        hs.append(h)
    scores = torch.stack(hs, 1) @ p64["w_out"].t() + p64["b_out"]
    logs = torch.log_softmax(scores, -1)
    logp = torch.where(t >= 0, logs.gather(-1, t.clamp_min(0)[..., None])[..., 0], 0.0)
    entropy = -(logs.exp() * logs).sum(-1)
    want = _loss(logp, entropy, torch.logsumexp(scores, -1), h)
    want.backward()
    assert abs(float(loss.detach()) - float(want.detach())) <= 2e-6 * (1 + abs(float(want.detach())))
    for name, q in net.named_parameters():
        g = p64[name].grad
        assert float((q.grad.double().cpu() - g).abs().max()) <= 2e-5 * float(g.abs().max()), name

    total = math.sqrt(sum(float(v.grad.square().sum()) for v in p64.values()))
    norm = P.grads.clip_grads([q.grad for q in net.parameters()], 0.5 * total)
    assert abs(float(norm) - total) <= 2e-5 * total
    after = math.sqrt(sum(float(q.grad.double().square().sum()) for q in net.parameters()))
    assert abs(after - 0.5 * total) <= 3e-5 * total


def test_steps_with_the_lattice_layer(dev, P):
    """The chain with the lattice layer in it runs, and its gradients reach every parameter."""
    torch.manual_seed(1)
    net = _Net(P, 5, 16, 6, 3, lattice=True).to(dev)
    rng = np.random.default_rng(4)
    ids = torch.from_numpy(rng.integers(0, 5, (20, 24))).to(dev)
    target = torch.from_numpy(rng.integers(-1, 6, (20, 24))).to(dev)
    for _ in range(2):
        net.zero_grad()
        _loss(*net(ids, target)).backward()
        norm = P.grads.clip_grads([q.grad for q in net.parameters()], 0.1)
        assert torch.isfinite(norm) and float(norm) > 0.1
        assert all(q.grad.abs().max() > 0 for q in net.parameters())
        assert abs(float(P.grads.grad_norm([q.grad for q in net.parameters()])) - 0.1) < 1e-4
        with torch.no_grad():
            for q in net.parameters():
                q -= 0.1 * q.grad


def _calls(P, dev, seed):
    """A call of each operator on inputs of its own: a function that makes them all, as a flat list."""
    R, G = P.rows, P.grads
    ids = torch.from_numpy(np.random.default_rng(seed).integers(-1, 40, 20000)).to(dev)
    table, gy = _randn((40, 32), seed).to(dev), _randn((20000, 32), seed + 1).bfloat16().to(dev)
    big = torch.from_numpy(np.random.default_rng(seed).integers(0, 5000, 9000)).to(dev)
    x, a = _randn((2, 3000, 16), seed + 2).to(dev), torch.sigmoid(_randn((2, 3000, 16), seed + 3)).to(dev)
    g = _randn((2, 3000, 16), seed + 4).to(dev)
    scores = [_randn((rows, n), seed + 5).to(dev) for rows, n in ((300, 21), (100, 700), (9, 9000), (2, 60000))]
    labels = [torch.arange(s.shape[0], device=dev) for s in scores]
    grads = [_randn((n,), seed + 6 + n).to(dev) for n in (5, 1000, 300000)]
    out = [torch.empty_like(v) for v in grads]

    def run():
        got = [R.embed(ids, table, 2.0), R.embed_backward(gy, ids, 40), R.embed_backward(gy[:9000], big, 5000),
               R.embed_backward(gy[:500], big[:500], 5000)]
        h, last, states = R.scan(x, a, keep=True)
        got += [h, last, *R.scan_backward(g, x, a, states)]
        for s, l in zip(scores, labels):
            r = R.log_probs(s, l, top=3)
            got += [*r, R.log_probs_backward(s, r, l, r.logp, r.entropy, r.lse)]
        got += [G.clip_grads(grads, 1.0, out=out), G.clip_grads(grads[:2], 1.0, out=out[:2])]
        return got + [o.clone() for o in out]
    return run


def test_repeated_calls_give_the_same_bits(dev, P):
    run = _calls(P, dev, 10)
    first = run()
    for _ in range(3):
        for a, b in zip(first, run()):
            assert torch.equal(a, b)


def test_captured_and_replayed(dev, P):
    """One graph holds a call of each; replays on new inputs in the same memory give what
    eager calls give."""
    run = _calls(P, dev, 20)
    run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = run()
    want = run()
    for v in got:
        v.zero_()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_two_graphs_side_by_side(dev, P):
    """Two captured graphs with workspaces of their own, replayed on two streams at once."""
    runs = [_calls(P, dev, seed) for seed in (30, 40)]
    wants = [run() for run in runs]
    graphs, gots = [], []
    for run in runs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            gots.append(run())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for got, want in zip(gots, wants):
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_two_streams_at_once(dev, P):
    runs = [_calls(P, dev, seed) for seed in (50, 60)]
    wants = [run() for run in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    gots = []
    for stream, run in zip(streams, runs):
        with torch.cuda.stream(stream):
            gots.append([run() for _ in range(3)])
    torch.cuda.synchronize()
    for got, want in zip(gots, wants):
        for one in got:
            for a, b in zip(one, want):
                assert torch.equal(a, b)


def test_calls_synchronise_with_nothing(dev, P):
    """No call waits for the GPU: with synchronising calls made errors by torch, and capture
    (which refuses them) tested above."""
    run = _calls(P, dev, 70)
    run()
    torch.cuda.set_sync_debug_mode("error")
    try:
        run()
    finally:
        torch.cuda.set_sync_debug_mode("default")


def test_without_the_extension(dev, P, monkeypatch):
    """The calls through ctypes give the same bits."""
    run = _calls(P, dev, 80)
    want = run()
    monkeypatch.setattr(P.rows, "_EXT", None)
    monkeypatch.setattr(P.grads, "_cpp", lambda: None)
    for a, b in zip(run(), want):
        assert torch.equal(a, b)


def test_messages_name_the_argument(dev, P):
    """What the extension passes over gets its message from the checks."""
    R, G = P.rows, P.grads
    x, ids = torch.zeros(4, 8, device=dev), torch.zeros(4, dtype=torch.int64, device=dev)
    for call, text in [(lambda: R.embed(ids.short(), x), "int64 or int32"), (lambda: R.embed(ids, x, float("inf")), "scale"),
                       (lambda: R.embed_backward(x, ids[:2], 5), "ids must be"), (lambda: R.scan(x[None], x[None, :2]), "gate"),
                       (lambda: R.scan(x[None], x[None], x[:1, :7].contiguous()), "state"), (lambda: R.log_probs(x, ids, top=9), "top"),
                       (lambda: R.log_probs(x, ids.cpu()), "must be CUDA"), (lambda: G.clip_grads([x], -2.0), "max_norm"),
                       (lambda: G.clip_grads([x], 1.0, out=[x.double()]), "out"), (lambda: G.grad_norm([x, x.t()]), "contiguous")]:
        with pytest.raises(RuntimeError, match=text):
            call()


def test_shapes_of_leading_dimensions(dev, P):
    """Any number of leading dimensions, none among them; empty ones give empty results."""
    R = P.rows
    x = _randn((2, 3, 4, 5), 90).to(dev)
    flat = R.log_probs(x.view(24, 5), torch.zeros(24, dtype=torch.int64, device=dev), top=2)
    deep = R.log_probs(x, torch.zeros(2, 3, 4, dtype=torch.int64, device=dev), top=2)
    for a, b in zip(flat, deep):
        assert torch.equal(a, b.reshape(a.shape))
    one = R.log_probs(x[0, 0, 0].contiguous(), torch.tensor(3, device=dev))
    assert one.logp.shape == () and torch.isfinite(one.logp)
    none = R.log_probs(x[:0], torch.zeros(0, 3, 4, dtype=torch.int64, device=dev), top=2)
    assert none.top_ids.shape == (0, 3, 4, 2)
    assert R.log_probs_backward(x[:0], none, grad_entropy=none.entropy).shape == (0, 3, 4, 5)
    h, last, states = R.scan(x, x, keep=True)
    h2, last2, _ = R.scan(x.view(6, 4, 5), x.view(6, 4, 5))
    assert torch.equal(h.view(6, 4, 5), h2) and states.shape == (2, 3, 1, 5) and last.shape == (2, 3, 5)
    assert torch.equal(last.view(6, 5), last2)
    line, _, _ = R.scan(x[0, 0].contiguous(), x[0, 0].contiguous())
    assert torch.equal(line, h[0, 0])
    assert R.embed_backward(x[:0], torch.zeros(0, 3, 4, dtype=torch.int64, device=dev), 7).count_nonzero() == 0


def test_backward_of_expanded_gradients(dev, P):
    """Gradients that autograd hands on without memory of their own (a sum's, a mean's)."""
    table = _randn((6, 10), 95).to(dev).requires_grad_(True)
    ids = torch.arange(6, device=dev).view(2, 3)
    x = P.RowEmbedFunction.apply(ids, table, 1.0)
    gate = torch.full_like(x, 0.5).requires_grad_(True)
    h, last = P.RowScanFunction.apply(x, gate, None, False, False)
    (h.sum() + last.mean()).backward()
    _, _, states = P.rows.scan(x.detach(), gate.detach(), keep=True)
    gx, ga, _ = P.rows.scan_backward(torch.ones_like(x), x.detach(), gate.detach(), states, torch.full_like(last, 1 / last.numel()).detach())
    assert torch.equal(gate.grad, ga) and torch.equal(table.grad, gx.view(6, 10))


def test_long_sums_and_many_rows(dev, P):
    """Sizes at which counts pass 16 bits: one label for 300000 rows, 70000 single rows of a
    few classes, lines of 70000 steps of ones (their sum is the step's number, exact in float32)."""
    R = P.rows
    g = torch.ones(300000, 3, device=dev)
    ids = torch.full((300000,), 2, device=dev)
    for n in (4, 4000):
        got = R.embed_backward(g, ids, n)
        assert (got[2] == 300000).all() and got.count_nonzero() == 3
    ones = torch.ones(1, 70000, 2, device=dev)
    h, last, states = R.scan(ones, ones, keep=True)
    assert torch.equal(h[0, :, 0], torch.arange(1.0, 70001, device=dev)) and (last == 70000).all()
    gx, ga, gs = R.scan_backward(ones, ones, ones, states)
    assert torch.equal(gx[0, :, 1], torch.arange(70000.0, 0, -1, device=dev)) and (gs == 70000).all()
    r = R.log_probs(torch.zeros(70000, 2, device=dev), torch.ones(70000, dtype=torch.int32, device=dev), top=2)
    assert (f64(r.logp) - math.log(0.5)).max() < 4 * U and (r.top_ids == torch.arange(2, device=dev)).all()
