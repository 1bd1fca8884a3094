"""A graph that holds a call of each label operator, replayed after its inputs have changed
in place: labels, scores, gates and gradients are read when the graph runs."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


class _Calls:
    """Inputs of every operator in memory that stays, `fill` with those of a seed, and the calls."""
    SCORES = ((300, 21), (100, 700), (40, 9000), (9, 40000), (2, 300000))

    def __init__(self, dev):
        new = lambda *s, dtype=torch.float32: torch.empty(s, dtype=dtype, device=dev)  # noqa: E731
        ids = lambda *s: new(*s, dtype=torch.int64)  # noqa: E731
        self.ids, self.big, self.few = ids(20000), ids(40000), ids(900)
        self.table, self.gy = new(30, 32), new(40000, 32, dtype=torch.bfloat16)
        self.x, self.gate, self.g = new(2, 3000, 16), new(2, 3000, 16), new(2, 3000, 16)
        self.state = new(2, 16)
        self.scores = [new(*s) for s in self.SCORES]
        self.labels = [ids(s[0]) for s in self.SCORES]
        self.grads = [new(n) for n in (5, 1000, 300000)]
        self.out = [torch.empty_like(v) for v in self.grads]

    def fill(self, seed):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        for t, n, zipf in ((self.ids, 30, False), (self.big, 3000, True), (self.few, 500, True)):
            v = np.minimum(rng.zipf(1.2 + 0.1 * (seed % 7), len(t)), n + 5) - 2 if zipf else rng.integers(-1, n + 1, len(t))
            t.copy_(torch.from_numpy(v))
        for t in (self.table, self.gy, self.x, self.g, self.state, *self.grads):
            t.copy_(torch.randn(t.shape, generator=g))
        gate = torch.sigmoid(torch.randn(self.gate.shape, generator=g))
        if seed % 2:   # products beyond float32, which go another way
            gate[:, 500:700], gate[:, 700:900] = 0.5, 2.0
        self.gate.copy_(gate)
        for s, l in zip(self.scores, self.labels):
            v = 3 * torch.randn(s.shape, generator=g)
            v[torch.rand(s.shape, generator=g) < 0.1 * (seed % 3)] = float("-inf")
            if seed % 2:
                v[-1] = 0.25   # equal scores
            s.copy_(v)
            l.copy_(torch.randint(-1, s.shape[1] + 1, l.shape, generator=g))

    def run(self, P):
        R, G = P.rows, P.grads
        got = [R.embed(self.ids, self.table, 2.0), R.embed_backward(self.gy[:20000], self.ids, 30),
               R.embed_backward(self.gy, self.big, 3000), R.embed_backward(self.gy[:20000], self.big[:20000], 3000),
               R.embed_backward(self.gy[:900], self.few, 500)]
        for reverse in (False, True):
            h, last, states = R.scan(self.x, self.gate, self.state, reverse=reverse, keep=True)
            got += [h, last, *R.scan_backward(self.g, self.x, self.gate, states, self.state, reverse=reverse)]
        for s, l in zip(self.scores, self.labels):
            r = R.log_probs(s, l, top=4)
            got += [*r, R.log_probs_backward(s, r, l, r.entropy, r.entropy, r.entropy)]
        got += [G.clip_grads(self.grads, 1.0, out=self.out), *(o.clone() for o in self.out)]
        return got


def test_replays_on_other_inputs(dev):
    import plattice_pytorch_b200 as P
    calls = _Calls(dev)
    calls.fill(100)
    calls.run(P)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls.run(P)
    for seed in (101, 102, 103, 100):
        calls.fill(seed)
        want = [v.clone() for v in calls.run(P)]
        for v in got:
            v.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for k, (a, b) in enumerate(zip(got, want)):
            a, b = (torch.nan_to_num(v, nan=1e9) if v.is_floating_point() else v for v in (a, b))
            assert torch.equal(a, b), (seed, k)
