"""The operators of a network that learns from label maps: cases, plain forms and the library's calls.

A row is a pixel's channel vector, a label map one class a pixel.  Four operators stand
beside the filter, the norm and the linear map where such a network is trained and asked:

* ``embed``  rows from labels, scaled; ``embed_train`` also the table's gradient.  A label
             outside the table (the "ignored" of label maps) gives zeros and no gradient
* ``scan``   gated linear recurrence along the lines of rows, h = a h + x or, blended,
             h = a h + (1 - a) x, its state carried in and out; ``scan_train`` also its gradients
* ``logp``   log probabilities of given labels from rows of scores, the rows' entropies and
             the best alternatives; ``logp_train`` also the scores' gradient.  A score of -inf
             is a class that the row may not have; a row with no other has entropy 0 and
             gradient 0
* ``clip``   the norm of all gradients together, and the gradients scaled down to a largest norm

``own`` selects between the plain forms (elementary torch operations in 32 bits, sums over
whole gradients in 64) and the library's calls.
"""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
MOST = 1 << 26   # values of a drawn case


def listed():
    return [
        # the label of one more pixel: latency
        {"name": "embed_1_50000x1024_bf16", "op": "embed", "ids": 1, "n": 50000, "c": 1024, "dtype": "bf16", "wide": True, "zipf": False},
        # training from the headline image's label map: few classes, many pixels each
        {"name": "embed_train_1024x1024_21x64_bf16", "op": "embed_train", "ids": 1048576, "n": 21, "c": 64, "dtype": "bf16",
         "wide": False, "zipf": True},
        # training with a large table whose entries occur with very different frequencies
        {"name": "embed_train_16384_50000x1024_bf16", "op": "embed_train", "ids": 16384, "n": 50000, "c": 1024, "dtype": "bf16",
         "wide": True, "zipf": True},
        # one more step of a recurrence whose state is kept between calls: latency
        {"name": "scan_step_4096_bf16", "op": "scan", "lines": 1, "t": 1, "c": 4096, "dtype": "bf16", "blend": False, "reverse": False, "state": True},
        # one very long line of a few channels
        {"name": "scan_1000003x16_fp32", "op": "scan", "lines": 1, "t": 1000003, "c": 16, "dtype": "fp32", "blend": False, "reverse": False,
         "state": True},
        # edge-aware smoothing along the lines of a 512x512 image, trained
        {"name": "scan_train_512x512x256_bf16", "op": "scan_train", "lines": 512, "t": 512, "c": 256, "dtype": "bf16", "blend": True,
         "reverse": False, "state": False},
        # the answer for one pixel among very many classes, with its alternatives: latency
        {"name": "logp_1x100003_top8_bf16", "op": "logp", "rows": 1, "n": 100003, "dtype": "bf16", "top": 8, "masked": False},
        # the answers for a 512x512 image of 256 classes, some of them closed
        {"name": "logp_512x512_256_top4_fp16", "op": "logp", "rows": 262144, "n": 256, "dtype": "fp16", "top": 4, "masked": True},
        # the loss of the headline image: few classes, an odd number of them
        {"name": "logp_train_1024x1024_21_fp32", "op": "logp_train", "rows": 1048576, "n": 21, "dtype": "fp32", "top": 0, "masked": False},
        # the loss over many classes
        {"name": "logp_train_8192_32768_bf16", "op": "logp_train", "rows": 8192, "n": 32768, "dtype": "bf16", "top": 0, "masked": False},
        # the gradients of one layer around the filter: a few small tensors, latency
        {"name": "clip_5_1352_fp32", "op": "clip", "tensors": 5, "total": 1352, "mix": "fp32", "out32": False, "ratio": 0.5},
        # the gradients of a large network, of odd sizes and two types, to float32 for the update
        {"name": "clip_60_134217728_mixed", "op": "clip", "tensors": 60, "total": 134217728, "mix": "mixed", "out32": True, "ratio": 0.1},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _even(rng, v, step=8):
    """Half of the sizes on whole vectors, the others as they fall."""
    return max(step, v // step * step) if rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(["embed", "embed_train", "embed_train", "scan", "scan_train", "scan_train", "logp", "logp", "logp_train", "clip"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("embed", "embed_train"):
        c = _even(rng, _log(rng, 1, 4096))
        n = _log(rng, 1, min(200000, MOST // c))
        return {"op": op, "ids": _log(rng, 1, min(1048576, MOST // c)), "n": n, "c": c, "dtype": dtype, "wide": rng.random() < 0.5,
                "zipf": rng.random() < 0.6}
    if op in ("scan", "scan_train"):
        c = _even(rng, _log(rng, 1, 4096))
        t = _log(rng, 1, min(1048576, MOST // c))
        return {"op": op, "lines": _log(rng, 1, max(1, min(65536, MOST // (c * t)))), "t": t, "c": c, "dtype": dtype,
                "blend": rng.random() < 0.5, "reverse": rng.random() < 0.3, "state": rng.random() < 0.5}
    if op in ("logp", "logp_train"):
        n = _even(rng, _log(rng, 2, 200000))
        rows = _log(rng, 1, max(1, min(1048576, MOST // n)))
        return {"op": op, "rows": rows, "n": n, "dtype": dtype,
                "top": min(n, rng.choice([0, 1, 3, 8, 20])) if op == "logp" else 0, "masked": rng.random() < 0.5}
    tensors = _log(rng, 1, 60)
    mix = rng.choice(["bf16", "fp16", "fp32", "mixed"])
    return {"op": op, "tensors": tensors, "total": _log(rng, tensors, MOST), "mix": mix, "out32": mix != "fp32" and rng.random() < 0.5,
            "ratio": rng.choice([0.02, 0.5, 3.0])}


def _sizes(case):
    """The tensors' sizes: spread over a factor of a thousand, `total` together."""
    k, total = case["tensors"], case["total"]
    rng = random.Random(1000 * k + total)
    share = [math.exp(rng.uniform(0.0, math.log(1000.0))) for _ in range(k)]
    sizes = [1 + int((total - k) * s / sum(share)) for s in share]
    sizes[0] += total - sum(sizes)
    return sizes


def _types(case):
    names = ["fp32", "bf16", "fp16"] if case["mix"] == "mixed" else [case["mix"]]
    return [DTYPES[names[i % len(names)]] for i in range(case["tensors"])]


# ---------------------------------------------------------------- inputs

def _labels(count, n, gen, zipf, wide, ignored):
    """Labels in 0..n-1, evenly or with frequencies that fall like 1 / rank (in a shuffled
    order); with `ignored` one in fifty is outside."""
    u = torch.rand(count, generator=gen, device="cuda", dtype=torch.float64)
    if zipf:   # the inverse of the distribution's continuous form
        rank = (torch.exp(u * math.log(n + 1.0)) - 1.0).long().clamp(0, n - 1)
        ids = torch.randperm(n, generator=gen, device="cuda")[rank]
    else:
        ids = (u * n).long().clamp(0, n - 1)
    if ignored:
        ids[torch.rand(count, generator=gen, device="cuda") < 0.02] = -1
    return ids if wide else ids.to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + 29)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    op = case["op"]
    state = {"case": case}
    if op == "clip":
        scale = 0.01
        state["grads"] = [(scale * rand(s)).to(t) for s, t in zip(_sizes(case), _types(case))]
        state["max_norm"] = case["ratio"] * scale * math.sqrt(case["total"])
        state["out"] = [torch.empty_like(g, dtype=torch.float32 if case["out32"] else g.dtype) for g in state["grads"]]
        return state
    dtype = DTYPES[case["dtype"]]
    if op in ("embed", "embed_train"):
        state["table"] = rand(case["n"], case["c"]).to(dtype)
        state["ids"] = _labels(case["ids"], case["n"], gen, case["zipf"], case["wide"], case["ids"] > 1)
        state["scale"] = math.sqrt(case["c"])
        if op == "embed_train":
            state["grad"] = rand(case["ids"], case["c"]).to(dtype)
    elif op in ("scan", "scan_train"):
        shape = (case["lines"], case["t"], case["c"])
        gate = torch.sigmoid(1.5 * rand(*shape) + 2.0)
        gate[torch.rand(shape[:2], generator=gen, device="cuda") < 0.002] = 0.0   # where a new segment begins
        state["gate"] = gate.to(dtype)
        state["x"] = rand(*shape).to(dtype)
        state["state"] = rand(case["lines"], case["c"]) if case["state"] else None
        if op == "scan_train":
            state["grad"] = rand(*shape).to(dtype)
            state["grad_last"] = rand(case["lines"], case["c"]) if case["state"] else None
    else:
        rows, n = case["rows"], case["n"]
        x = rand(rows, n)
        x *= 1.0 + 2.0 * torch.rand(rows, 1, generator=gen, device="cuda")
        x += 3.0 * rand(rows, 1)
        if case["masked"]:
            x[torch.rand(rows, n, generator=gen, device="cuda") < 0.05] = -math.inf
            x[torch.rand(rows, generator=gen, device="cuda") < 0.001] = -math.inf
        state["x"] = x.to(dtype)
        state["labels"] = _labels(rows, n, gen, False, True, rows > 1)
        if op == "logp_train":
            state["grad_logp"] = rand(rows)
            state["grad_entropy"] = 0.1 * rand(rows)
    return state


# ---------------------------------------------------------------- one pass

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _recurrence(a, b):
    """h[t] = a[t] h[t-1] + b[t] over dim 1 in 32 bits, from h = 0 before the first: pairs
    of steps joined to ever longer ones."""
    a, b, d = a.clone(), b.clone(), 1
    while d < a.shape[1]:
        b[:, d:] = b[:, d:] + a[:, d:] * b[:, :-d]
        a[:, d:] = a[:, d:] * a[:, :-d]
        d *= 2
    return b


def _scan_plain(st, case):
    dtype = DTYPES[case["dtype"]]
    turn = (lambda v: v.flip(1)) if case["reverse"] else (lambda v: v)
    a, x = turn(st["gate"].float()), turn(st["x"].float())
    b = (1.0 - a) * x if case["blend"] else x
    s0 = torch.zeros_like(a[:, 0]) if st["state"] is None else st["state"]
    h = _recurrence(a, torch.cat([(b[:, :1] + a[:, :1] * s0[:, None]), b[:, 1:]], 1))
    got = {"h": turn(h).to(dtype).contiguous(), "last": h[:, -1].contiguous()}
    if case["op"] == "scan":
        return got
    g = turn(st["grad"].float())
    if st["grad_last"] is not None:
        g = torch.cat([g[:, :-1], g[:, -1:] + st["grad_last"][:, None]], 1)
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    gh = _recurrence(later.flip(1), g.flip(1)).flip(1)
    before = torch.cat([s0[:, None], h[:, :-1]], 1)
    gx = (1.0 - a) * gh if case["blend"] else gh
    ga = gh * (before - x) if case["blend"] else gh * before
    return got | {"grad_x": turn(gx).to(dtype).contiguous(), "grad_gate": turn(ga).to(dtype).contiguous(),
                  "grad_state": a[:, 0] * gh[:, 0]}


def _logp_plain(st, case):
    x, labels, n = st["x"].float(), st["labels"], case["n"]
    most = x.amax(1, keepdim=True)
    empty = most == -math.inf
    d = torch.where(empty, -math.inf, x - torch.where(empty, 0.0, most))
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    logp = d - torch.where(empty, 0.0, torch.log(total))
    p = torch.where(empty, 0.0, e / total)
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(1)
    inside = (labels >= 0) & (labels < n)
    at = torch.where(inside, labels, 0)
    got = {"logp": torch.where(inside, logp.gather(1, at[:, None])[:, 0], 0.0), "entropy": entropy}
    if case["top"]:
        ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :case["top"]]
        got |= {"top_logp": logp.gather(1, ids), "top_ids": ids.contiguous()}
    if case["op"] == "logp":
        return got
    g = torch.where(inside, st["grad_logp"], 0.0)[:, None]
    gx = -p * (g + st["grad_entropy"][:, None] * torch.where(p > 0, logp + entropy[:, None], 0.0))
    gx = torch.where(empty, 0.0, gx.scatter_add(1, at[:, None], g))
    return got | {"grad_x": gx.to(st["x"].dtype)}


def _run_plain(st):
    case = st["case"]
    op = case["op"]
    if op == "clip":
        norm = torch.stack([g.float().square().sum(dtype=torch.float64) for g in st["grads"]]).sum().sqrt()
        factor = (st["max_norm"] / (norm + EPS)).clamp(max=1.0).float()
        return {"norm": norm.float(), "grads": [(g.float() * factor).to(o.dtype) for g, o in zip(st["grads"], st["out"])]}
    if op in ("scan", "scan_train"):
        return _scan_plain(st, case)
    if op in ("logp", "logp_train"):
        return _logp_plain(st, case)
    ids, n, dtype = st["ids"].long(), case["n"], DTYPES[case["dtype"]]
    inside = (ids >= 0) & (ids < n)
    at = torch.where(inside, ids, 0)
    y = torch.where(inside[:, None], st["table"][at].float() * st["scale"], 0.0).to(dtype)
    if op == "embed":
        return y
    g = torch.where(inside[:, None], st["grad"].float(), 0.0)
    grad = torch.zeros(n, case["c"], device="cuda").index_add_(0, at, g)
    return {"y": y, "grad_table": (grad * st["scale"]).to(dtype)}


def _run_own(st):
    from plattice_pytorch_b200 import grads as G, rows as R
    case = st["case"]
    op = case["op"]
    if op == "clip":
        norm = G.clip_grads(st["grads"], st["max_norm"], out=st["out"], eps=EPS)
        return {"norm": norm, "grads": st["out"]}
    if op in ("embed", "embed_train"):
        y = R.embed(st["ids"], st["table"], scale=st["scale"])
        if op == "embed":
            return y
        return {"y": y, "grad_table": R.embed_backward(st["grad"], st["ids"], case["n"], scale=st["scale"])}
    if op in ("scan", "scan_train"):
        h, last, states = R.scan(st["x"], st["gate"], st["state"], blend=case["blend"], reverse=case["reverse"],
                                 keep=op == "scan_train")
        if op == "scan":
            return {"h": h, "last": last}
        gx, ga, gs = R.scan_backward(st["grad"], st["x"], st["gate"], states, st["grad_last"], blend=case["blend"],
                                     reverse=case["reverse"])
        return {"h": h, "last": last, "grad_x": gx, "grad_gate": ga, "grad_state": gs}
    r = R.log_probs(st["x"], st["labels"], top=case["top"])
    got = {"logp": r.logp, "entropy": r.entropy}
    if case["top"]:
        got |= {"top_logp": r.top_logp, "top_ids": r.top_ids}
    if op == "logp":
        return got
    return got | {"grad_x": R.log_probs_backward(st["x"], r, st["labels"], grad_logp=st["grad_logp"],
                                                 grad_entropy=st["grad_entropy"])}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    op = case["op"]
    if op == "clip":   # every gradient read once and written once
        b = sum(s * (t.itemsize + (4 if case["out32"] else t.itemsize)) for s, t in zip(_sizes(case), _types(case)))
        return {"bytes": b + 4, "flops": 3.0 * case["total"]}
    e = DTYPES[case["dtype"]].itemsize
    if op in ("embed", "embed_train"):   # table rows that occur in, rows out; rows' gradients in, the table's out
        count, n, c = case["ids"], case["n"], case["c"]
        b = count * (8 if case["wide"] else 4) + min(count, n) * c * e + count * c * e
        b += count * c * e + n * c * e if op == "embed_train" else 0
        return {"bytes": b, "flops": (2.0 if op == "embed_train" else 1.0) * count * c}
    if op in ("scan", "scan_train"):   # x, gate and the rows' gradients in, h and two gradients out
        values, states = case["lines"] * case["t"] * case["c"], 4 * case["lines"] * case["c"]
        train = op == "scan_train"
        b = values * e * (6 if train else 3) + states * (1 + (1 if case["state"] else 0)) * (2 if train else 1)
        return {"bytes": b, "flops": values * ((10.0 if train else 2.0) + (3.0 if case["blend"] else 0.0))}
    rows, n = case["rows"], case["n"]
    b = rows * (n * e + 16 + 12 * case["top"])
    if op == "logp":
        return {"bytes": b, "flops": rows * 6.0 * n}
    return {"bytes": b + rows * (n * e + 8), "flops": rows * 12.0 * n}


# ---------------------------------------------------------------- the definition in 64 bits

def _in_order(a, b, first):
    """h[t] = a[t] h[t-1] + b[t] over dim 1 from h[-1] = first, step by step: the line is cut
    into about sqrt(t) pieces that take their steps side by side, then their starts in order."""
    lines, t, c = a.shape
    cut = max(1, math.isqrt(t))
    pieces = -(-t // cut)
    whole = lambda v, fill: torch.cat(  # noqa: E731
        [v, v.new_full((lines, pieces * cut - t, c), fill)], 1).view(lines, pieces, cut, c)
    a, b = whole(a, 1.0), whole(b, 0.0)
    from_zero, from_one = torch.zeros_like(b), torch.zeros_like(a)
    h, f = torch.zeros_like(b[:, :, 0]), torch.ones_like(a[:, :, 0])
    for i in range(cut):
        h = a[:, :, i] * h + b[:, :, i]
        f = a[:, :, i] * f
        from_zero[:, :, i], from_one[:, :, i] = h, f
    starts, s = [], first
    for j in range(pieces):
        starts.append(s)
        s = from_one[:, j, -1] * s + from_zero[:, j, -1]
    got = from_zero + from_one * torch.stack(starts, 1)[:, :, None]
    return got.view(lines, pieces * cut, c)[:, :t]


def _scan_exact(st, case):
    back = [1] if case["reverse"] else []
    a, x = torch.flip(st["gate"], back).double(), torch.flip(st["x"], back).double()
    first = a.new_zeros(case["lines"], case["c"]) if st["state"] is None else st["state"].double()
    h = _in_order(a, torch.lerp(x, torch.zeros_like(x), a) if case["blend"] else x, first)
    got = {"h": torch.flip(h, back), "last": h[:, -1]}
    if case["op"] == "scan":
        return got
    g = torch.flip(st["grad"], back).double()
    late = a.new_zeros(case["lines"], case["c"]) if st["grad_last"] is None else st["grad_last"].double()
    # what reaches step t from later ones: r[t] = a[t+1] (g[t+1] + r[t+1]), r at the last step is grad_last
    r = torch.empty_like(a)
    r[:, -1] = late
    if case["t"] > 1:
        up = torch.flip(a[:, 1:], [1])
        r[:, :-1] = torch.flip(_in_order(up, up * torch.flip(g[:, 1:], [1]), late), [1])
    r += g
    del g
    h = torch.roll(h, 1, 1)
    h[:, 0] = first
    gate = r * h.sub_(x) if case["blend"] else r * h
    gx = r - a * r if case["blend"] else r
    return got | {"grad_x": torch.flip(gx, back), "grad_gate": torch.flip(gate, back), "grad_state": r[:, 0] * a[:, 0]}


def _logp_exact(st, case):
    x, labels = st["x"].double(), st["labels"]
    empty = torch.isneginf(x).all(1)
    floor = -1e30   # exp of it beside any score is 0
    x = torch.nan_to_num(x, neginf=floor).requires_grad_(case["op"] == "logp_train")
    with torch.enable_grad():
        logs = torch.log_softmax(x, 1)
        entropy = torch.special.entr(torch.exp(logs)).sum(1) if not x.requires_grad else -(torch.exp(logs) * logs).sum(1)
        ignored = (labels < 0) | (labels >= case["n"])
        picked = torch.where(ignored, 0.0, logs[torch.arange(case["rows"], device="cuda"), labels.masked_fill(ignored, 0)])
        if x.requires_grad:
            gx, = torch.autograd.grad((picked * st["grad_logp"].double() + entropy * st["grad_entropy"].double()).sum(), x)
            gx[empty] = 0.0
    logs, entropy, picked = logs.detach(), entropy.detach().masked_fill(empty, 0.0), picked.detach()
    closed = lambda v: v.masked_fill(v < 0.5 * floor, -math.inf)  # noqa: E731
    got = {"logp": torch.where(empty & ~ignored, -math.inf, closed(picked)), "entropy": entropy}
    if case["top"]:
        order = torch.argsort(st["x"].double(), dim=1, descending=True, stable=True)[:, :case["top"]]
        top = closed(torch.take_along_dim(logs, order, 1))
        got |= {"top_logp": top.masked_fill(empty[:, None], -math.inf), "top_ids": order}
    return got | ({"grad_x": gx} if case["op"] == "logp_train" else {})


def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    if op == "clip":
        norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g.double()).square()) for g in st["grads"]))
        factor = min(1.0, st["max_norm"] / (norm + EPS))
        return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": [g.double().mul_(factor) for g in st["grads"]]}
    if op in ("scan", "scan_train"):
        return _scan_exact(st, case)
    if op in ("logp", "logp_train"):
        return _logp_exact(st, case)
    ids = st["ids"].long()
    ids = torch.where((ids < 0) | (ids >= case["n"]), case["n"], ids)   # the ignored have a row of their own
    table = torch.cat([st["table"].double(), torch.zeros(1, case["c"], dtype=torch.float64, device="cuda")])
    y = torch.index_select(table, 0, ids) * st["scale"]
    if op == "embed":
        return y
    order = torch.argsort(ids, stable=True)
    ends = torch.bincount(ids, minlength=case["n"] + 1).cumsum(0)[:-1]
    sums = st["grad"].double()[order].cumsum(0)
    sums = torch.cat([torch.zeros_like(sums[:1]), sums])[ends]
    return {"y": y, "grad_table": torch.diff(sums, dim=0, prepend=torch.zeros_like(sums[:1])) * st["scale"]}
