"""The row operators beside the lattice filter: cases, plain forms and the library's calls.

A row is a pixel's channel vector.  Four operators work on rows on either side
of the filter, where a network learns the filter's features and values:

* ``pack``      a tensor's checkpoint in 8 bits (e4m3 codes, one power-of-two scale per 32
                channels) and back
* ``norm``      root-mean-square norm with the residual's addition, its result optionally in
                8 bits with scales, and its backward pass (``norm_bwd``)
* ``linear``    y = act(x w^T + b) + residual, x plain or in 8 bits, the result optionally
                split in two tensors (the filter's features and values), the pre-activation
                optionally kept in 8 bits
* ``linear_bwd``  its backward pass from the 8-bit checkpoints (or plain tensors)

``own`` selects between the plain forms (elementary torch operations in 32 bits) and the
library's calls.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
BLOCK = 32          # channels that share one scale
S_MIN, S_MAX = -110, 120   # exponents of the scales


def listed():
    return [
        # the 3- to 8-channel values of a 64x64 image, kept for the feature gradient
        {"name": "pack_64x64_c8_fp32", "op": "pack", "rows": 4096, "c": 8, "dtype": "fp32"},
        # one layer's activations of a 512x512 image, kept for the backward pass
        {"name": "pack_512x512_c256_bf16", "op": "pack", "rows": 262144, "c": 256, "dtype": "bf16"},
        # a single row through the norm: latency
        {"name": "norm_1row_c1024_bf16", "op": "norm", "rows": 1, "c": 1024, "dtype": "bf16", "residual": True, "pack": True},
        # the norm before a projection: residual stream of a 512x512 image, result in 8 bits
        {"name": "norm_512x512_c256_bf16", "op": "norm", "rows": 262144, "c": 256, "dtype": "bf16", "residual": True, "pack": True},
        # a ragged image and an odd number of channels
        {"name": "norm_bwd_13x29_c50_fp16", "op": "norm_bwd", "rows": 377, "c": 50, "dtype": "fp16", "grad_h": False},
        # its backward at a training size, the residual stream's gradient added
        {"name": "norm_bwd_512x512_c256_bf16", "op": "norm_bwd", "rows": 262144, "c": 256, "dtype": "bf16", "grad_h": True},
        # one row through a wide projection: the weight is read once, latency and bandwidth
        {"name": "linear_1row_1024_4096_bf16", "op": "linear", "rows": 1, "k": 1024, "n": 4096, "dtype": "bf16", "act": "silu",
         "residual": True, "x8": False, "split": 0, "keep": False, "out32": False},
        # a ragged float32 image projected to the widest features and values (pd 16, vd 8)
        {"name": "linear_13x29_50_24_fp32", "op": "linear", "rows": 377, "k": 50, "n": 24, "dtype": "fp32", "act": "none",
         "residual": False, "x8": False, "split": 16, "keep": False, "out32": True},
        # the headline image: 64 channels in 8 bits to features (pd 5) and values (vd 3) in float32
        {"name": "linear_1024x1024_64_8_x8", "op": "linear", "rows": 1048576, "k": 64, "n": 8, "dtype": "bf16", "act": "none",
         "residual": False, "x8": True, "split": 5, "keep": False, "out32": True},
        # a wide layer: compute-bound, activation and residual in the epilogue, pre-activation kept
        {"name": "linear_32768_1024_4096_bf16", "op": "linear", "rows": 32768, "k": 1024, "n": 4096, "dtype": "bf16", "act": "gelu",
         "residual": True, "x8": False, "split": 0, "keep": True, "out32": False},
        # backward of the projection to features (pd 16) and values (vd 8) of a 512x512 image
        {"name": "linear_bwd_512x512_64_24_x8", "op": "linear_bwd", "rows": 262144, "k": 64, "n": 24, "dtype": "bf16", "act": "none",
         "x8": True, "split": 16, "out32": True},
        # backward of the wide layer from its two 8-bit checkpoints
        {"name": "linear_bwd_32768_1024_4096_x8", "op": "linear_bwd", "rows": 32768, "k": 1024, "n": 4096, "dtype": "bf16",
         "act": "gelu", "x8": True, "split": 0, "out32": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _rows(rng, per_row, most, top=1048576):
    return _log(rng, 1, max(1, min(top, int(most // per_row))))


def draw(rng):
    op = rng.choice(["pack", "norm", "norm_bwd", "linear", "linear", "linear_bwd", "linear_bwd"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("pack", "norm", "norm_bwd"):
        c = _log(rng, 1, 4096)
        if rng.random() < 0.5:
            c = max(8, c // 8 * 8)
        case = {"op": op, "rows": _rows(rng, c, 1 << 26), "c": c, "dtype": dtype}
        if op == "norm":
            case |= {"residual": rng.random() < 0.6, "pack": rng.random() < 0.5}
        if op == "norm_bwd":
            case["grad_h"] = rng.random() < 0.6
        return case
    x8 = rng.random() < 0.5
    if x8 and dtype == "fp16":
        dtype = "bf16"
    k, n = _log(rng, 3, 1024 if dtype == "fp32" else 4096), _log(rng, 2, 1024 if dtype == "fp32" else 4096)
    if rng.random() < 0.6:
        k, n = max(8, k // 8 * 8), max(8, n // 8 * 8)
    act = rng.choice(["none", "relu", "gelu", "silu"])
    split = rng.randrange(1, n) if act == "none" and n <= 64 and rng.random() < 0.6 else 0
    most = min((1 << 27) / max(k, n), 2.7e11 / (4.0 if dtype == "fp32" else 1.0) / (2.0 * k * n))
    case = {"op": op, "rows": _log(rng, 1, max(1, min(1048576, int(most)))), "k": k, "n": n, "dtype": dtype, "act": act}
    if op == "linear":
        keep = act != "none" and rng.random() < 0.5
        return case | {"residual": not split and rng.random() < 0.5, "x8": x8, "split": split, "keep": keep,
                       "out32": dtype == "fp32" or split > 0 or rng.random() < 0.2}
    return case | {"x8": x8, "split": split, "out32": dtype == "fp32" or split > 0}


# ---------------------------------------------------------------- 8-bit rows, plain

def _blocks(x):
    """x [rows, c] as [rows, blocks, 32], zeros behind the last channel."""
    c = x.shape[1]
    return torch.nn.functional.pad(x, (0, -c % BLOCK)).view(x.shape[0], -1, BLOCK)


def _pack(x):
    """Codes [rows, ceil(c/32)*32] and exponents' bytes [rows, ceil(c/32)] of x in 32 bits:
    2^s is the smallest power of two with amax / 2^s <= 448; what is not finite becomes NaN."""
    b = _blocks(x)
    fine = torch.isfinite(b)
    m, e = torch.frexp(torch.where(fine, b.abs(), 0.0).amax(-1, keepdim=True))
    s = torch.where(m > 0, e - 9 + (m > 0.875), S_MIN).clamp(S_MIN, S_MAX)
    q = torch.where(fine, b * torch.exp2(-s.float()), float("nan")).to(torch.float8_e4m3fn)
    return q.view(torch.uint8).reshape(x.shape[0], -1), (s + 127).to(torch.uint8).squeeze(-1)


def _unpack(q, scale, c):
    v = q.view(torch.float8_e4m3fn).float().view(q.shape[0], -1, BLOCK)
    return (v * torch.exp2(scale.float() - 127.0).unsqueeze(-1)).reshape(q.shape[0], -1)[:, :c]


def _down(x, dtype):
    """Rounded to dtype; what 16 bits of fp16 cannot reach becomes their largest value."""
    return x.clamp(-65504.0, 65504.0).to(dtype) if dtype is torch.float16 else x.to(dtype)


# ---------------------------------------------------------------- inputs

def _act(x, gen, dtype):
    """Activations: normal, with channels of different size and rows that are nearly zero."""
    rows, c = x
    v = torch.randn(rows, c, generator=gen, device="cuda", dtype=torch.float32)
    v *= torch.exp(0.5 * torch.randn(c, generator=gen, device="cuda"))
    return v.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + 17)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    rows, dtype, op = case["rows"], DTYPES[case["dtype"]], case["op"]
    state = {"case": case}
    if op == "pack":
        state["x"] = _act((rows, case["c"]), gen, dtype)
    elif op in ("norm", "norm_bwd"):
        c = case["c"]
        state["gain"] = 1.0 + 0.2 * rand(c)
        if op == "norm":
            state["x"] = _act((rows, c), gen, dtype)
            state["residual"] = _act((rows, c), gen, dtype) if case["residual"] else None
        else:
            state["h"] = _act((rows, c), gen, dtype)
            state["rstd"] = torch.rsqrt(state["h"].float().square().mean(1) + EPS)
            state["grad"] = rand(rows, c).to(dtype)
            state["grad_h"] = rand(rows, c).to(dtype) if case["grad_h"] else None
    else:
        k, n = case["k"], case["n"]
        state["w"] = (rand(n, k) / math.sqrt(k)).to(dtype)
        x = _act((rows, k), gen, torch.float32 if case["x8"] else dtype)
        state["x"] = _pack(x) if case["x8"] else x
        out = torch.float32 if case["out32"] else dtype
        if op == "linear":
            state["b"] = 0.1 * rand(n)
            state["residual"] = rand(rows, n).to(out) if case["residual"] else None
        else:
            cut = case["split"]
            g = rand(rows, n).to(out)
            state["grad"] = (g[:, :cut].contiguous(), g[:, cut:].contiguous()) if cut else g
            state["z"] = _pack(rand(rows, n)) if case["act"] != "none" else None
    return state


# ---------------------------------------------------------------- one pass

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _apply(z, act):
    if act == "relu":
        return z.clamp_min(0.0)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    s = 1.0 / (1.0 + torch.exp(-z))
    return s * (1.0 + z * (1.0 - s))


def _run_plain(st):
    case = st["case"]
    op, dtype = case["op"], DTYPES[case["dtype"]]
    if op == "pack":
        return _down(_unpack(*_pack(st["x"].float()), case["c"]), dtype)
    if op == "norm":
        h = st["x"].float()
        if st["residual"] is not None:
            h = h + st["residual"].float()
        rstd = torch.rsqrt(h.square().mean(1) + EPS)
        y = h * rstd[:, None] * st["gain"]
        y = _down(_unpack(*_pack(y), case["c"]), dtype) if case["pack"] else y.to(dtype)
        return {"y": y, "rstd": rstd} | ({"h": h.to(dtype)} if st["residual"] is not None else {})
    if op == "norm_bwd":
        rstd = st["rstd"][:, None]
        g, xn = st["grad"].float(), st["h"].float() * rstd
        gn = g * st["gain"]
        gx = rstd * (gn - xn * (gn * xn).mean(1, keepdim=True))
        if st["grad_h"] is not None:
            gx = gx + st["grad_h"].float()
        return {"grad_x": gx.to(dtype), "grad_gain": (g * xn).sum(0)}
    w = st["w"].float()
    x = _unpack(*st["x"], case["k"]) if case["x8"] else st["x"].float()
    if op == "linear":
        out = torch.float32 if case["out32"] else dtype
        z = x @ w.t() + st["b"]
        y = _apply(z, case["act"])
        if st["residual"] is not None:
            y = y + st["residual"].float()
        y = y.to(out)
        got = {"y": (y[:, :case["split"]].contiguous(), y[:, case["split"]:].contiguous()) if case["split"] else y}
        if case["keep"]:
            got["z"] = _down(_unpack(*_pack(z), case["n"]), dtype)
        return got
    g = torch.cat(st["grad"], 1).float() if case["split"] else st["grad"].float()
    if case["act"] != "none":
        g = g * _slope(_unpack(*st["z"], case["n"]), case["act"])
    return {"grad_x": (g @ w).to(dtype), "grad_w": (g.t() @ x).to(dtype), "grad_b": g.sum(0)}


def _run_own(st):
    from plattice_pytorch_b200 import rows as R
    case = st["case"]
    op, dtype = case["op"], DTYPES[case["dtype"]]
    if op == "pack":
        return R.unpack8(R.pack8(st["x"]), dtype)
    if op == "norm":
        y, h, rstd = R.rms_norm(st["x"], st["gain"], st["residual"], eps=EPS, pack=case["pack"])
        y = R.unpack8(y, dtype) if case["pack"] else y
        return {"y": y, "rstd": rstd} | ({"h": h} if st["residual"] is not None else {})
    if op == "norm_bwd":
        gx, gg = R.rms_norm_backward(st["grad"], st["h"], st["rstd"], st["gain"], st["grad_h"])
        return {"grad_x": gx, "grad_gain": gg}
    rows, k, n = case["rows"], case["k"], case["n"]
    x = R.Rows8(*st["x"], (rows, k)) if case["x8"] else st["x"]
    if op == "linear":
        y, z = R.linear(x, st["w"], st["b"], act=case["act"], residual=st["residual"], split=case["split"],
                        out_dtype=torch.float32 if case["out32"] else None, keep="8bit" if case["keep"] else None)
        return {"y": y} | ({"z": R.unpack8(z, dtype)} if case["keep"] else {})
    z = R.Rows8(*st["z"], (rows, n)) if st["z"] is not None else None
    gx, gw, gb = R.linear_backward(st["grad"], x, st["w"], z, act=case["act"], bias_dtype=torch.float32)
    return {"grad_x": gx, "grad_w": gw, "grad_b": gb}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    rows, e = case["rows"], DTYPES[case["dtype"]].itemsize
    eight = lambda c: c + -(-c // BLOCK)  # noqa: E731  bytes of a row in 8 bits
    op = case["op"]
    if op == "pack":   # the tensor in, codes and scales out and in again, the tensor out
        return {"bytes": rows * (2 * case["c"] * e + 2 * eight(case["c"])), "flops": rows * 4.0 * case["c"]}
    if op == "norm":
        c = case["c"]
        b = c * e * (2 if case["residual"] else 1) + (c * e if case["residual"] else 0) + 4
        b += 2 * eight(c) + c * e if case["pack"] else c * e
        return {"bytes": rows * b + 4 * c, "flops": rows * 5.0 * c}
    if op == "norm_bwd":
        c = case["c"]
        return {"bytes": rows * (c * e * (4 if case["grad_h"] else 3) + 4) + 8 * c, "flops": rows * 10.0 * c}
    k, n, o = case["k"], case["n"], 4 if case["out32"] else e
    xb = eight(k) if case["x8"] else k * e
    if op == "linear":
        b = rows * (xb + n * o * (2 if case["residual"] else 1)) + n * k * e + 4 * n
        b += rows * (2 * eight(n) + n * e) if case["keep"] else 0
        return {"bytes": b, "flops": 2.0 * rows * k * n}
    b = rows * (xb + n * o + k * e + (eight(n) if case["act"] != "none" else 0)) + 2 * n * k * e + 4 * n
    return {"bytes": b, "flops": 4.0 * rows * k * n}


# ---------------------------------------------------------------- the definition in 64 bits

def _exact8(v):
    """The values that the 8-bit rows of v (float64 [rows, c]) stand for, by the format's
    grid: step 2^(max(exponent, -6) - 3) below 448, ties to even."""
    rows, c = v.shape
    width = -(-c // BLOCK)
    grid = torch.zeros(rows, width * BLOCK, dtype=torch.float64, device=v.device)
    grid[:, :c] = v
    grid = grid.view(rows, width, BLOCK)
    most = grid.abs().amax(2, keepdim=True)
    s = torch.ceil(torch.log2(most.clamp_min(2.0 ** -140) / 448.0))
    s = torch.where(most > 448.0 * torch.pow(2.0, s), s + 1, s)      # log2 rounded the wrong way
    s = torch.where(most <= 448.0 * torch.pow(2.0, s - 1), s - 1, s)
    unit = torch.pow(2.0, s.clamp(S_MIN, S_MAX))
    t = grid / unit
    step = torch.pow(2.0, torch.floor(torch.log2(t.abs().clamp_min(2.0 ** -6))) - 3.0)
    return (torch.round(t / step) * step * unit).view(rows, -1)[:, :c]


def _read8(pair, c):
    """What codes and scales stand for, from the codes' fields."""
    q, scale = pair
    q, e = q.to(torch.int32), scale.to(torch.float64) - 127.0
    field, frac = (q >> 3) & 15, (q & 7).double()
    mag = torch.where(field > 0, (1.0 + frac / 8.0) * torch.pow(2.0, field.double() - 7.0), frac / 512.0)
    mag = torch.where(q >= 128, -mag, mag)
    return (mag.view(q.shape[0], -1, BLOCK) * torch.pow(2.0, e)[:, :, None]).view(q.shape[0], -1)[:, :c]


def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    if op == "pack":
        return _exact8(st["x"].double())
    if op == "norm":
        h = st["x"].double()
        h = h if st["residual"] is None else h.add(st["residual"].double())
        rms = torch.sqrt(torch.linalg.vector_norm(h, dim=1).square() / case["c"] + EPS)
        y = None if case["pack"] else torch.einsum("rc,r,c->rc", h, 1.0 / rms, st["gain"].double())
        return {"y": y, "rstd": 1.0 / rms} | ({"h": h} if st["residual"] is not None else {})
    if op == "norm_bwd":
        h, g, r = st["h"].double(), st["grad"].double(), st["rstd"].double()
        gg = torch.einsum("rc,rc,r->c", g, h, r)
        dot = torch.einsum("rc,c,rc->r", g, st["gain"].double(), h)
        gx = torch.einsum("rc,c,r->rc", g, st["gain"].double(), r) - h * (dot * r.pow(3) / case["c"])[:, None]
        return {"grad_x": gx if st["grad_h"] is None else gx.add(st["grad_h"].double()), "grad_gain": gg}
    x = _read8(st["x"], case["k"]) if case["x8"] else st["x"].double()
    act = {"none": lambda t: t, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}[case["act"]]
    if op == "linear":
        y = act(torch.addmm(st["b"].double(), x, st["w"].double().t()))
        y = y if st["residual"] is None else y.add(st["residual"].double())
        got = {"y": list(y.split([case["split"], case["n"] - case["split"]], 1)) if case["split"] else y}
        return got | ({"z": None} if case["keep"] else {})
    g = torch.hstack(list(st["grad"])).double() if case["split"] else st["grad"].double()
    if case["act"] != "none":
        z = _read8(st["z"], case["n"]).contiguous().requires_grad_(True)
        with torch.enable_grad():
            g, = torch.autograd.grad(act(z), z, g)
    return {"grad_x": g.mm(st["w"].double()), "grad_w": g.t().mm(x), "grad_b": g.sum(0)}
