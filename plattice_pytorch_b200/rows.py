"""Operators on rows (a pixel's channels) beside the lattice filter.

A network that learns the filter's features and values has, on either side of
:func:`PLOO.lattice_forward`, a norm of each pixel's channels, a projection of
them to features (1..16) and values (1..8), a projection back with activation
and residual, and activations to keep for the backward pass.  These are the
library's calls for that, without autograd (``plattice.py`` has the autograd
Functions and the module that chains them):

* :func:`pack8` / :func:`unpack8` -- a tensor in 8 bits (:class:`Rows8`): e4m3
  codes with one power-of-two scale per 32 channels, a quarter to an eighth of
  float32's bytes (1.03 bytes per value), off by at most 2^-4 of a value
  or, for values far below their block's largest, 2^-17 of that largest.
* :func:`rms_norm` / :func:`rms_norm_backward` -- with the residual's addition;
  the result optionally as Rows8.
* :func:`linear` / :func:`linear_backward` -- ``act(x w^T + b) + residual`` with
  ``x`` a tensor or Rows8; the backward reads the same Rows8 that the forward
  read, and the pre-activation from Rows8 too.

* :func:`embed` / :func:`embed_backward` -- rows from a label map, and the
  gradient of the table they come from.
* :func:`scan` / :func:`scan_backward` -- a gated linear recurrence along the
  lines of rows (an image's lines: edge-aware smoothing with learned gates).
* :func:`log_probs` / :func:`log_probs_backward` -- from rows of scores the log
  probabilities of given labels, the entropies and the best alternatives.

Tensors are contiguous CUDA tensors ``[..., channels]`` of float32, bfloat16
or float16; as for the filter, a failed check raises RuntimeError, kernels run
on PyTorch's current stream of the tensors' device, and no call synchronises.
No reference counterpart.
"""
import collections
import ctypes

import torch

from . import _lib
from .PLOO import _call, _check_input, _lib_h, _raise, _raw_stream, _require

__all__ = ["Rows8", "pack8", "unpack8", "rms_norm", "rms_norm_backward", "linear", "linear_backward", "ACTIVATIONS",
           "embed", "embed_backward", "scan", "scan_backward", "LogProbs", "log_probs", "log_probs_backward"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
_KEEP = {None: 0, "8bit": 1, "full": 2}
_MAX_NORM = 16384
_MAX_CHANNELS = 1 << 30
_MAX_EMBED = 1 << 21
_MAX_TOP = 32
_SCAN_KEEP = 16   # steps between the states that a scan keeps
_MOST = torch.finfo(torch.float32).max


def _width8(c):
    return (c + 31) // 32 * 32


class Rows8:
    """A tensor ``[..., c]`` in 8 bits: ``q`` uint8 ``[rows, width]`` (e4m3
    codes, ``width`` = c rounded up to 32, zeros behind the last channel) and
    ``scale`` uint8 ``[rows, width / 32]``; channel i of a row stands for
    ``q[i] * 2^(scale[i // 32] - 127)``.  ``shape`` is the tensor's shape."""

    __slots__ = ("q", "scale", "shape")

    def __init__(self, q, scale, shape):
        shape = tuple(int(s) for s in shape)
        _check_input(q, "q")
        _check_input(scale, "scale")
        _require(q.dtype == torch.uint8 and scale.dtype == torch.uint8, "q and scale must be uint8")
        _require(len(shape) >= 1 and min(shape) >= 0 and 1 <= shape[-1] <= _MAX_CHANNELS,
                 "shape must be [..., c] with 1 <= c <= 2^30")
        rows, width = _rows_of(shape), _width8(shape[-1])
        _require(tuple(q.shape) == (rows, width), f"q must be [{rows}, {width}] for shape {shape}")
        _require(tuple(scale.shape) == (rows, width // 32), f"scale must be [{rows}, {width // 32}] for shape {shape}")
        _require(q.device == scale.device, "q and scale must be on the same device")
        _require(q.data_ptr() % 16 == 0, "q must be 16-byte aligned")
        self.q, self.scale, self.shape = q, scale, shape

    @property
    def device(self):
        return self.q.device


def _rows_of(shape):
    n = 1
    for s in shape[:-1]:
        n *= int(s)
    return n


def _empty8(shape, device):
    rows, width = _rows_of(shape), _width8(int(shape[-1]))
    return _made8(torch.empty((rows, width), dtype=torch.uint8, device=device),
                  torch.empty((rows, width // 32), dtype=torch.uint8, device=device), tuple(int(s) for s in shape))


def _check_rows(t, name, channels=None):
    _check_input(t, name)
    _require(t.dtype in _DTYPES, f"{name} must be float32, bfloat16 or float16")
    _require(t.dim() >= 1 and 1 <= t.shape[-1] <= _MAX_CHANNELS, f"{name} must be [..., channels], at most 2^30")
    _require(channels is None or int(t.shape[-1]) == channels, f"{name} must have {channels} channels")


def _check_like(t, name, shape, dtype, device):
    _check_input(t, name)
    _require(tuple(t.shape) == tuple(shape), f"{name} must be {tuple(shape)}")
    _require(t.dtype == dtype, f"{name} must be {str(dtype)[6:]}")
    _require(t.device == device, f"{name} must be on the rows' device")


def _check_param(t, name, n, device):
    _check_input(t, name)
    _require(tuple(t.shape) == (n,), f"{name} must be [{n}]")
    _require(t.dtype in _DTYPES, f"{name} must be float32, bfloat16 or float16")
    _require(t.device == device, f"{name} must be on the rows' device")


def _ptr(t):
    return None if t is None else t.data_ptr()


_UNSET = object()
_EXT = _UNSET
_CALLS = ("plattice_rows_pack8", "plattice_rows_unpack8", "plattice_rms_norm",
          "plattice_rms_norm_backward_workspace_size", "plattice_rms_norm_backward", "plattice_linear_workspace_size",
          "plattice_linear", "plattice_linear_backward_workspace_size", "plattice_linear_backward")
_MORE_CALLS = ("plattice_embed", "plattice_embed_backward_workspace_size", "plattice_embed_backward",
               "plattice_scan_workspace_size", "plattice_scan", "plattice_scan_backward_workspace_size",
               "plattice_scan_backward", "plattice_log_probs", "plattice_log_probs_backward",
               "plattice_clip_grads_workspace_size", "plattice_clip_grads")


def _cpp():
    """The torch extension's forms of the calls below (the same tests,
    allocations and library calls in one step), pointed at the loaded library;
    None when the extension is not built, or from older sources.  They answer None to arguments that
    fail a test: the Python form then finds which and raises its message."""
    global _EXT
    if _EXT is _UNSET:
        try:
            from . import _plattice_torch as m
            at = lambda names: [ctypes.cast(getattr(_lib.lib(), n), ctypes.c_void_p).value for n in names]  # noqa: E731
            m.set_rows_entry_points(at(_CALLS))
            m.set_more_entry_points(at(_MORE_CALLS))
            _EXT = m
        except (ImportError, AttributeError):   # AttributeError: built before these calls
            _EXT = None
    return _EXT


def _made8(q, scale, shape):
    r = Rows8.__new__(Rows8)   # made by the library to the format: nothing to check
    r.q, r.scale, r.shape = q, scale, shape
    return r


# ---------------------------------------------------------------- 8-bit rows

def pack8(x):
    """``x [..., c]`` in 8 bits, as :class:`Rows8`.  What is not finite comes
    back as NaN; its neighbours keep their values."""
    cpp = _cpp()
    if cpp is not None and (got := cpp.rows_pack8(x)) is not None:
        if type(got) is int:
            _raise("plattice_rows_pack8", got, f"shape={tuple(x.shape)}")
        return _made8(*got, tuple(x.shape))
    _check_rows(x, "x")
    r = _empty8(x.shape, x.device)
    rc = _call(x.device.index, _lib_h().plattice_rows_pack8, r.q.data_ptr(), r.scale.data_ptr(), x.data_ptr(),
               _DTYPES[x.dtype], r.q.shape[0], x.shape[-1], _raw_stream(x.device.index))
    if rc:
        _raise("plattice_rows_pack8", rc, f"shape={tuple(x.shape)}")
    return r


def unpack8(r, dtype=torch.float32):
    """The tensor ``[..., c]`` that ``r`` stands for (exact in float32 and
    bfloat16; in float16 rounded, and at most 65504)."""
    _require(isinstance(r, Rows8), "r must be Rows8")
    _require(dtype in _DTYPES, "dtype must be float32, bfloat16 or float16")
    cpp = _cpp()
    if cpp is not None and (got := cpp.rows_unpack8(r.q, r.scale, r.shape, _DTYPES[dtype])) is not None:
        if type(got) is int:
            _raise("plattice_rows_unpack8", got, f"shape={r.shape}")
        return got
    r = Rows8(r.q, r.scale, r.shape)   # its fields may have been changed since it was made
    y = torch.empty(r.shape, dtype=dtype, device=r.device)
    rc = _call(r.device.index, _lib_h().plattice_rows_unpack8, y.data_ptr(), _DTYPES[dtype], r.q.data_ptr(),
               r.scale.data_ptr(), r.q.shape[0], r.shape[-1], _raw_stream(r.device.index))
    if rc:
        _raise("plattice_rows_unpack8", rc, f"shape={r.shape}")
    return y


# ---------------------------------------------------------------- the norm

def rms_norm(x, gain, residual=None, eps=1e-6, pack=False):
    """Root-mean-square norm of ``h = x + residual``: ``(y, h, rstd)`` with
    ``rstd [...] = (mean h^2 + eps)^-1/2`` (float32) and ``y = h rstd gain``, in
    the type of ``x`` or, with ``pack``, as :class:`Rows8`.  ``h`` is ``x``
    itself without a residual.  ``gain [c]`` of any of the three types."""
    cpp = _cpp()
    if cpp is not None and (got := cpp.rows_rms_norm(x, gain, residual, eps, pack)) is not None:
        if type(got) is int:
            _raise("plattice_rms_norm", got, f"shape={tuple(x.shape)}")
        return (_made8(*got[0], tuple(x.shape)), got[1], got[2]) if pack else got
    _check_rows(x, "x")
    c, dev = int(x.shape[-1]), x.device
    _require(c <= _MAX_NORM, f"x must have at most {_MAX_NORM} channels")
    _check_param(gain, "gain", c, dev)
    if residual is not None:
        _check_like(residual, "residual", x.shape, x.dtype, dev)
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    h = x if residual is None else torch.empty_like(x)
    y = _empty8(x.shape, dev) if pack else torch.empty_like(x)
    rc = _call(dev.index, _lib_h().plattice_rms_norm, (y.q if pack else y).data_ptr(), _ptr(y.scale) if pack else None,
               None if residual is None else h.data_ptr(), rstd.data_ptr(), x.data_ptr(), _ptr(residual),
               gain.data_ptr(), _DTYPES[x.dtype], _DTYPES[gain.dtype], float(eps), rstd.numel(), c,
               _raw_stream(dev.index))
    if rc:
        _raise("plattice_rms_norm", rc, f"shape={tuple(x.shape)}")
    return y, h, rstd


_NORM_WS = {}


def rms_norm_backward(grad_y, h, rstd, gain, grad_h=None):
    """Gradients of :func:`rms_norm` from its ``h`` and ``rstd``: ``(grad_x,
    grad_gain)``; ``grad_x`` is the gradient of ``x`` and of the residual, with
    ``grad_h`` (the gradient that reaches ``h`` from elsewhere) added."""
    cpp = _cpp()
    if cpp is not None and (got := cpp.rows_rms_norm_backward(grad_y, h, rstd, gain, grad_h)) is not None:
        if type(got) is int:
            _raise("plattice_rms_norm_backward", got, f"shape={tuple(h.shape)}")
        return got
    _check_rows(h, "h")
    c, dev = int(h.shape[-1]), h.device
    _require(c <= _MAX_NORM, f"h must have at most {_MAX_NORM} channels")
    _check_like(grad_y, "grad_y", h.shape, h.dtype, dev)
    _check_like(rstd, "rstd", h.shape[:-1], torch.float32, dev)
    _check_param(gain, "gain", c, dev)
    if grad_h is not None:
        _check_like(grad_h, "grad_h", h.shape, h.dtype, dev)
    rows = rstd.numel()
    wsb = _NORM_WS.get((rows, c))
    if wsb is None:
        b = ctypes.c_size_t(0)
        rc = _lib_h().plattice_rms_norm_backward_workspace_size(rows, c, ctypes.byref(b))
        if rc:
            _raise("plattice_rms_norm_backward_workspace_size", rc, f"shape={tuple(h.shape)}")
        wsb = _NORM_WS[(rows, c)] = b.value
    grad_x = torch.empty_like(h)
    grad_gain = torch.empty_like(gain)
    ws = torch.empty(wsb, dtype=torch.uint8, device=dev)
    rc = _call(dev.index, _lib_h().plattice_rms_norm_backward, grad_x.data_ptr(), grad_gain.data_ptr(),
               grad_y.data_ptr(), h.data_ptr(), rstd.data_ptr(), gain.data_ptr(), _ptr(grad_h), ws.data_ptr(), wsb,
               _DTYPES[h.dtype], _DTYPES[gain.dtype], rows, c, _raw_stream(dev.index))
    if rc:
        _raise("plattice_rms_norm_backward", rc, f"shape={tuple(h.shape)}")
    return grad_x, grad_gain


# ---------------------------------------------------------------- the linear map

def _linear_common(x, weight, act, out_dtype, lead=None):
    """Checked (args struct, shape before the channels, out dtype, device) of a
    linear call; ``lead`` is that shape where ``x`` is None."""
    _check_input(weight, "weight")
    _require(weight.dtype in _DTYPES, "weight must be float32, bfloat16 or float16")
    _require(weight.dim() == 2 and 1 <= weight.shape[0] <= _MAX_CHANNELS and 1 <= weight.shape[1] <= _MAX_CHANNELS,
             "weight must be [n, k], each at most 2^30")
    n, k = (int(s) for s in weight.shape)
    if isinstance(x, Rows8):
        _require(weight.dtype != torch.float16, "weight must be float32 or bfloat16 for 8-bit rows")
        x = Rows8(x.q, x.scale, x.shape)
        _require(x.shape[-1] == k, f"x must have {k} channels")
    elif x is not None:
        _check_rows(x, "x", k)
        _require(x.dtype == weight.dtype, "x and weight must have the same type")
    dev = weight.device
    _require(x is None or x.device == dev, "x and weight must be on the same device")
    _require(act in ACTIVATIONS, f"act must be one of {', '.join(ACTIVATIONS)}")
    out_dtype = weight.dtype if out_dtype is None else out_dtype
    _require(out_dtype in (weight.dtype, torch.float32), "out_dtype must be float32 or the weight's type")
    a = _lib.LinearArgs()
    a.x, a.x_scale = (x.q.data_ptr(), x.scale.data_ptr()) if isinstance(x, Rows8) else (_ptr(x), None)
    a.w = weight.data_ptr()
    lead = tuple(x.shape[:-1]) if lead is None else lead
    a.rows, a.k, a.n, a.act = _rows_of(lead + (k,)), k, n, ACTIVATIONS[act]
    a.dtype = a.bias_dtype = _DTYPES[weight.dtype]
    a.out_dtype = _DTYPES[out_dtype]
    return a, lead, out_dtype, dev


def _linear_call(name, a, dev):
    """Workspace and call of plattice_linear or plattice_linear_backward."""
    b = ctypes.c_size_t(0)
    rc = _call(dev.index, getattr(_lib_h(), name + "_workspace_size"), ctypes.byref(a), ctypes.byref(b))
    if rc:
        _raise(name + "_workspace_size", rc, f"rows={a.rows} k={a.k} n={a.n} split={a.split}")
    ws = torch.empty(b.value, dtype=torch.uint8, device=dev)
    a.workspace, a.workspace_bytes = ws.data_ptr(), b.value
    rc = _call(dev.index, getattr(_lib_h(), name), ctypes.byref(a), _raw_stream(dev.index))
    if rc:
        _raise(name, rc, f"rows={a.rows} k={a.k} n={a.n} split={a.split}")


def linear(x, weight, bias=None, act="none", residual=None, split=0, out_dtype=None, keep=None):
    """``y = act(x weight^T + bias) + residual``: ``(y, z)``.

    ``x [..., k]`` in the weight's type, or :class:`Rows8` (weight float32 or
    bfloat16); ``weight [n, k]``; ``bias [n]`` of any of the three types; ``act``
    one of "none", "relu", "gelu", "silu"; ``residual [..., n]`` in the output's
    type, which is the weight's or float32 (``out_dtype``).  ``split`` (without
    activation and residual): ``y`` is the pair ``([..., split], [..., n -
    split])``, such as the features and values of a filter call.  ``keep``:
    the pre-activation ``z`` for the backward of an activation, "8bit" as Rows8
    or "full" in the output's type (None: ``z`` is None)."""
    cpp = _cpp()
    if (cpp is not None and act in ACTIVATIONS and keep in _KEEP and type(split) is int and isinstance(weight, torch.Tensor)
            and (out_dtype is None or out_dtype is torch.float32 or out_dtype is weight.dtype)):
        eight = type(x) is Rows8
        got = cpp.rows_linear(x.q if eight else x, x.scale if eight else None, x.shape if eight else None, weight, bias,
                              ACTIVATIONS[act], residual, split,
                              out_dtype is torch.float32 or weight.dtype is torch.float32, _KEEP[keep])
        if got is not None:
            if type(got) is int:
                _raise("plattice_linear", got, f"x={tuple(x.shape)} weight={tuple(weight.shape)} split={split}")
            y0, y1, z, z_scale = got
            if z_scale is not None:
                z = _made8(z, z_scale, (*x.shape[:-1], weight.shape[0]))
            return (y0 if y1 is None else (y0, y1)), z
    a, lead, out_dtype, dev = _linear_common(x, weight, act, out_dtype)
    n, split = a.n, int(split)
    _require(0 <= split < n, "split must be in [0, n)")
    _require(not split or (act == "none" and residual is None), "split takes no activation and no residual")
    _require(keep in (None, "8bit", "full"), "keep must be None, '8bit' or 'full'")
    if bias is not None:
        _check_param(bias, "bias", n, dev)
        a.bias, a.bias_dtype = bias.data_ptr(), _DTYPES[bias.dtype]
    if residual is not None:
        _check_like(residual, "residual", lead + (n,), out_dtype, dev)
        a.residual = residual.data_ptr()
    a.split = split
    if split:
        y = (torch.empty(lead + (split,), dtype=out_dtype, device=dev),
             torch.empty(lead + (n - split,), dtype=out_dtype, device=dev))
        a.y0, a.y1 = y[0].data_ptr(), y[1].data_ptr()
    else:
        y = torch.empty(lead + (n,), dtype=out_dtype, device=dev)
        a.y0 = y.data_ptr()
    z = None
    if keep == "8bit":
        z = _empty8(lead + (n,), dev)
        a.z, a.z_scale = z.q.data_ptr(), z.scale.data_ptr()
    elif keep == "full":
        z = torch.empty(lead + (n,), dtype=out_dtype, device=dev)
        a.z = z.data_ptr()
    _linear_call("plattice_linear", a, dev)
    return y, z


def linear_backward(grad_y, x, weight, z=None, act="none", bias_dtype=None, need=(True, True, True)):
    """Gradients of :func:`linear`: ``(grad_x, grad_weight, grad_bias)``, the
    first two in the weight's type, ``grad_bias`` in ``bias_dtype`` (default the
    weight's); ``need`` says which are wanted (None for the others).

    ``grad_y`` as the forward's ``y`` (a pair after a split); ``x`` and ``z`` what
    the forward read and kept, tensors or :class:`Rows8` (``z`` only with an
    activation; ``x`` may be None when ``grad_weight`` is not wanted).  The
    gradient of the residual is ``grad_y`` itself."""
    pair = isinstance(grad_y, (tuple, list))
    _require(not pair or (len(grad_y) == 2 and all(isinstance(g, torch.Tensor) for g in grad_y)),
             "grad_y must be a tensor or a pair of tensors")
    cpp = _cpp()
    if cpp is not None and act in ACTIVATIONS and x is not None:
        eight, z8 = type(x) is Rows8, type(z) is Rows8
        got = cpp.rows_linear_backward(
            *(grad_y if pair else (grad_y, None)), x.q if eight else x, x.scale if eight else None,
            x.shape if eight else None, weight, z.q if z8 else z, z.scale if z8 else None, z.shape if z8 else None,
            ACTIVATIONS[act], _DTYPES.get(getattr(weight, "dtype", None) if bias_dtype is None else bias_dtype, -1),
            bool(need[0]), bool(need[1]), bool(need[2]))
        if got is not None:
            if type(got) is int:
                _raise("plattice_linear_backward", got, f"x={tuple(x.shape)} weight={tuple(weight.shape)}")
            return got
    first = grad_y[0] if pair else grad_y
    _check_rows(first, "grad_y")
    _require(x is not None or not need[1], "x is needed for grad_weight")
    a, lead, out_dtype, dev = _linear_common(x, weight, act, first.dtype, tuple(first.shape[:-1]) if x is None else None)
    n = a.n
    if pair:
        a.split = int(first.shape[-1])
        _require(a.split < n, "grad_y's two tensors must have n channels together")
        _require(act == "none", "split takes no activation and no residual")
        _check_like(first, "grad_y[0]", lead + (a.split,), out_dtype, dev)
        _check_like(grad_y[1], "grad_y[1]", lead + (n - a.split,), out_dtype, dev)
        a.grad0, a.grad1 = first.data_ptr(), grad_y[1].data_ptr()
    else:
        _check_like(grad_y, "grad_y", lead + (n,), out_dtype, dev)
        a.grad0 = grad_y.data_ptr()
    if act != "none":
        _require(z is not None, "z is needed for the backward of an activation")
        if isinstance(z, Rows8):
            z = Rows8(z.q, z.scale, z.shape)
            _require(z.shape == lead + (n,), f"z must be {lead + (n,)}")
            _require(z.device == dev, "z must be on the rows' device")
            a.z, a.z_scale = z.q.data_ptr(), z.scale.data_ptr()
        else:
            _check_like(z, "z", lead + (n,), out_dtype, dev)
            a.z = z.data_ptr()
    bias_dtype = weight.dtype if bias_dtype is None else bias_dtype
    _require(bias_dtype in _DTYPES, "bias_dtype must be float32, bfloat16 or float16")
    a.bias_dtype = _DTYPES[bias_dtype]
    grad_x = torch.empty(lead + (a.k,), dtype=weight.dtype, device=dev) if need[0] else None
    grad_w = torch.empty_like(weight) if need[1] else None
    grad_b = torch.empty((n,), dtype=bias_dtype, device=dev) if need[2] else None
    a.grad_x, a.grad_w, a.grad_bias = _ptr(grad_x), _ptr(grad_w), _ptr(grad_b)
    _linear_call("plattice_linear_backward", a, dev)
    return grad_x, grad_w, grad_b


# ---------------------------------------------------------------- rows from labels

def _check_labels(t, name, shape, device):
    _check_input(t, name)
    _require(t.dtype in (torch.int64, torch.int32), f"{name} must be int64 or int32")
    _require(shape is None or tuple(t.shape) == tuple(shape), f"{name} must be {None if shape is None else tuple(shape)}")
    _require(t.device == device, f"{name} must be on the rows' device")


def _check_scale(scale):
    _require(isinstance(scale, (int, float)) and abs(scale) <= _MOST, "scale must be a finite number of float32")


def embed(ids, table, scale=1.0):
    """Rows from labels: ``y [..., c] = scale * table[ids]`` in the type of
    ``table [n, c]`` (at most 2^21 channels), ``ids [...]`` int64 or int32.  A
    label outside ``0..n-1`` (the "ignored" of label maps) gives a row of zeros."""
    cpp = _cpp()
    if cpp is not None and type(scale) in (float, int) and abs(scale) <= _MOST and (got := cpp.rows_embed(ids, table, scale)) is not None:
        if type(got) is int:
            _raise("plattice_embed", got, f"ids={tuple(ids.shape)} table={tuple(table.shape)}")
        return got
    _check_input(table, "table")
    _require(table.dtype in _DTYPES, "table must be float32, bfloat16 or float16")
    _require(table.dim() == 2 and 1 <= table.shape[0] < 1 << 31 and 1 <= table.shape[1] <= _MAX_EMBED,
             "table must be [n, c], c at most 2^21")
    _check_labels(ids, "ids", None, table.device)
    _check_scale(scale)
    n, c = (int(s) for s in table.shape)
    y = torch.empty((*ids.shape, c), dtype=table.dtype, device=table.device)
    rc = _call(y.device.index, _lib_h().plattice_embed, y.data_ptr(), ids.data_ptr(), int(ids.dtype == torch.int64),
               table.data_ptr(), _DTYPES[table.dtype], scale, ids.numel(), n, c, _raw_stream(y.device.index))
    if rc:
        _raise("plattice_embed", rc, f"ids={tuple(ids.shape)} table={tuple(table.shape)}")
    return y


def embed_backward(grad_y, ids, n, scale=1.0, dtype=None):
    """Gradient of :func:`embed`'s table: ``[n, c]`` in ``dtype`` (default
    ``grad_y``'s), row v the sum of ``scale * grad_y`` over the places where
    ``ids`` is v.  Fewer than 2^31 ids."""
    cpp = _cpp()
    if (cpp is not None and type(scale) in (float, int) and abs(scale) <= _MOST and type(n) is int and (dtype is None or dtype in _DTYPES) and 0 < n < 1 << 31
            and (got := cpp.rows_embed_backward(grad_y, ids, n, scale, -1 if dtype is None else _DTYPES[dtype])) is not None):
        if type(got) is int:
            _raise("plattice_embed_backward", got, f"ids={tuple(ids.shape)} n={n} c={grad_y.shape[-1]}")
        return got
    _check_rows(grad_y, "grad_y")
    c, dev = int(grad_y.shape[-1]), grad_y.device
    _require(c <= _MAX_EMBED, "grad_y must have at most 2^21 channels")
    _check_labels(ids, "ids", grad_y.shape[:-1], dev)
    _require(ids.numel() < 1 << 31, "ids must be fewer than 2^31")
    _require(isinstance(n, int) and 1 <= n < 1 << 31, "n must be in [1, 2^31)")
    _check_scale(scale)
    dtype = grad_y.dtype if dtype is None else dtype
    _require(dtype in _DTYPES, "dtype must be float32, bfloat16 or float16")
    b = ctypes.c_size_t(0)
    rc = _lib_h().plattice_embed_backward_workspace_size(ids.numel(), n, c, ctypes.byref(b))
    if rc:
        _raise("plattice_embed_backward_workspace_size", rc, f"ids={tuple(ids.shape)} n={n} c={c}")
    grad = torch.empty((n, c), dtype=dtype, device=dev)
    ws = torch.empty(b.value, dtype=torch.uint8, device=dev)
    rc = _call(dev.index, _lib_h().plattice_embed_backward, grad.data_ptr(), _DTYPES[dtype], grad_y.data_ptr(),
               _DTYPES[grad_y.dtype], ids.data_ptr(), int(ids.dtype == torch.int64), scale, ws.data_ptr(), b.value,
               ids.numel(), n, c, _raw_stream(dev.index))
    if rc:
        _raise("plattice_embed_backward", rc, f"ids={tuple(ids.shape)} n={n} c={c}")
    return grad


# ---------------------------------------------------------------- recurrence along lines

def _scan_common(x, gate, blend, reverse):
    """Checked (args struct, shape of a state, shape of the kept states, device) of a scan."""
    _check_rows(x, "x")
    _require(x.dim() >= 2, "x must be [..., steps, channels]")
    _check_like(gate, "gate", x.shape, x.dtype, x.device)
    a = _lib.ScanArgs()
    a.x, a.gate = x.data_ptr(), gate.data_ptr()
    a.steps, a.c = int(x.shape[-2]), int(x.shape[-1])
    a.lines = _rows_of(x.shape[:-1])
    a.dtype, a.blend, a.reverse = _DTYPES[x.dtype], bool(blend), bool(reverse)
    lead = tuple(x.shape[:-2])
    return a, lead + (a.c,), lead + (-(-a.steps // _SCAN_KEEP), a.c), x.device


def _scan_call(name, a, dev):
    b = ctypes.c_size_t(0)
    rc = _call(dev.index, getattr(_lib_h(), name + "_workspace_size"), ctypes.byref(a), ctypes.byref(b))
    if rc:
        _raise(name + "_workspace_size", rc, f"lines={a.lines} steps={a.steps} c={a.c}")
    ws = torch.empty(b.value, dtype=torch.uint8, device=dev)
    a.workspace, a.workspace_bytes = ws.data_ptr(), b.value
    rc = _call(dev.index, getattr(_lib_h(), name), ctypes.byref(a), _raw_stream(dev.index))
    if rc:
        _raise(name, rc, f"lines={a.lines} steps={a.steps} c={a.c}")


def scan(x, gate, state=None, blend=False, reverse=False, keep=False):
    """Gated linear recurrence along the lines of ``x [..., steps, c]``:
    ``h[t] = gate[t] h[t-1] + x[t]``, with ``blend`` ``gate[t] h[t-1] + (1 -
    gate[t]) x[t]``, for every line and channel by itself: ``(h, last, states)``.

    ``gate`` as ``x`` (0 starts afresh, so that lines of several lengths can lie
    behind one another; beyond 1 in magnitude is allowed, as long as the recurrence
    stays in float32).  ``state [..., c]`` float32: h before the first step (None: zeros).  ``last [..., c]`` float32: h after the last, to go
    on from (a single step at a time is ``steps`` 1).  ``reverse``: the steps are
    taken from the last to the first.  The recurrence is held in float32, ``h`` is
    its rounding to the type of ``x``.  ``states``: with ``keep`` what
    :func:`scan_backward` needs, h before every 16th step in float32."""
    cpp = _cpp()
    if cpp is not None and (got := cpp.rows_scan(x, gate, state, bool(blend), bool(reverse), bool(keep))) is not None:
        if type(got) is int:
            _raise("plattice_scan", got, f"x={tuple(x.shape)}")
        return got
    a, one, many, dev = _scan_common(x, gate, blend, reverse)
    if state is not None:
        _check_like(state, "state", one, torch.float32, dev)
        a.state = state.data_ptr()
    h = torch.empty_like(x)
    last = torch.empty(one, dtype=torch.float32, device=dev)
    states = torch.empty(many, dtype=torch.float32, device=dev) if keep else None
    a.h, a.last, a.states = h.data_ptr(), last.data_ptr(), _ptr(states)
    _scan_call("plattice_scan", a, dev)
    return h, last, states


def scan_backward(grad_h, x, gate, states, grad_last=None, blend=False, reverse=False):
    """Gradients of :func:`scan` from its inputs and the ``states`` it kept:
    ``(grad_x, grad_gate, grad_state)``, the first two in the type of ``x``, the
    last ``[..., c]`` in float32.  ``grad_last`` (float32) is the gradient of
    ``last``, None for zeros."""
    cpp = _cpp()
    if (cpp is not None
            and (got := cpp.rows_scan_backward(grad_h, x, gate, states, grad_last, bool(blend), bool(reverse))) is not None):
        if type(got) is int:
            _raise("plattice_scan_backward", got, f"x={tuple(x.shape)}")
        return got
    a, one, many, dev = _scan_common(x, gate, blend, reverse)
    _check_like(grad_h, "grad_h", x.shape, x.dtype, dev)
    _check_like(states, "states", many, torch.float32, dev)
    if grad_last is not None:
        _check_like(grad_last, "grad_last", one, torch.float32, dev)
        a.grad_last = grad_last.data_ptr()
    grad_x, grad_gate = torch.empty_like(x), torch.empty_like(x)
    grad_state = torch.empty(one, dtype=torch.float32, device=dev)
    a.grad_h, a.states = grad_h.data_ptr(), states.data_ptr()
    a.grad_x, a.grad_gate, a.grad_state = grad_x.data_ptr(), grad_gate.data_ptr(), grad_state.data_ptr()
    _scan_call("plattice_scan_backward", a, dev)
    return grad_x, grad_gate, grad_state


# ---------------------------------------------------------------- log probabilities

class LogProbs(collections.namedtuple("LogProbs", "logp entropy lse stats top_logp top_ids")):
    """What :func:`log_probs` gives: ``logp [...]`` of the labels (None without
    labels), ``entropy [...]``, ``lse [...]`` the logarithm of the sum of the
    scores' exponentials, ``stats [..., 2]`` its two parts (the largest score, the
    logarithm of the sum relative to it) for the backward, ``top_logp [..., top]``
    and ``top_ids [..., top]`` the best alternatives (None without); all float32
    but the int64 ids."""

    __slots__ = ()


def _log_probs_common(logits, labels):
    _check_rows(logits, "logits")
    a = _lib.LogProbsArgs()
    a.logits, a.dtype = logits.data_ptr(), _DTYPES[logits.dtype]
    a.rows, a.n = _rows_of(logits.shape), int(logits.shape[-1])
    if labels is not None:
        _check_labels(labels, "labels", logits.shape[:-1], logits.device)
        a.labels, a.labels_wide = labels.data_ptr(), labels.dtype == torch.int64
    return a, tuple(logits.shape[:-1]), logits.device


def log_probs(logits, labels=None, top=0):
    """Log probabilities under the softmax of the rows ``logits [..., n]``:
    those of ``labels [...]`` (int64 or int32; outside ``0..n-1``, the "ignored"
    of label maps, 0), the rows' entropies and the ``top`` (at most 32) best
    alternatives, falling, of equal scores the lowest class first.  Gives
    :class:`LogProbs`.

    A score of -inf is a class that the row may not have; a row of nothing else
    has log probabilities of -inf and entropy 0.  NaN or +inf in a row make its
    numbers NaN (of the alternatives' classes NaN is the last choice)."""
    cpp = _cpp()
    if cpp is not None and type(top) is int and 0 <= top <= _MAX_TOP and (got := cpp.rows_log_probs(logits, labels, top)) is not None:
        if type(got) is int:
            _raise("plattice_log_probs", got, f"logits={tuple(logits.shape)} top={top}")
        return LogProbs._make(got)
    a, lead, dev = _log_probs_common(logits, labels)
    _require(isinstance(top, int) and 0 <= top <= min(_MAX_TOP, a.n), f"top must be in [0, min(n, {_MAX_TOP})]")
    new = lambda *s, dtype=torch.float32: torch.empty(lead + s, dtype=dtype, device=dev)  # noqa: E731
    r = LogProbs(None if labels is None else new(), new(), new(), new(2), new(top) if top else None,
                 new(top, dtype=torch.int64) if top else None)
    a.logp, a.entropy, a.lse, a.stats = _ptr(r.logp), r.entropy.data_ptr(), r.lse.data_ptr(), r.stats.data_ptr()
    a.top, a.top_logp, a.top_ids = top, _ptr(r.top_logp), _ptr(r.top_ids)
    rc = _call(dev.index, _lib_h().plattice_log_probs, ctypes.byref(a), _raw_stream(dev.index))
    if rc:
        _raise("plattice_log_probs", rc, f"logits={tuple(logits.shape)} top={top}")
    return r


def log_probs_backward(logits, result, labels=None, grad_logp=None, grad_entropy=None, grad_lse=None):
    """Gradient of the ``logits`` of :func:`log_probs` in their type, from its
    ``result``, the same ``labels`` and the gradients (float32 ``[...]``, None for
    zeros) of ``logp``, ``entropy`` and ``lse``.  The alternatives have none.  A row
    of -inf only has gradient 0."""
    cpp = _cpp()
    if (cpp is not None and type(result) is LogProbs
            and (got := cpp.rows_log_probs_backward(logits, result.stats, result.entropy, labels, grad_logp, grad_entropy,
                                                    grad_lse)) is not None):
        if type(got) is int:
            _raise("plattice_log_probs_backward", got, f"logits={tuple(logits.shape)}")
        return got
    a, lead, dev = _log_probs_common(logits, labels)
    _require(isinstance(result, LogProbs), "result must be LogProbs")
    _check_like(result.stats, "result.stats", lead + (2,), torch.float32, dev)
    _require(grad_logp is None or labels is not None, "labels are needed for grad_logp")
    a.stats = result.stats.data_ptr()
    if grad_entropy is not None:
        _check_like(result.entropy, "result.entropy", lead, torch.float32, dev)
        a.entropy = result.entropy.data_ptr()
    for name, g in (("grad_logp", grad_logp), ("grad_entropy", grad_entropy), ("grad_lse", grad_lse)):
        if g is not None:
            _check_like(g, name, lead, torch.float32, dev)
            setattr(a, name, g.data_ptr())
    grad = torch.empty_like(logits)
    a.grad_logits = grad.data_ptr()
    rc = _call(dev.index, _lib_h().plattice_log_probs_backward, ctypes.byref(a), _raw_stream(dev.index))
    if rc:
        _raise("plattice_log_probs_backward", rc, f"logits={tuple(logits.shape)}")
    return grad
