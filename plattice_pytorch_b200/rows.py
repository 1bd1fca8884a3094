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

Tensors are contiguous CUDA tensors ``[..., channels]`` of float32, bfloat16
or float16; as for the filter, a failed check raises RuntimeError, kernels run
on PyTorch's current stream of the tensors' device, and no call synchronises.
No reference counterpart.
"""
import ctypes

import torch

from . import _lib
from .PLOO import _call, _check_input, _lib_h, _raise, _raw_stream, _require

__all__ = ["Rows8", "pack8", "unpack8", "rms_norm", "rms_norm_backward", "linear", "linear_backward", "ACTIVATIONS"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
_KEEP = {None: 0, "8bit": 1, "full": 2}
_MAX_NORM = 16384
_MAX_CHANNELS = 1 << 30


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


def _cpp():
    """The torch extension's forms of the calls below (the same tests,
    allocations and library calls in one step), pointed at the loaded library;
    None when the extension is not built, or from older sources.  They answer None to arguments that
    fail a test: the Python form then finds which and raises its message."""
    global _EXT
    if _EXT is _UNSET:
        try:
            from . import _plattice_torch as m
            m.set_rows_entry_points([ctypes.cast(getattr(_lib.lib(), n), ctypes.c_void_p).value for n in _CALLS])
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
