"""The step between a backward pass and an update: the norm of all gradients
together, and the gradients scaled down to a largest norm.

* :func:`grad_norm`  -- ``sqrt(sum g^2)`` over all values of all tensors
* :func:`clip_grads` -- ``out = g * min(1, max_norm / (norm + eps))``

Tensors are contiguous CUDA tensors of any shape, float32, bfloat16 or float16
(mixed as they come), on one device.  The norm stays on the device; as for the
row operators, a failed check raises RuntimeError, kernels run on PyTorch's
current stream of that device, and no call synchronises.  No reference
counterpart.
"""
import ctypes

import torch

from . import _lib
from .PLOO import _call, _check_input, _lib_h, _raise, _raw_stream, _require
from .rows import _DTYPES, _MOST, _check_like, _cpp

__all__ = ["grad_norm", "clip_grads"]

_SHARED = "(none may share memory with what is written)"


def _fits(max_norm):
    return 0 <= max_norm <= _MOST or max_norm == float("inf")


def _listed(tensors, name):
    _require(not isinstance(tensors, torch.Tensor), f"{name} must be a list of tensors")
    tensors = list(tensors)
    _require(len(tensors) > 0, f"{name} must be at least one tensor")
    for i, t in enumerate(tensors):
        _check_input(t, f"{name}[{i}]")
        _require(t.dtype in _DTYPES, f"{name}[{i}] must be float32, bfloat16 or float16")
        _require(t.device == tensors[0].device, f"{name}[{i}] must be on the device of {name}[0]")
    return tensors


def _run(tensors, out, max_norm, eps, norm_in):
    dev = tensors[0].device
    table = (_lib.Grad * len(tensors))()
    for i, t in enumerate(tensors):
        q = table[i]
        q.g, q.size, q.dtype = t.data_ptr(), t.numel(), _DTYPES[t.dtype]
        if out is not None:
            q.out, q.out_dtype = out[i].data_ptr(), _DTYPES[out[i].dtype]
    norm = torch.empty((), dtype=torch.float32, device=dev) if norm_in is None else norm_in
    b = ctypes.c_size_t(0)
    rc = _lib_h().plattice_clip_grads_workspace_size(table, len(tensors), ctypes.byref(b))
    if rc:
        _raise("plattice_clip_grads_workspace_size", rc, f"{len(tensors)} tensors")
    ws = torch.empty(b.value, dtype=torch.uint8, device=dev) if norm_in is None else None
    rc = _call(dev.index, _lib_h().plattice_clip_grads, table, len(tensors), max_norm, eps,
               None if norm_in is None else norm_in.data_ptr(), None if norm_in is not None else norm.data_ptr(),
               None if ws is None else ws.data_ptr(), b.value, _raw_stream(dev.index))
    if rc:
        _raise("plattice_clip_grads", rc, f"{len(tensors)} tensors {_SHARED}")
    return norm


def grad_norm(tensors):
    """Norm of all values of ``tensors`` together: ``sqrt(sum g^2)``, a float32
    tensor without dimensions.  Squares that float32 does not hold are added in
    float64, sums of more than eight always."""
    if not isinstance(tensors, (list, torch.Tensor)):
        tensors = list(tensors)
    cpp = _cpp()
    if cpp is not None and type(tensors) is list and (got := cpp.clip_grads(tensors, None, 0.0, 0.0, None)) is not None:
        if type(got) is int:
            _raise("plattice_clip_grads", got, f"{len(tensors)} tensors")
        return got
    return _run(_listed(tensors, "tensors"), None, 0.0, 0.0, None)


def clip_grads(tensors, max_norm, out=None, norm=None, eps=1e-6):
    """Scales gradients down to a norm of at most ``max_norm``: ``out = g *
    min(1, max_norm / (norm + eps))``; returns the norm before (float32, on the
    device).

    ``out``: tensors like ``tensors``, each in its tensor's type or float32 (None:
    in place; then nothing is written where the norm is small enough).  ``norm``: a
    float32 tensor without dimensions to use instead of the tensors' own norm, such
    as one over the gradients of several processes.  ``max_norm`` may be infinite
    (``out`` is then a copy).  A norm that is not finite scales by 0 or NaN, as
    the formula says.  What is written may share no memory with another tensor of
    either list or with ``norm``, nor may a tensor that is scaled in place be listed twice."""
    if not isinstance(tensors, (list, torch.Tensor)):
        tensors = list(tensors)
    if not isinstance(out, (list, torch.Tensor, type(None))):
        out = list(out)
    cpp = _cpp()
    if (cpp is not None and type(tensors) is list and type(max_norm) in (float, int) and _fits(max_norm)
            and type(eps) in (float, int) and 0 <= eps <= _MOST
            and (got := cpp.clip_grads(tensors, tensors if out is None else out, max_norm, eps, norm)) is not None):
        if type(got) is int:
            _raise("plattice_clip_grads", got, f"{len(tensors)} tensors {_SHARED}")
        return got
    tensors = _listed(tensors, "tensors")
    _require(isinstance(max_norm, (int, float)) and _fits(max_norm), "max_norm must be a number of float32, at least 0")
    _require(isinstance(eps, (int, float)) and 0 <= eps <= _MOST, "eps must be a finite number of float32, at least 0")
    if out is None:
        out = tensors
    else:
        out = _listed(out, "out")
        _require(len(out) == len(tensors), "out must have as many tensors")
        for i, (t, o) in enumerate(zip(tensors, out)):
            _check_like(o, f"out[{i}]", t.shape, o.dtype, t.device)
            _require(o.dtype in (t.dtype, torch.float32), f"out[{i}] must have its tensor's type or float32")
    for i, o in enumerate(out):
        _require(not (o.requires_grad and torch.is_grad_enabled()),
                 f"{'tensors' if out is tensors else 'out'}[{i}] requires grad: write to it under torch.no_grad()")
    if norm is not None:
        _check_like(norm, "norm", (), torch.float32, tensors[0].device)
    got = _run(tensors, out, max_norm, eps, norm)
    torch.autograd.graph.increment_version([o for o in out if not o.is_inference()])
    return got
