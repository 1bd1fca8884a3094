"""Drop-in replacement of the reference's plattice.py (plattice.py:7-23).

``PermutoLatticeFunction`` is the autograd Function: forward returns the
filtered values and saves ``(weight, feature)``; backward returns
``(None, grad_values)``: no gradient flows to the features, as in the
reference (plattice.py:19).  ``PermutoLattice`` is the nn.Module wrapper.

Unlike the reference, the lattice that forward builds is kept on the autograd
context and reused by backward (no rebuild), unless ``PLOO.set_keep_lattice(False)``
(or PLATTICE_KEEP_LATTICE=0) asks for the reference's behaviour: nothing kept,
the lattice rebuilt in backward.

``PermutoLatticeBatchFunction`` (no counterpart in the reference) is
``PermutoLatticeFunction`` over a batch ``[B,H,W,...]`` in one library call,
one lattice per image.

``PermutoLatticeFeatureFunction`` (no counterpart in the reference) is
``PermutoLatticeFunction`` with a gradient for the features as well: the
slope of the piecewise-linear filter inside each pixel's simplex.

``LatticeFilterFunction`` (no counterpart in the reference) filters further
values on a kept lattice -- the ``PLOO.Lattice`` of an earlier forward on the
same features -- without rebuilding it, as the iterations of a mean-field CRF
do; its backward is the value gradient on the same lattice.

``RowLinearFunction`` and ``RowNormLinearFunction`` (no counterpart in the
reference) are the row operators of ``rows.py`` under autograd, and
``PermutoLatticeLayer`` chains them around the filter: norm, projection to
learned features and values, filter, projection back, residual.
"""
import ctypes
import math

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable
from torch.nn import Module, Parameter

from . import PLOO, _lib, rows

_UNSET = object()
_EXT = _UNSET


def _cpp_function():
    """The C++ build of PermutoLatticeFunction (extension module _plattice_torch,
    built next to the library), pointed at the loaded library's entry points;
    None when the extension is not built."""
    global _EXT
    if _EXT is _UNSET:
        try:
            from . import _plattice_torch as m
        except ImportError:
            _EXT = None
            return None
        L = _lib.lib()
        addr = lambda f: ctypes.cast(f, ctypes.c_void_p).value
        m.set_entry_points(addr(L.plattice_forward), addr(L.plattice_backward), addr(L.plattice_workspace_sizes),
                           addr(L.plattice_reuse_scratch_size), addr(L.plattice_error_string),
                           addr(L.plattice_last_error_detail))
        _EXT = m.permuto_lattice
    return _EXT

__all__ = ["PermutoLatticeFunction", "PermutoLattice", "LatticeFilterFunction", "PermutoLatticeBatchFunction",
           "PermutoLatticeFeatureFunction", "RowLinearFunction", "RowNormLinearFunction", "PermutoLatticeLayer"]


class PermutoLatticeFunction(Function):
    """``PermutoLatticeFunction.apply(feature, values) -> out``.

    ``apply`` runs the C++ build of this Function (the same checks, messages,
    kept lattice and library calls as forward / backward below, without the
    Python interpreter between the autograd engine and the library) when the
    extension is built and PLATTICE_CHECK is off; otherwise, and for arguments
    that are not tensors, the Python Function below.  Either way the filter
    runs in libplattice_b200.so."""

    @classmethod
    def apply(cls, feature, values):
        fn = None if PLOO._CHECK else _cpp_function()
        if fn is not None and type(feature) is torch.Tensor and type(values) is torch.Tensor:
            return fn(feature, values, PLOO._KEEP)
        return super().apply(feature, values)

    @staticmethod
    def forward(ctx, feature, values):
        weight, out, lat = PLOO.lattice_forward(feature, values)
        ctx.save_for_backward(weight, feature)
        ctx.lattice = lat if PLOO._KEEP else None
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        weight, feature = ctx.saved_tensors
        grad_values = PLOO.lattice_backward(feature, grad_output.contiguous(), weight,
                                            getattr(ctx, "lattice", None), saved=True)
        return None, grad_values


class PermutoLattice(Module):
    def forward(self, feature, values):
        return PermutoLatticeFunction.apply(feature, values)


class LatticeFilterFunction(Function):
    """``LatticeFilterFunction.apply(values, lattice) -> out``: the forward filter
    of ``values`` on the kept ``lattice``; gradient to ``values`` only."""

    @staticmethod
    def forward(ctx, values, lattice):
        weight, out = PLOO.lattice_filter(lattice, values)
        ctx.save_for_backward(weight)
        ctx.lattice = lattice
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        (weight,) = ctx.saved_tensors
        return PLOO.lattice_filter_backward(ctx.lattice, grad_output.contiguous(), weight), None


class PermutoLatticeBatchFunction(Function):
    """``PermutoLatticeBatchFunction.apply(features [B,H,W,pd], values [B,H,W,vd])``."""

    @staticmethod
    def forward(ctx, feature, values):
        weight, out, lat = PLOO.batch_forward(feature, values)
        ctx.save_for_backward(weight, feature)
        ctx.lattice = lat if PLOO._KEEP else None
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        weight, feature = ctx.saved_tensors
        grad_values = PLOO.batch_backward(feature, grad_output.contiguous(), weight,
                                          getattr(ctx, "lattice", None), saved=True)
        return None, grad_values


def _long_rows(shape):
    """The shape as which an image [H, W, vd] is kept in 8 bits: one long row,
    with blocks of 32 values across pixels (a pixel's own 1 to 8 values would
    fill a block of their own), or one per line of an image that no row holds."""
    n = math.prod(shape)
    return (n,) if n <= rows._MAX_CHANNELS else (shape[0], n // shape[0])


class PermutoLatticeFeatureFunction(Function):
    """``PermutoLatticeFeatureFunction.apply(features, values) -> out`` with
    gradients for both inputs.  The feature gradient needs ``values`` and
    ``out`` again; ``PLOO.set_checkpoint_precision("8bit")`` keeps them in 8 bits."""

    @staticmethod
    def forward(ctx, feature, values):
        weight, out, lat = PLOO.lattice_forward(feature, values)
        ctx.lattice = lat
        ctx.shape = out.shape
        ctx.eight = PLOO._CHECKPOINT8 and out.numel() > 0
        if ctx.eight:
            kept = [rows.pack8(t.view(_long_rows(t.shape))) for t in (values, out)] if ctx.needs_input_grad[0] else []
            ctx.save_for_backward(weight, feature, *(t for r in kept for t in (r.q, r.scale)))
        else:
            ctx.save_for_backward(weight, feature, values, out)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        weight, feature, *kept = ctx.saved_tensors
        g = grad_output.contiguous()
        grad_features = None
        if ctx.needs_input_grad[0]:
            if ctx.eight:
                values, out = (rows.unpack8(rows.Rows8(kept[i], kept[i + 1], _long_rows(ctx.shape))).view(ctx.shape)
                               for i in (0, 2))
            else:
                values, out = kept
            grad_features = PLOO.feature_grad(ctx.lattice, feature, values, g, weight, out)
        grad_values = None
        if ctx.needs_input_grad[1]:
            grad_values = PLOO.lattice_backward(feature, g, weight, ctx.lattice, saved=True)
        return grad_features, grad_values


# ---------------------------------------------------------------- row operators

def _save(ctx, *kept):
    """save_for_backward of tensors, Rows8 and None; _saved gives them back."""
    flat, ctx.layout = [], []
    for t in kept:
        ctx.layout.append(t.shape if isinstance(t, rows.Rows8) else t is not None)
        flat += [t.q, t.scale] if isinstance(t, rows.Rows8) else [] if t is None else [t]
    ctx.save_for_backward(*flat)


def _saved(ctx):
    flat = iter(ctx.saved_tensors)
    return [rows.Rows8(next(flat), next(flat), what) if isinstance(what, tuple) else next(flat) if what else None
            for what in ctx.layout]


class RowLinearFunction(Function):
    """``RowLinearFunction.apply(x, weight, bias, residual, act, checkpoint8) ->
    act(x weight^T + bias) + residual`` over ``x [..., k]``, gradients for the
    first four.  ``checkpoint8``: what the backward needs of the activations is
    kept in 8 bits (``x`` only where that is smaller: 33 bytes per 32 channels,
    so not for a few channels of a 16-bit type, nor for float16 weights), else as
    it is."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act="none", checkpoint8=False):
        y, z = rows.linear(x, weight, bias, act=act, residual=residual,
                           keep=None if act == "none" else "8bit" if checkpoint8 else "full")
        ctx.act, ctx.bias_dtype = act, None if bias is None else bias.dtype
        kept = None
        if ctx.needs_input_grad[1]:
            k = x.shape[-1]
            small = -(-k // 32) * 33 < k * x.element_size()
            kept = rows.pack8(x) if checkpoint8 and small and weight.dtype != torch.float16 else x
        _save(ctx, kept, weight, z)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        x, weight, z = _saved(ctx)
        need = ctx.needs_input_grad
        g = grad_y.contiguous()
        gx, gw, gb = rows.linear_backward(g, x, weight, z, act=ctx.act, bias_dtype=ctx.bias_dtype,
                                          need=(need[0], need[1], need[2]))
        return gx, gw, gb, g if need[3] else None, None, None


class RowNormLinearFunction(Function):
    """``RowNormLinearFunction.apply(x, residual, gain, weight, bias, eps, act,
    split, out_dtype, checkpoint8)``: the root-mean-square norm of ``h = x +
    residual`` and the linear map of its result, as :func:`rows.rms_norm` and
    :func:`rows.linear`; gradients for the first five.  Returns ``y`` (with
    ``split`` its two tensors), followed by ``h`` when there is a residual.

    ``checkpoint8`` (on by default: False for results without 8-bit roundings):
    the norm's result exists only in 8 bits, which the forward and the backward
    both read, and the pre-activation is kept in 8 bits (float16 rows keep both
    as they are).  ``x`` and ``weight`` then may be float32 and bfloat16 or the
    other way; without, they have the same type."""

    @staticmethod
    def forward(ctx, x, residual, gain, weight, bias, eps=1e-6, act="none", split=0, out_dtype=None,
                checkpoint8=True):
        eight = checkpoint8 and x.dtype != torch.float16
        n, h, rstd = rows.rms_norm(x, gain, residual, eps=eps, pack=eight)
        y, z = rows.linear(n, weight, bias, act=act, split=split, out_dtype=out_dtype,
                           keep=None if act == "none" else "8bit" if eight else "full")
        ctx.act, ctx.split, ctx.two = act, split, residual is not None
        ctx.bias_dtype = None if bias is None else bias.dtype
        _save(ctx, n, h, rstd, gain, weight, z)
        outs = (*(y if split else (y,)), *((h,) if ctx.two else ()))
        return outs if len(outs) > 1 else outs[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        n, h, rstd, gain, weight, z = _saved(ctx)
        need = ctx.needs_input_grad
        grads = [g.contiguous() for g in grads]
        gh = grads.pop() if ctx.two else None
        gn, gw, gb = rows.linear_backward(tuple(grads) if ctx.split else grads[0], n, weight, z, act=ctx.act,
                                          bias_dtype=ctx.bias_dtype,
                                          need=(need[0] or need[1] or need[2], need[3], need[4]))
        gx = gg = None
        if gn is not None:   # in the weight's type, which 8-bit rows leave open
            gx, gg = rows.rms_norm_backward(gn.to(h.dtype), h, rstd, gain, gh)
        return (gx if need[0] else None, gx if need[1] else None, gg if need[2] else None, gw, gb,
                None, None, None, None, None)


class PermutoLatticeLayer(Module):
    """A residual layer around the filter with learned features and values:

        n = rms_norm(x) gain;  (f, v) = n W_in^T + b_in;  o = filter(f, v)
        y = act(o W_out^T + b_out) + x

    for ``x [H, W, channels]`` in the parameters' type (float32, bfloat16 or
    float16; the filter itself runs in float32).  ``pd`` features and ``vd``
    values per pixel.  ``checkpoint8``: the norm's result, also as the forward
    reads it, and what the backward needs of the projections are kept in 8 bits
    (each off by at most 2^-4 of itself), else in the parameters' type."""

    def __init__(self, channels, pd, vd, act="none", eps=1e-6, checkpoint8=False, dtype=torch.float32, device=None):
        super().__init__()
        PLOO._check_dims(pd, vd)
        PLOO._require(act in rows.ACTIVATIONS, f"act must be one of {', '.join(rows.ACTIVATIONS)}")
        self.pd, self.act, self.eps, self.checkpoint8 = pd, act, eps, checkpoint8

        def uniform(n, k):
            w = torch.empty(n, k, dtype=torch.float32, device=device).uniform_(-1.0, 1.0)
            return Parameter((w / math.sqrt(k)).to(dtype))
        self.gain = Parameter(torch.ones(channels, dtype=dtype, device=device))
        self.w_in = uniform(pd + vd, channels)
        self.b_in = Parameter(torch.zeros(pd + vd, dtype=dtype, device=device))
        self.w_out = uniform(channels, vd)
        self.b_out = Parameter(torch.zeros(channels, dtype=dtype, device=device))

    def forward(self, x):
        f, v = RowNormLinearFunction.apply(x, None, self.gain, self.w_in, self.b_in, self.eps, "none", self.pd,
                                           torch.float32, self.checkpoint8)
        o = PermutoLatticeFeatureFunction.apply(f, v)
        return RowLinearFunction.apply(o.to(x.dtype), self.w_out, self.b_out, x, self.act, self.checkpoint8)
