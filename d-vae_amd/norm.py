"""Layer norm over the last dimension on libdvae_hip, with gradients: ``layer_norm`` and the module ``LayerNorm``.

The networks of the reference normalise over images (BatchNorm2d, InstanceNorm2d: configs/models/resnet.py:27-30,
:2014-2020); this is the normalisation over a vector's own elements, with torch.nn.LayerNorm's formula, parameter names and
``state_dict``.  Data is fp32 or bf16, parameters and their gradients are fp32, statistics are fp32 whatever the data.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib as L

_DTYPES = {torch.float32: L.F32, torch.bfloat16: L.BF16}


def _check(x, weight, bias, eps):
    L.refuse_tangents("layer_norm", x, weight, bias)
    if not x.is_cuda:
        raise RuntimeError("layer_norm runs on libdvae_hip: x must be a device tensor")
    if x.dtype not in _DTYPES:
        raise RuntimeError(f"layer_norm: x is {x.dtype}; float32 and bfloat16 are supported")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise RuntimeError(f"layer_norm: x of shape {tuple(x.shape)} has no elements to normalise over")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and (p.dtype != torch.float32 or p.device != x.device or p.dim() != 1 or p.shape[0] != x.shape[-1]):
            raise RuntimeError(f"layer_norm: {name} must be float32 of shape ({x.shape[-1]},) on {x.device}, got {p.dtype} "
                               f"{tuple(p.shape)} on {p.device}")
    if not eps >= 0.0:
        raise RuntimeError(f"layer_norm: eps {eps}")


def _rows(t, c):
    """t as rows of c adjacent elements: a view wherever strides allow it (padded, sliced and expanded rows do)."""
    if t.dim() != 2:
        t = t.reshape(-1, c)
    return t if t.stride(1) == 1 or c == 1 else t.contiguous()


def _param(p):
    return p if p is None or p.is_contiguous() else p.contiguous()


def _forward(x, weight, bias, eps, save):
    c = x.shape[-1]
    x2 = _rows(x, c)
    rows = x2.shape[0]
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device) if save else None
    if rows:
        weight, bias = _param(weight), _param(bias)
        mean = stats.data_ptr() if save else None
        L.check(L.lib().dvae_layer_norm_fwd(x2.data_ptr(), x2.stride(0), L.ptr(weight), L.ptr(bias), y.data_ptr(), c, mean,
                                            mean + 4 * rows if save else None, rows, c, eps, _DTYPES[x.dtype], L.stream()))
    return y, stats


def _backward(ctx, dy):
    x, weight, stats = ctx.saved_tensors
    want_x, want_w, want_b, _ = ctx.needs_input_grad
    if dy.dtype != x.dtype:
        dy = dy.to(x.dtype)
    with L.on_device(x.device):
        c = x.shape[-1]
        x2, dy2 = _rows(x, c), _rows(dy, c)
        rows, dtype, lib = x2.shape[0], _DTYPES[x.dtype], L.lib()
        dx = torch.empty_like(x, memory_format=torch.contiguous_format) if want_x else None
        dw = torch.empty(c, device=x.device, dtype=torch.float32) if want_w else None
        db = torch.empty(c, device=x.device, dtype=torch.float32) if want_b else None
        ws, n = None, 0
        if want_w or want_b:
            n = lib.dvae_layer_norm_workspace_bytes(rows, c, dtype)
            ws = torch.empty(n, device=x.device, dtype=torch.uint8)
        weight = _param(weight)
        mean = stats.data_ptr()
        L.check(lib.dvae_layer_norm_bwd(dy2.data_ptr(), dy2.stride(0), x2.data_ptr(), x2.stride(0), L.ptr(weight), mean,
                                        mean + 4 * rows, L.ptr(dx), c, L.ptr(dw), L.ptr(db), L.ptr(ws), n, rows, c, dtype,
                                        L.stream()))
    return dx, dw, db, None


class _FirstGradient(torch.autograd.Function):
    """The identity on one of the gradients, as a function of the tensors it depends on: where any of them is being
    differentiated the gradient says so (requires_grad), and its own backward raises."""

    @staticmethod
    def forward(ctx, grad, *of):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("layer_norm: its gradients can be taken once; there are no second derivatives")


def _backward_once(ctx, dy):
    with torch.no_grad():
        dx, dw, db, _ = _backward(ctx, dy)
    x, weight, _ = ctx.saved_tensors
    return (None if dx is None else _FirstGradient.apply(dx, dy, x, weight), None if dw is None else _FirstGradient.apply(dw, dy, x),
            None if db is None else _FirstGradient.apply(db, dy), None)


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        return y

    @staticmethod
    def backward(ctx, dy):
        # the guard against second derivatives costs a third of a small call's backward: only where a graph is being built
        return _backward_once(ctx, dy) if torch.is_grad_enabled() else _backward(ctx, dy)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of ``x``.

    ``x``: float32 or bfloat16 on the device, any shape and strides; rows that are slices of wider ones (an activation map
    without its padding channels) are read in place, other layouts are copied once.  ``weight`` / ``bias``: float32 of the
    last dimension's size, or None.  The result is contiguous and of x's type.  Gradients flow to all three and can be taken
    once (no second derivatives, no forward mode).  A step captured into a graph follows torch's rule for captured backward passes: no eager
    graph of the same leaves may be alive during the capture."""
    _check(x, weight, bias, eps)
    with L.on_device(x.device):
        if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                        (bias is not None and bias.requires_grad)):
            return _LayerNormFunction.apply(x, weight, bias, eps)
        return _forward(x, weight, bias, eps, False)[0]


class LayerNorm(nn.Module):
    """torch.nn.LayerNorm over the last dimension (same parameter names) on ``layer_norm``.  The parameters have to be
    float32, whatever type the data has: after a ``.bfloat16()`` or ``.half()`` of the module its calls are refused."""

    def __init__(self, channels, eps=1e-5, affine=True):
        super().__init__()
        self.channels, self.eps = int(channels), float(eps)
        self.weight = nn.Parameter(torch.ones(self.channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(self.channels)) if affine else None

    def forward(self, x):
        if x.shape[-1] != self.channels:
            raise RuntimeError(f"LayerNorm({self.channels}): the last dimension of x is {x.shape[-1]}")
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return f"{self.channels}, eps={self.eps}, affine={self.weight is not None}"
